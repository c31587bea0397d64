// The next tokens from logits and given random numbers: temperature, top-k, top-p and min-p of each row.
//
// With m the largest logit, T the temperature and w_i = exp((x_i - m) / T), in the order of x (the larger first, of equal ones the
// lower index): the first k tokens are kept; of these the shortest prefix whose weights reach top_p of theirs; of these the
// tokens with w_i >= min_p; the first one in any case. The token is the first one, by index, at which the running sum of the kept
// weights is above u times their total. T = 0: the largest logit, of equal ones the lowest index. NaN counts as -inf, a subnormal
// logit as 0.
//
// Weights are integers, w_i rounded to 2^-40, from an exponential that is good to about 2^-30: x - m and the product with
// log2(e) / T are carried in two floats, 2^(j/32) comes from a table and the rest from a polynomial. Sums of integers do not depend on
// their order, so that a row gives the same token in any batch and with any number of CTAs, and a border between
// two tokens is as sharp as the weights themselves.
//
// A cluster of CTAs takes a row, and each lane keeps its 32 logits in shared memory where eight CTAs can (up to 131072; rows of more
// are read again in every pass, from the caches): a pass costs its arithmetic and an exchange through distributed shared memory.
// (1) Largest logit, and the mean of a sample. (2) Where k or p limits the row: counts (and weights, for p alone) in bins
// of equal width from the largest logit down to about the mean, which spread the atomics of a few thousand candidates over as many
// addresses. (3) The bins down to the one that decides hold few tokens as a rule: these go to a list in one CTA, where the token is
// decided. Where a p alone keeps too many, only the deciding bin is listed, and where even that is too long the deciding value
// is found digit by digit over the row, 11 + 11 + 10 bits of the order-preserving integer of a float. (4) The token from sums of
// 256 neighbours.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../mlf_api.h"

namespace mlf {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int SM_WARPS = 16;
constexpr int SM_THREADS = SM_WARPS * 32;
constexpr int SM_STEP = 256;                   // logits that a warp takes at a time, eight a lane
constexpr int SM_HELD = 4;                     // such steps that a warp can keep in shared memory
constexpr int SM_STEPS = 64;                   // at most, per warp
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 2048;
constexpr int SM_CLUSTER = 8;                  // CTAs per row, at most
constexpr int SM_ONE = 40;                     // log2 of the weight of the largest logit

struct SampleParams {
  const void* logits;
  long long ld;
  int rows, vocab, steps, vec;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  long long* tokens;
  float* logprobs;
};

__constant__ unsigned c_exp2[32] = {           // 2^(j / 32) in units of 2^-31
    0x80000000u, 0x82cd8699u, 0x85aac368u, 0x88980e81u, 0x8b95c1e4u, 0x8ea4398bu, 0x91c3d374u, 0x94f4efa9u, 0x9837f052u, 0x9b8d39bau, 0x9ef53261u,
    0xa2704303u, 0xa5fed6aau, 0xa9a15ab5u, 0xad583eeau, 0xb123f582u, 0xb504f334u, 0xb8fbaf47u, 0xbd08a39fu, 0xc12c4ccau, 0xc5672a11u, 0xc9b9bd86u,
    0xce248c15u, 0xd2a81d92u, 0xd744fccbu, 0xdbfbb798u, 0xe0ccdeecu, 0xe5b906e7u, 0xeac0c6e8u, 0xefe4b99cu, 0xf5257d15u, 0xfa83b2dbu};

struct SampleSmem {
  u64 list[SM_LIST];
  union {
    struct { unsigned lo[SM_BINS], hi[SM_BINS]; };          // weights of the bins
    u64 local[SM_LIST];                                     // the list's entries of this CTA, later scratch of the list
    ulonglong2 pair[SM_THREADS];
  };
  union {
    alignas(16) unsigned cnt[SM_BINS];         // counts of the bins
    u64 step[SM_WARPS * SM_STEPS];             // sums of 256 logits' values
  };
  u64 slot[6][4][SM_CLUSTER];                  // one set per exchange of a launch: values of every CTA
  u64 warp[SM_WARPS];
  u64 res[4];
  unsigned exp2[32];
  int n_list, base;
  int n_local;
  alignas(16) uint4 held[1];                   // SM_HELD steps, as far as the launch has room for them
};

// Order-preserving integer of a float that is not NaN; -0 and subnormal numbers are 0.
__device__ __forceinline__ unsigned sm_key(float x) {
  const unsigned u = __float_as_uint(__fadd_rn(x, 0.f));
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sm_value(unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ u64 sm_entry(float x, int i) { return (u64)(~sm_key(x)) << 32 | (unsigned)i; }      // ascending: the order of the tokens
__device__ __forceinline__ float sm_entry_value(u64 e) { return sm_value(~(unsigned)(e >> 32)); }

struct SampleWeight {
  float m, ch, cl;                             // log2(e) / T in two floats
  const unsigned* table;
  __device__ __forceinline__ u64 operator()(float x) const {     // NaN and -inf: 0
    if (x == m) return 1ull << SM_ONE;
    const float s = __fsub_rn(x, m), t = __fsub_rn(s, x);
    const float r = __fadd_rn(__fsub_rn(x, __fsub_rn(s, t)), -__fadd_rn(m, t));     // x - m = s + r
    const float p = __fmul_rn(s, ch);
    if (!(p > -(SM_ONE + 2.f))) return 0ull;
    const float e = __fmaf_rn(r, ch, __fmaf_rn(s, cl, __fmaf_rn(s, ch, -p)));
    const float big = __fmaf_rn(p, 32.f, 12582912.f);                               // p in 32nds, an integer in the low bits
    const int j = __float_as_int(big) - 0x4b400000;
    const float f = __fadd_rn(__fmaf_rn(__fsub_rn(big, 12582912.f), -0.03125f, p), e);
    // 2^f - 1 = e^(f ln 2) - 1, |f| <= 1 / 64: four terms of the series, the fifth is 2^-39
    const float q = __fmul_rn(f, __fmaf_rn(f, __fmaf_rn(f, __fmaf_rn(f, 0.0096181291f, 0.055504109f), 0.24022651f), 0.69314718f));
    const unsigned tj = table[j & 31];
    const u64 w = (u64)(tj + (unsigned)__float2int_rn(__fmul_rn(q, (float)tj))) << (SM_ONE - 31);
    const int down = -(j >> 5);
    return down > 0 ? (w + (1ull << (down - 1))) >> down : w;
  }
};

__device__ __forceinline__ u64 sm_warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 sm_warp_scan(u64 v) {       // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
// Exclusive prefix over the CTA's threads; *total: the sum. Two barriers.
__device__ __forceinline__ u64 sm_block_scan(u64 v, SampleSmem& s, u64* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const u64 inc = sm_warp_scan(v);
  __syncthreads();
  if (lane == 31) s.warp[warp] = inc;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < SM_WARPS; ++i) {
    const u64 x = s.warp[i];
    before += i < warp ? x : 0;
    all += x;
  }
  *total = all;
  return before + inc - v;
}

// Ascending sort of n entries (a power of two, up to SM_LIST) in shared memory.
__device__ __forceinline__ void sm_sort(u64* a, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += SM_THREADS) {
        const int i = 2 * t - (t & (j - 1));
        const u64 x = a[i], y = a[i + j];
        if ((x > y) == ((i & k) == 0)) { a[i] = y; a[i + j] = x; }
      }
    }
  __syncthreads();
}

// Smallest integer sum that reaches p of `total`; that is above u of it.
__device__ __forceinline__ u64 sm_reach(double p, u64 total) {
  const double t = ceil(p * (double)total);
  return t <= 0. ? 0ull : min((u64)t, total);
}
__device__ __forceinline__ u64 sm_above(float u, u64 total) {
  const double t = floor((double)u * (double)total);
  return t >= 0. ? min((u64)t + 1ull, total) : (t < 0. ? 1ull : total);       // NaN: the last token
}

// A warp's run of a row: `steps` times 256 logits, eight a lane, kept in shared memory (HELD) or read again each time. What lies behind
// the vocabulary is -inf.
template <typename T, bool HELD>
struct SampleRow {
  static constexpr int WORDS = sizeof(T) == 2 ? 4 : 8;
  const T* row;
  int vocab, steps, first, vec;
  uint4* held;                                 // this lane's 16 bytes of step 0 in shared memory; a step is WORDS / 4 pieces of 512 lanes

  __device__ __forceinline__ int index(int step) const { return first + step * SM_STEP + (threadIdx.x & 31) * 8; }
  __device__ __forceinline__ void fetch(int step, unsigned (&w)[WORDS]) const {
    const int i = index(step);
    if (vec && i + 8 <= vocab) {
#pragma unroll
      for (int j = 0; j < WORDS; j += 4) {
        const uint4 r = reinterpret_cast<const uint4*>(row + i)[j / 4];
        w[j] = r.x; w[j + 1] = r.y; w[j + 2] = r.z; w[j + 3] = r.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = i + j < vocab ? (float)row[i + j] : -INFINITY;
        if (sizeof(T) == 4) w[j % WORDS] = __float_as_uint(x);
        else w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | (__float_as_uint(x) & 0xffff0000u) : __float_as_uint(x) >> 16;
      }
    }
  }
  __device__ __forceinline__ void hold() {
    if (HELD) {
      for (int st = 0; st < steps; ++st) {
        const int i = index(st);
        if (vec && i + 8 <= vocab) {
#pragma unroll
          for (int j = 0; j < WORDS / 4; ++j)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + (st * (WORDS / 4) + j) * SM_THREADS)), "l"(reinterpret_cast<const uint4*>(row + i) + j) : "memory");
        } else {
          unsigned w[WORDS];
          fetch(st, w);
#pragma unroll
          for (int j = 0; j < WORDS / 4; ++j) held[(st * (WORDS / 4) + j) * SM_THREADS] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  }
  __device__ __forceinline__ void words(int step, unsigned (&w)[WORDS]) const {
    if (HELD) {                                // a lane reads what it has written
#pragma unroll
      for (int j = 0; j < WORDS / 4; ++j) {
        const uint4 r = held[(step * (WORDS / 4) + j) * SM_THREADS];
        w[4 * j] = r.x; w[4 * j + 1] = r.y; w[4 * j + 2] = r.z; w[4 * j + 3] = r.w;
      }
    } else {
      fetch(step, w);
    }
  }
  __device__ __forceinline__ void values(int step, float (&x)[8]) const {
    unsigned w[WORDS];
    words(step, w);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = __uint_as_float(sizeof(T) == 4 ? w[j % WORDS] : j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int st = 0; st < steps; ++st) f(st);
  }
};

struct SampleSplit { unsigned bin; u64 cnt, w, target; };   // the deciding bin (SM_BINS: none), what lies above it, what was looked for

// First bin at which the cluster's running count (by_weight: weight) reaches `target`, or all there is where that is less (all_there).
__device__ __forceinline__ SampleSplit sm_find(cg::cluster_group& cl, SampleSmem& s, int C, bool by_weight, bool weights, u64 target, bool all_there, unsigned* in_bin) {
  constexpr int PER = SM_BINS / SM_THREADS;
  const int b0 = threadIdx.x * PER;
  unsigned c[PER];
  u64 w[PER], sum_c = 0, sum_w = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) { c[j] = 0; w[j] = 0; }
  for (int r = 0; r < C; ++r) {
    const uint4 x = *reinterpret_cast<const uint4*>(cl.map_shared_rank(s.cnt, r) + b0);
    c[0] += x.x; c[1] += x.y; c[2] += x.z; c[3] += x.w;
    if (weights) {
      const uint4 lo = *reinterpret_cast<const uint4*>(cl.map_shared_rank(s.lo, r) + b0), hi = *reinterpret_cast<const uint4*>(cl.map_shared_rank(s.hi, r) + b0);
      w[0] += (u64)hi.x << 32 | lo.x; w[1] += (u64)hi.y << 32 | lo.y; w[2] += (u64)hi.z << 32 | lo.z; w[3] += (u64)hi.w << 32 | lo.w;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) { sum_c += c[j]; sum_w += w[j]; }
  u64 all;
  u64 before_c = sm_block_scan(sum_c, s, &all), before_w = 0;
  if (all_there && !by_weight) target = min(target, all);
  if (weights) before_w = sm_block_scan(sum_w, s, &all);
  if (threadIdx.x == 0) s.res[0] = SM_BINS;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const u64 b = by_weight ? before_w : before_c, a = by_weight ? w[j] : c[j];
    if (a > 0 && b < target && b + a >= target) {
      s.res[0] = b0 + j;
      s.res[1] = before_c;
      s.res[2] = before_w;
      s.res[3] = c[j];
    }
    before_c += c[j];
    before_w += w[j];
  }
  __syncthreads();
  SampleSplit out;
  out.bin = (unsigned)s.res[0];
  out.cnt = s.res[1];
  out.w = s.res[2];
  out.target = target;
  *in_bin = (unsigned)s.res[3];
  return out;
}
static_assert(SM_BINS == 4 * SM_THREADS, "four bins a thread");

// One weight into a bin: 64 bits from two native 32-bit atomics, whatever their order.
__device__ __forceinline__ void sm_add(SampleSmem& s, int b, u64 w) {
  const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32);
  const unsigned old = atomicAdd(&s.lo[b], lo);
  const unsigned up = hi + (old + lo < old ? 1u : 0u);
  if (up) atomicAdd(&s.hi[b], up);
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(SM_THREADS, 2) sample_rows_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t sm_raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(sm_raw);
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  cl.barrier_arrive();                         // no CTA of the cluster is written to before it runs
  if (tid < 32) s.exp2[tid] = c_exp2[tid];
  if (tid == 0) s.n_list = s.n_local = 0;
  for (int i = tid; i < SM_BINS; i += SM_THREADS) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
  pdl_wait();
  const int r = blockIdx.x / C;
  SampleRow<T, HELD> row;
  row.row = reinterpret_cast<const T*>(p.logits) + (long long)r * p.ld;
  row.vocab = p.vocab;
  row.first = (rank * SM_WARPS + warp) * p.steps * SM_STEP;
  row.steps = max(0, min(p.steps, (p.vocab - row.first + SM_STEP - 1) / SM_STEP));
  row.vec = p.vec;
  row.held = s.held + tid;
  row.hold();
  const float temp = p.temperature[r], top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f, u = p.u[r];
  const int top_k = p.top_k ? p.top_k[r] : 0;
  const bool greedy = !(temp > 0.f) || min_p > 1.f;          // the first token of the order alone

  // ---- (1) the largest logit, with its first index where that is the answer, and a mean
  float best = -INFINITY, sum = 0.f;
  int best_st = 0, n_sum = 0;
  row.each([&](int st) {
    unsigned w[SampleRow<T, HELD>::WORDS];
    row.words(st, w);
    float v;
    if (sizeof(T) == 2) {
      __nv_bfloat162 h = __hmax2(__hmax2(*reinterpret_cast<__nv_bfloat162*>(&w[0]), *reinterpret_cast<__nv_bfloat162*>(&w[1])),
                                 __hmax2(*reinterpret_cast<__nv_bfloat162*>(&w[2]), *reinterpret_cast<__nv_bfloat162*>(&w[3])));
      v = fmaxf(__low2float(h), __high2float(h));
    } else {
      v = __uint_as_float(w[0]);
#pragma unroll
      for (int j = 1; j < SampleRow<T, HELD>::WORDS; ++j) v = fmaxf(v, __uint_as_float(w[j]));
    }
    if (v > best) { best = v; best_st = st; }
    if (st == 0) {
      float x[8];
      row.values(st, x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x[j] > -INFINITY) { sum += x[j]; ++n_sum; }
    }
  });
  u64 top;
  if (greedy) {
    int best_i = 0x7fffffff;
    if (row.steps > 0) {
      float x[8];
      row.values(best_st, x);
#pragma unroll
      for (int j = 7; j >= 0; --j)
        if (x[j] >= best) best_i = row.index(best_st) + j;
    }
    top = (u64)sm_key(best) << 32 | (unsigned)~best_i;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 t = __shfl_xor_sync(0xffffffffu, top, o);
      top = t > top ? t : top;
    }
  } else {
    top = (u64)__reduce_max_sync(0xffffffffu, sm_key(best)) << 32;
    n_sum = __reduce_add_sync(0xffffffffu, n_sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane == 0) { s.list[warp] = top; s.list[SM_WARPS + warp] = (u64)__float_as_uint(sum) << 32 | (unsigned)n_sum; }
  __syncthreads();
  cl.barrier_wait();
  if (tid < C) {                               // thread i tells CTA i
    u64 t = 0;
    float f = 0.f;
    unsigned n = 0;
    for (int i = 0; i < SM_WARPS; ++i) {
      t = max(t, s.list[i]);
      f += __uint_as_float((unsigned)(s.list[SM_WARPS + i] >> 32));
      n += (unsigned)s.list[SM_WARPS + i];
    }
    u64* to = cl.map_shared_rank(&s.slot[0][0][0], tid);
    to[rank] = t;
    to[SM_CLUSTER + rank] = (u64)__float_as_uint(f) << 32 | n;
  }
  cl.sync();
  float mean = 0.f, n_mean = 0.f;
  top = 0;
  for (int i = 0; i < C; ++i) {
    top = max(top, s.slot[0][0][i]);
    mean += __uint_as_float((unsigned)(s.slot[0][1][i] >> 32));
    n_mean += (float)(unsigned)s.slot[0][1][i];
  }
  const float m = sm_value((unsigned)(top >> 32));
  if (m == -INFINITY || greedy) {
    if (rank == 0 && tid == 0) {
      p.tokens[r] = m == -INFINITY ? 0 : (long long)(unsigned)~(unsigned)top;
      if (p.logprobs) p.logprobs[r] = m == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  mean = __fdiv_rn(mean, n_mean);
  SampleWeight weight;
  const double scale = 1.4426950408889634074 / (double)temp;
  weight.m = m;
  weight.ch = (float)scale;
  weight.cl = isinf(weight.ch) ? 0.f : (float)(scale - (double)weight.ch);
  weight.table = s.exp2;
  auto finish = [&](long long token, u64 total) {           // one thread of the row
    p.tokens[r] = token;
    if (p.logprobs) {
      const float x = (float)row.row[token];
      const double lw = x == m ? 0. : ((double)x - (double)m) / (double)temp;
      p.logprobs[r] = (float)(lw - log((double)total * (1. / (double)(1ull << SM_ONE))));
    }
  };
  // the lowest logit that min_p keeps: x >= m + T ln(min_p)
  float least = -INFINITY;
  if (min_p > 0.f) least = fminf(m, __double2float_ru((double)m + (double)temp * log((double)min_p)));
  const bool need_k = top_k > 0 && top_k < p.vocab, need_p = top_p < 1.f;
  float last_x = -INFINITY;                                 // logits above this are kept, of equal ones those up to index last_i
  int last_i = 0x7fffffff;

  int ex = 1;                                               // exchanges so far
  auto exchange_sum = [&](u64 v) {                          // of one value of every CTA: the sum, and that of the ranks below
    if (tid < C) cl.map_shared_rank(&s.slot[ex][0][0], tid)[rank] = v;
    cl.sync();
    u64 all = 0, below = 0;
    for (int i = 0; i < C; ++i) {
      all += s.slot[ex][0][i];
      below += i < rank ? s.slot[ex][0][i] : 0;
    }
    ++ex;
    return make_ulonglong2(all, below);
  };
  // ---- (4) the first index at which the running sum of value(logit, index) reaches target(total): found(index, total) in one thread
  auto locate = [&](auto value, auto target, auto found) {
    row.each([&](int st) {
      float x[8];
      row.values(st, x);
      const int i = row.index(st);
      u64 v = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) v += value(x[j], i + j);
      v = sm_warp_sum(v);
      if (lane == 0) s.step[warp * p.steps + st] = v;
    });
    for (int st = row.steps + lane; st < p.steps; st += 32) s.step[warp * p.steps + st] = 0;
    __syncthreads();
    // every warp over all of them: a run of entries per lane
    const int n = SM_WARPS * p.steps, chunk = (n + 31) / 32;
    u64 v = 0;
    for (int i = lane * chunk; i < min(n, (lane + 1) * chunk); ++i) v += s.step[i];
    u64 end = sm_warp_scan(v), begin = end - v;
    const u64 here = __shfl_sync(0xffffffffu, end, 31);
    const ulonglong2 a = exchange_sum(here);
    const u64 t = target(a.x);
    if (t <= a.y || t > a.y + here) return;                 // another CTA's
    begin += a.y;
    end += a.y;
    const int owner = __ffs(__ballot_sync(0xffffffffu, begin < t && end >= t)) - 1;
    int at = -1;
    if (lane == owner)
      for (int i = lane * chunk; at < 0; ++i) {
        if (begin + s.step[i] >= t) at = i;
        else begin += s.step[i];
      }
    at = __shfl_sync(0xffffffffu, at, owner);
    begin = __shfl_sync(0xffffffffu, begin, owner);
    if (at / p.steps != warp) return;
    const int step = at - warp * p.steps;
    float x[8];
    row.values(step, x);
    const int i = row.index(step);
    u64 e[8];
    v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { e[j] = value(x[j], i + j); v += e[j]; }
    const u64 to = begin + sm_warp_scan(v);
    u64 from = to - v;
    if (from < t && to >= t) {
      int j = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        from += e[q];
        if (from < t) j = q + 1;
      }
      found(i + j, a.x);
    }
  };

  if (need_k || need_p) {
    // ---- (2) bins of equal width from the largest logit down; p alone may reach below the mean
    float per = __fdiv_rn((float)(SM_BINS - 1), (m - mean) * (need_k ? 1.f : 1.5f));
    if (!(per > 0.f && per < 3e38f)) per = 0.f;
    auto bin_of = [&](float x) {                            // NaN, -inf and what is below: the last one, in which nothing is counted
      const float f = __fmul_rn(__fsub_rn(m, x), per);
      return x > -INFINITY && f < (float)(SM_BINS - 1) ? (int)f : SM_BINS - 1;
    };
    u64 w_here = 0;
    row.each([&](int st) {
      float x[8];
      row.values(st, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int b = bin_of(x[j]);
        if (b < SM_BINS - 1) atomicAdd(&s.cnt[b], 1u);
        if (!need_k) {
          const u64 w = weight(x[j]);
          if (b < SM_BINS - 1) sm_add(s, b, w);
          w_here += w;
        }
      }
    });
    u64 w_all = 0;
    if (!need_k) {
      u64 t;
      sm_block_scan(w_here, s, &t);
      w_all = exchange_sum(t).x;
    } else {
      cl.sync();
    }
    unsigned in_bin;
    const u64 target_p = need_k ? ~0ull : max(1ull, sm_reach(top_p, w_all));
    const SampleSplit sp = sm_find(cl, s, C, !need_k, !need_k, need_k ? (u64)top_k : target_p, false, &in_bin);
    const bool whole = sp.cnt + in_bin <= SM_LIST;          // every candidate fits the list, not just the deciding bin
    if (sp.bin < SM_BINS && (whole || (!need_k && in_bin <= SM_LIST))) {
      // ---- (3) the list: gathered here, then in rank 0
      if (!need_k) cl.sync();                  // the others have read the weights, whose place it takes
      row.each([&](int st) {
        float x[8];
        row.values(st, x);
        const int i = row.index(st);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int b = bin_of(x[j]);
          if (whole ? b <= (int)sp.bin : b == (int)sp.bin) s.local[atomicAdd(&s.n_local, 1)] = sm_entry(x[j], i + j);
        }
      });
      __syncthreads();
      if (tid == 0) s.base = atomicAdd(cl.map_shared_rank(&s.n_list, 0), s.n_local);
      __syncthreads();
      u64* to = cl.map_shared_rank(s.list, 0) + s.base;
      for (int i = tid; i < s.n_local; i += SM_THREADS) to[i] = s.local[i];
      cl.sync();
      if (rank != 0 && whole) return;
      if (rank == 0) {
        const int n = (int)(whole ? sp.cnt + in_bin : in_bin), n_k = need_k ? top_k : n;
        const u64 above = whole ? 0 : sp.w;    // weights that are kept and not in the list
        auto last_one = [&](u64 e) {           // one thread: the last token that p keeps, to every CTA
          for (int q = 0; q < C; ++q) cl.map_shared_rank(&s.slot[5][0][0], q)[0] = e;
        };
        if (n <= SM_THREADS) {
          // a token per thread: what comes before it is counted and summed directly
          u64 mine = ~0ull, w = 0, before = above;
          int ahead = 0;
          if (tid < n) {
            mine = s.list[tid];
            w = weight(sm_entry_value(mine));
            s.pair[tid] = make_ulonglong2(mine, w);
          }
          __syncthreads();
          if (tid < n)
            for (int j = 0; j < n; ++j) {
              const ulonglong2 o = s.pair[j];
              if (o.x < mine) { ++ahead; before += o.y; }
            }
          u64 target = target_p;
          if (need_k && need_p) {
            u64 all;
            sm_block_scan(tid < n && ahead < n_k ? w : 0ull, s, &all);
            target = sm_reach(top_p, all);
          }
          if (!whole) {
            if (tid < n && before < target && before + w >= target) last_one(mine);
          } else {
            // kept: what begins below the target, is among the first k and not below min_p; the first token always
            const bool in = tid < n && ahead < n_k && (ahead == 0 || ((!need_p || before < target) && sm_entry_value(mine) >= least));
            __syncthreads();
            if (tid < n) s.pair[tid] = make_ulonglong2(mine, in ? w : 0ull);
            __syncthreads();
            if (in) {
              u64 all = 0;
              before = 0;
              for (int j = 0; j < n; ++j) {
                const ulonglong2 o = s.pair[j];
                all += o.y;
                before += (unsigned)o.x < (unsigned)mine ? o.y : 0;
              }
              const u64 t = sm_above(u, all);
              if (before < t && before + w >= t) finish((long long)(unsigned)mine, all);
            }
            return;
          }
        } else {
          int pow2 = 2;
          while (pow2 < n) pow2 <<= 1;
          for (int i = n + tid; i < pow2; i += SM_THREADS) s.list[i] = ~0ull;
          sm_sort(s.list, pow2);
          constexpr int PER = SM_LIST / SM_THREADS;
          const int each = pow2 / SM_THREADS;
          u64 w[PER], mine = 0, all;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const int i = tid * each + j;
            w[j] = j < each && i < n && i < n_k ? weight(sm_entry_value(s.list[i])) : 0ull;
            mine += w[j];
          }
          u64 before = above + sm_block_scan(mine, s, &all);
          const u64 target = need_k && need_p ? sm_reach(top_p, all) : target_p;
          u64 kept = 0;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const int i = tid * each + j;
            const bool there = j < each && i < n && i < n_k;
            if (!whole && there && before < target && before + w[j] >= target) last_one(s.list[i]);
            if (there && (i == 0 || ((!need_p || before < target) && sm_entry_value(s.list[i]) >= least))) ++kept;
            before += w[j];
          }
          if (whole) {
            u64 n_kept;
            sm_block_scan(kept, s, &n_kept);
            const int nk = (int)n_kept;
            int pow2k = 2;                     // the same by index
            while (pow2k < nk) pow2k <<= 1;
            for (int i = tid; i < pow2k; i += SM_THREADS) {
              const u64 e = s.list[i];
              s.local[i] = i < nk ? e << 32 | e >> 32 : ~0ull;
            }
            sm_sort(s.local, pow2k);
            const int each_k = (pow2k + SM_THREADS - 1) / SM_THREADS;
            mine = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const int i = tid * each_k + j;
              w[j] = j < each_k && i < nk ? weight(sm_value(~(unsigned)s.local[i])) : 0ull;
              mine += w[j];
            }
            before = sm_block_scan(mine, s, &all);
            const u64 t = sm_above(u, all);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              if (before < t && before + w[j] >= t) finish((long long)(s.local[tid * each_k + j] >> 32), all);
              before += w[j];
            }
            return;
          }
        }
      }
      cl.sync();
      const u64 e = s.slot[5][0][0];
      last_x = sm_entry_value(e);
      last_i = (int)(unsigned)e;
    } else {
      // ---- the deciding value by digits of its key, over the row
      auto decide = [&](bool by_weight, u64 target, u64* n_class, u64* n_above, u64* w_above) {
        unsigned prefix = 0;
        *n_above = *w_above = 0;
        int done = 0;
        for (int level = 0; level < 3; ++level) {
          const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
          cl.sync();                           // the others have read the bins
          for (int i = tid; i < SM_BINS; i += SM_THREADS) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
          __syncthreads();
          row.each([&](int st) {
            float x[8];
            row.values(st, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const unsigned key = sm_key(x[j]);
              if (!(x[j] > -INFINITY) || (done > 0 && key >> (32 - done) != prefix)) continue;
              const int b = (1 << bits) - 1 - (int)((key >> shift) & ((1u << bits) - 1));
              atomicAdd(&s.cnt[b], 1u);
              if (need_p) sm_add(s, b, weight(x[j]));
            }
          });
          cl.sync();
          unsigned in_class;
          const SampleSplit d = sm_find(cl, s, C, by_weight, need_p, target, level == 0, &in_class);
          prefix = prefix << bits | ((1u << bits) - 1 - d.bin);
          done += bits;
          target = d.target - (by_weight ? d.w : d.cnt);
          *n_above += d.cnt;
          *w_above += d.w;
          *n_class = in_class;
        }
        cl.sync();                             // the others have read the counts, whose place the sums take
        return prefix;
      };
      u64 n_class, n_above, w_above, n_take = 0, w_total = w_all;
      unsigned key = 0;
      if (need_k) {
        key = decide(false, (u64)top_k, &n_class, &n_above, &w_above);
        n_take = min((u64)top_k - n_above, n_class);
        w_total = w_above + n_take * weight(sm_value(key));
      }
      if (need_p) {
        const u64 target = max(1ull, sm_reach(top_p, w_total));
        u64 c, na, wa;
        const unsigned k2 = decide(true, target, &c, &na, &wa);
        const u64 w1 = weight(sm_value(k2));
        u64 take = w1 > 0 ? (target - wa + w1 - 1) / w1 : 1;
        if (need_k && k2 == key) take = min(take, n_take);
        key = k2;
        n_take = take;
        n_class = c;
      }
      last_x = sm_value(key);
      if (n_take < n_class) {                  // some of the tokens with this logit: those of the lowest indices
        locate([&](float x, int) { return x == last_x ? 1ull : 0ull; }, [&](u64) { return n_take; },
               [&](int i, u64) {
                 for (int q = 0; q < C; ++q) cl.map_shared_rank(&s.slot[5][0][0], q)[0] = (u64)i;
               });
        cl.sync();
        last_i = (int)s.slot[5][0][0];
      }
    }
  }
  if (least > last_x) {
    last_x = least;
    last_i = 0x7fffffff;
  }
  locate([&](float x, int i) { return x > last_x || (x == last_x && i <= last_i) ? weight(x) : 0ull; }, [&](u64 total) { return sm_above(u, total); },
         [&](int i, u64 total) { finish(i, total); });
}

}  // namespace mlf

using namespace mlf;

// CTAs per row: as many as keep the row in shared memory, and beyond that as bring the launch to two on every SM, up to SM_CLUSTER,
// none of them with less than 4096 logits.
static int sample_cluster(long long rows, int vocab) {
  int c = 1;
  while (c < SM_CLUSTER && (vocab > c * SM_WARPS * SM_STEP * SM_HELD || (rows * c < 2 * sm_count() && vocab > c * 4096))) c *= 2;
  return c;
}

// logits [rows, vocab] (pitch ld), bf16 or fp32 (is_fp32); u and temperature [rows]; top_k, top_p, min_p [rows] or null (no limit);
// tokens [rows] int64; logprobs [rows] or null: the logarithm of the token's probability among the kept ones.
MLF_API int mlf_sample_rows(const void* logits, int is_fp32, long long rows, long long ld, int vocab, const float* u, const float* temperature,
                            const int* top_k, const float* top_p, const float* min_p, long long* tokens, float* logprobs, uint64_t stream) {
  if (rows <= 0) return 0;
  MLF_REQUIRE(vocab > 0 && vocab <= SM_CLUSTER * SM_WARPS * SM_STEP * SM_STEPS, "sample_rows: vocabulary of %d (1 to %d)", vocab,
              SM_CLUSTER * SM_WARPS * SM_STEP * SM_STEPS);
  const int C = sample_cluster(rows, vocab);
  MLF_REQUIRE(rows <= (1LL << 31) / SM_CLUSTER - 1, "sample_rows: %lld rows", rows);
  SampleParams p;
  p.logits = logits; p.ld = ld; p.rows = (int)rows; p.vocab = vocab;
  p.steps = (vocab + C * SM_WARPS * SM_STEP - 1) / (C * SM_WARPS * SM_STEP);
  p.vec = (ld * (is_fp32 ? 4 : 2)) % 16 == 0 && (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
  p.u = u; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.tokens = tokens; p.logprobs = logprobs;
  const bool held = p.steps <= SM_HELD;
  const auto kernel = is_fp32 ? (held ? sample_rows_kernel<float, true> : sample_rows_kernel<float, false>)
                              : (held ? sample_rows_kernel<__nv_bfloat16, true> : sample_rows_kernel<__nv_bfloat16, false>);
  // shared memory for the most steps that are held: one size for every launch of a kernel
  const size_t smem = sizeof(SampleSmem) + (held ? (size_t)SM_HELD * SM_THREADS * 8 * (is_fp32 ? 4 : 2) : 0);
  static bool attr_set[64][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  bool& set = attr_set[dev & 63][(is_fp32 ? 2 : 0) + (held ? 1 : 0)];
  if (!set) {
    MLF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    set = true;
  }
  MLF_CHECK_CUDA(launch_pdl_cluster(kernel, dim3((unsigned)(rows * C)), dim3(SM_THREADS), smem, (unsigned)C,
                                    reinterpret_cast<cudaStream_t>(stream), p));
  count_launch();
  return 0;
}
