// The next tokens from logits and given random numbers: temperature, top-k, top-p and min-p of each row.
//
// With m the largest logit, T the temperature and w_i = exp((x_i - m) / T), in the order of x (the larger first, of equal ones the
// lower index): the first k tokens are kept; of these the shortest prefix whose weights reach top_p of theirs; of these the
// tokens with w_i >= min_p; the first one in any case. The token is the first one, by index, at which the running sum of the kept weights is above
// u times their total. T = 0: the largest logit, of equal ones the lowest index. NaN counts as -inf.
//
// Weights are integers, w_i rounded to 2^-40, from an exponential that is good to about 2^-30: x - m and the product with
// log2(e) / T are carried in two floats, 2^(j/32) comes from a table and the rest from a polynomial. Sums of integers do not depend on
// their order, so that a row gives the same token in any batch and with any number of CTAs, and a border between
// two tokens is as sharp as the weights themselves.
//
// A cluster of CTAs takes a row; a pass over its logits, which the caches hold after the first one, is followed by an
// exchange through distributed shared memory. (1) largest logit and mean. (2) Where k or p limits the row: counts (and
// weights, for p alone) in bins of equal width between the largest logit and the mean, which spread the atomics of a few thousand
// candidates over as many addresses. (3) The bins down to the one that decides hold few tokens as a rule: these go to a list in one
// CTA, are sorted there and decided and drawn from. Otherwise the deciding value is found digit by digit over the row,
// 11 + 11 + 10 bits of the order-preserving integer of a float, and (4) the token from sums of 256 neighbours.
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
constexpr int SM_STEPS = 64;                   // at most, per warp
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 2048;
constexpr int SM_CLUSTER = 8;                  // CTAs per row, at most
constexpr int SM_ONE = 40;                     // log2 of the weight of the largest logit
constexpr unsigned SM_ABSENT = 0x007fffffu;    // key of -inf: a token that cannot be drawn

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
  u64 w[SM_BINS];
  u64 step[SM_WARPS * SM_STEPS];
  u64 slot[6][4][SM_CLUSTER];                  // one set per exchange of a launch: values of every CTA
  u64 warp[SM_WARPS + 1];
  u64 res[4];
  alignas(16) unsigned cnt[SM_BINS];
  unsigned exp2[32];
  int n_list, base;
  int n_local;
};

// Order-preserving integer of a float; -0 is 0 and NaN is -inf.
__device__ __forceinline__ unsigned sm_key(float x) {
  unsigned u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sm_value(unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

struct SampleWeight {
  float m, ch, cl;                             // log2(e) / T in two floats
  const unsigned* table;
  __device__ __forceinline__ u64 operator()(unsigned key) const {
    const float x = sm_value(key);
    if (x == m) return 1ull << SM_ONE;
    if (key <= SM_ABSENT) return 0ull;
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

template <typename T>
struct SampleRow {
  const T* row;
  int vocab, steps, first, vec;                // first: of this warp's run
  // logits first + step * 256 + lane * 8 .. + 7 as keys; what lies behind the vocabulary is absent
  __device__ __forceinline__ int load(int step, unsigned (&key)[8]) const {
    const int i = first + step * SM_STEP + (threadIdx.x & 31) * 8;
    if (vec && i + 8 <= vocab) {
      if (sizeof(T) == 2) {
        const uint4 r = *reinterpret_cast<const uint4*>(row + i);
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          key[2 * j] = sm_key(__uint_as_float(w[j] << 16));
          key[2 * j + 1] = sm_key(__uint_as_float(w[j] & 0xffff0000u));
        }
      } else {
        const float4 a = *reinterpret_cast<const float4*>(row + i), b = *reinterpret_cast<const float4*>(row + i + 4);
        const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) key[j] = sm_key(f[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) key[j] = i + j < vocab ? sm_key((float)row[i + j]) : SM_ABSENT;
    }
    return i;
  }
};

struct SampleSplit { unsigned bin; u64 cnt, w; };   // the deciding bin and what lies above it; bin SM_BINS: none

// First bin at which the cluster's running count (by_weight: weight) reaches `target`.
__device__ __forceinline__ SampleSplit sm_find(cg::cluster_group& cl, SampleSmem& s, int C, bool by_weight, bool weights, u64 target, unsigned* in_bin) {
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
      const ulonglong2* p = reinterpret_cast<const ulonglong2*>(cl.map_shared_rank(s.w, r) + b0);
      const ulonglong2 a = p[0], b = p[1];
      w[0] += a.x; w[1] += a.y; w[2] += b.x; w[3] += b.y;
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) { sum_c += c[j]; sum_w += w[j]; }
  u64 all;
  u64 before_c = sm_block_scan(sum_c, s, &all), before_w = 0;
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
  *in_bin = (unsigned)s.res[3];
  return out;
}
static_assert(SM_BINS == 4 * SM_THREADS, "four bins a thread");

template <typename T>
__global__ void __launch_bounds__(SM_THREADS) sample_rows_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t sm_raw[];
  SampleSmem& s = *reinterpret_cast<SampleSmem*>(sm_raw);
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  cl.barrier_arrive();                         // no CTA of the cluster is written to before it runs
  if (tid < 32) s.exp2[tid] = c_exp2[tid];
  if (tid == 0) s.n_list = s.n_local = 0;
  for (int i = tid; i < SM_BINS; i += SM_THREADS) { s.cnt[i] = 0; s.w[i] = 0; }
  pdl_wait();
  const int r = blockIdx.x / C;
  SampleRow<T> row;
  row.row = reinterpret_cast<const T*>(p.logits) + (long long)r * p.ld;
  row.vocab = p.vocab;
  row.steps = p.steps;
  row.first = (rank * SM_WARPS + warp) * p.steps * SM_STEP;
  row.vec = p.vec;
  const int steps = max(0, min(p.steps, (p.vocab - row.first + SM_STEP - 1) / SM_STEP));
  const float temp = p.temperature[r], top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f, u = p.u[r];
  const int top_k = p.top_k ? p.top_k[r] : 0;

  // ---- (1) the largest logit, its first index, how many can be drawn and the mean of the finite ones
  unsigned best = 0, n_here = 0;
  int best_i = 0x7fffffff;
  float sum = 0.f;
  for (int st = 0; st < steps; ++st) {
    unsigned key[8];
    const int i = row.load(st, key);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (key[j] > best) { best = key[j]; best_i = i + j; }
      const bool there = key[j] > SM_ABSENT;
      n_here += there ? 1 : 0;
      sum += there ? sm_value(key[j]) : 0.f;
    }
  }
  u64 top = (u64)best << 32 | (unsigned)~best_i;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 t = __shfl_xor_sync(0xffffffffu, top, o);
    top = t > top ? t : top;
    n_here += __shfl_xor_sync(0xffffffffu, n_here, o);
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane == 0) { s.step[warp] = top; s.step[SM_WARPS + warp] = n_here; s.step[2 * SM_WARPS + warp] = __float_as_uint(sum); }
  __syncthreads();
  cl.barrier_wait();
  if (tid < C) {                               // thread i tells CTA i
    u64 t = 0, n = 0;
    float f = 0.f;
    for (int i = 0; i < SM_WARPS; ++i) {
      t = max(t, s.step[i]);
      n += s.step[SM_WARPS + i];
      f += __uint_as_float((unsigned)s.step[2 * SM_WARPS + i]);
    }
    u64* to = cl.map_shared_rank(&s.slot[0][0][0], tid);
    to[rank] = t;
    to[SM_CLUSTER + rank] = n;
    to[2 * SM_CLUSTER + rank] = __float_as_uint(f);
  }
  cl.sync();
  u64 n_row = 0;
  float mean = 0.f;
  top = 0;
  for (int i = 0; i < C; ++i) {
    top = max(top, s.slot[0][0][i]);
    n_row += s.slot[0][1][i];
    mean += __uint_as_float((unsigned)s.slot[0][2][i]);
  }
  const unsigned top_key = (unsigned)(top >> 32);
  const bool none = top_key <= SM_ABSENT;
  if (none || !(temp > 0.f) || min_p > 1.f) {  // the first token of the order alone
    if (rank == 0 && tid == 0) {
      p.tokens[r] = none ? 0 : (long long)(unsigned)~(unsigned)top;
      if (p.logprobs) p.logprobs[r] = none ? -INFINITY : 0.f;
    }
    return;
  }
  mean /= (float)n_row;
  const float m = sm_value(top_key);
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
      p.logprobs[r] = (float)(lw - log((double)total * exp2(-(double)SM_ONE)));
    }
  };
  unsigned least = SM_ABSENT + 1;                           // lowest key that min_p keeps: x >= m + T ln(min_p)
  if (min_p > 0.f) least = max(least, sm_key(__double2float_ru((double)m + (double)temp * log((double)min_p))));
  least = min(least, top_key);
  const bool need_k = top_k > 0 && (u64)top_k < n_row, need_p = top_p < 1.f;
  unsigned last_key = SM_ABSENT + 1;                        // keys above this are kept, of equal ones those up to last_i
  int last_i = 0x7fffffff;

  int ex = 1;                                               // exchanges so far
  auto exchange_sum = [&](u64 v) {                          // of one value of every CTA: their sum, and that of the ranks below in s.res[0]
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
  // ---- (4) the first index at which the running sum of value(key, index) reaches target(total); calls found(index, total) in one thread
  auto locate = [&](auto value, auto target, auto found) {
    for (int st = 0; st < steps; ++st) {
      unsigned key[8];
      const int i = row.load(st, key);
      u64 v = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) v += value(key[j], i + j);
      v = sm_warp_sum(v);
      if (lane == 0) s.step[warp * p.steps + st] = v;
    }
    for (int st = steps + lane; st < p.steps; st += 32) s.step[warp * p.steps + st] = 0;
    __syncthreads();
    const int n = SM_WARPS * p.steps;
    u64 mine = 0;
    for (int i = tid; i < n; i += SM_THREADS) mine += s.step[i];
    u64 here;
    sm_block_scan(mine, s, &here);
    const ulonglong2 a = exchange_sum(here);
    const u64 t = target(a.x);
    if (warp == 0 && t > a.y && t <= a.y + here) {
      const int chunk = (n + 31) / 32;
      u64 v = 0;
      for (int i = lane * chunk; i < min(n, (lane + 1) * chunk); ++i) v += s.step[i];
      u64 end = a.y + sm_warp_scan(v), begin = end - v;
      const int owner = __ffs(__ballot_sync(0xffffffffu, begin < t && end >= t)) - 1;
      int at = -1;
      if (lane == owner)
        for (int i = lane * chunk; at < 0; ++i) {
          if (begin + s.step[i] >= t) at = i;
          else begin += s.step[i];
        }
      at = __shfl_sync(0xffffffffu, at, owner);
      begin = __shfl_sync(0xffffffffu, begin, owner);
      SampleRow<T> run = row;
      run.first = (rank * SM_WARPS + at / p.steps) * p.steps * SM_STEP;
      unsigned key[8];
      const int i = run.load(at % p.steps, key);
      u64 e[8];
      v = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) { e[j] = value(key[j], i + j); v += e[j]; }
      end = begin + sm_warp_scan(v);
      begin = end - v;
      if (begin < t && end >= t) {
        int j = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          begin += e[q];
          if (begin < t) j = q + 1;
        }
        found(i + j, a.x);
      }
    }
  };

  if (need_k || need_p) {
    // ---- (2) bins of equal width from the largest logit down to the mean; what is below it is counted in none
    float per = (float)(SM_BINS - 1) / (m - mean);
    if (!(per > 0.f && per < 3e38f)) per = 0.f;
    auto bin_of = [&](unsigned key) {
      const float f = __fmul_rn(__fsub_rn(m, sm_value(key)), per);
      return f < (float)(SM_BINS - 1) ? (int)f : (f == f ? SM_BINS - 1 : 0);
    };
    u64 w_here = 0;
    for (int st = 0; st < steps; ++st) {
      unsigned key[8];
      row.load(st, key);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (key[j] <= SM_ABSENT) continue;
        const int b = bin_of(key[j]);
        if (b < SM_BINS - 1) atomicAdd(&s.cnt[b], 1u);
        if (!need_k) {
          const u64 w = weight(key[j]);
          if (b < SM_BINS - 1) atomicAdd(&s.w[b], w);
          w_here += w;
        }
      }
    }
    u64 w_all = 0;
    if (!need_k) {
      u64 t;
      sm_block_scan(w_here, s, &t);
      w_all = exchange_sum(t).x;
    } else {
      cl.sync();
    }
    unsigned in_bin;
    const SampleSplit sp = sm_find(cl, s, C, !need_k, !need_k, need_k ? (u64)top_k : max(1ull, sm_reach(top_p, w_all)), &in_bin);
    const u64 n_list = sp.cnt + in_bin;
    if (sp.bin < SM_BINS && n_list <= SM_LIST) {
      // ---- (3) the list: gathered here, then in rank 0
      if (!need_k) cl.sync();                  // the others have read the weights, whose place it takes
      for (int st = 0; st < steps; ++st) {
        unsigned key[8];
        const int i = row.load(st, key);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key[j] > SM_ABSENT && bin_of(key[j]) <= (int)sp.bin) s.w[atomicAdd(&s.n_local, 1)] = (u64)(~key[j]) << 32 | (unsigned)(i + j);
      }
      __syncthreads();
      if (tid == 0) s.base = atomicAdd(cl.map_shared_rank(&s.n_list, 0), s.n_local);
      __syncthreads();
      u64* to = cl.map_shared_rank(s.list, 0) + s.base;
      for (int i = tid; i < s.n_local; i += SM_THREADS) to[i] = s.w[i];
      cl.sync();
      if (rank != 0) return;
      const int n = (int)n_list;
      int pow2 = 2;
      while (pow2 < n) pow2 <<= 1;
      for (int i = n + tid; i < pow2; i += SM_THREADS) s.list[i] = ~0ull;
      sm_sort(s.list, pow2);                   // the larger logit first, of equal ones the lower index
      constexpr int PER = SM_LIST / SM_THREADS;
      const int each = (pow2 + SM_THREADS - 1) / SM_THREADS;
      const int n_k = need_k ? top_k : n;
      u64 w[PER], mine = 0, all;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = tid * each + j;
        w[j] = j < each && i < n_k ? weight(~(unsigned)(s.list[i] >> 32)) : 0ull;
        mine += w[j];
      }
      u64 before = sm_block_scan(mine, s, &all);
      const u64 target = need_p ? sm_reach(top_p, need_k ? all : w_all) : ~0ull;
      // kept: what begins below the target, is among the first k and not below min_p; the first token always
      u64 kept = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = tid * each + j;
        const bool in = j < each && i < n_k && (i == 0 || (before < target && ~(unsigned)(s.list[i] >> 32) >= least));
        before += w[j];
        kept += in ? 1 : 0;
      }
      u64 n_kept;
      sm_block_scan(kept, s, &n_kept);
      const int nk = (int)n_kept;
      // the same by index
      int pow2k = 2;
      while (pow2k < nk) pow2k <<= 1;
      for (int i = tid; i < pow2k; i += SM_THREADS) {
        const u64 e = s.list[i];
        s.w[i] = i < nk ? e << 32 | (unsigned)~(unsigned)(e >> 32) : ~0ull;
      }
      sm_sort(s.w, pow2k);
      const int each_k = (pow2k + SM_THREADS - 1) / SM_THREADS;
      mine = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = tid * each_k + j;
        w[j] = j < each_k && i < nk ? weight((unsigned)s.w[i]) : 0ull;
        mine += w[j];
      }
      before = sm_block_scan(mine, s, &all);
      const u64 t = sm_above(u, all);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (before < t && before + w[j] >= t) finish((long long)(s.w[tid * each_k + j] >> 32), all);
        before += w[j];
      }
      return;
    }
    // ---- the deciding value by digits of its key, over the row
    auto decide = [&](bool by_weight, u64 target, u64* n_class, u64* n_above, u64* w_above) {
      unsigned prefix = 0;
      *n_above = *w_above = 0;
      int done = 0;
      for (int level = 0; level < 3; ++level) {
        const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
        cl.sync();                             // the others have read the bins
        for (int i = tid; i < SM_BINS; i += SM_THREADS) { s.cnt[i] = 0; s.w[i] = 0; }
        __syncthreads();
        for (int st = 0; st < steps; ++st) {
          unsigned key[8];
          row.load(st, key);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (key[j] <= SM_ABSENT || (done > 0 && key[j] >> (32 - done) != prefix)) continue;
            const int b = (1 << bits) - 1 - (int)((key[j] >> shift) & ((1u << bits) - 1));
            atomicAdd(&s.cnt[b], 1u);
            if (need_p) atomicAdd(&s.w[b], weight(key[j]));
          }
        }
        cl.sync();
        unsigned in_bin2;
        const SampleSplit d = sm_find(cl, s, C, by_weight, need_p, target, &in_bin2);
        prefix = prefix << bits | ((1u << bits) - 1 - d.bin);
        done += bits;
        target -= by_weight ? d.w : d.cnt;
        *n_above += d.cnt;
        *w_above += d.w;
        *n_class = in_bin2;
      }
      return prefix;
    };
    u64 n_class, n_above, w_above, n_take = 0, w_total = w_all;
    if (need_k) {
      last_key = decide(false, (u64)top_k, &n_class, &n_above, &w_above);
      n_take = (u64)top_k - n_above;
      w_total = w_above + n_take * weight(last_key);
    }
    if (need_p) {
      const u64 target = max(1ull, sm_reach(top_p, w_total));
      u64 c, na, wa;
      const unsigned k2 = decide(true, target, &c, &na, &wa);
      const u64 w1 = weight(k2);
      u64 take = w1 > 0 ? (target - wa + w1 - 1) / w1 : 1;
      if (need_k && k2 == last_key) take = min(take, n_take);
      last_key = k2;
      n_take = take;
      n_class = c;
    }
    if (n_take < n_class) {                    // some of the tokens with this logit: those of the lowest indices
      const unsigned key = last_key;
      if (tid == 0) s.res[3] = ~0ull;
      locate([&](unsigned k, int) { return k == key ? 1ull : 0ull; }, [&](u64) { return n_take; },
             [&](int i, u64) {
               for (int q = 0; q < C; ++q) cl.map_shared_rank(&s.slot[5][0][0], q)[0] = (u64)i;
             });
      cl.sync();
      last_i = (int)s.slot[5][0][0];
    }
  }
  const unsigned lk = max(last_key, least);
  const int li = least > last_key ? 0x7fffffff : last_i;
  locate([&](unsigned k, int i) { return k > lk || (k == lk && i <= li) ? weight(k) : 0ull; }, [&](u64 total) { return sm_above(u, total); },
         [&](int i, u64 total) { finish(i, total); });
}

}  // namespace mlf

using namespace mlf;

// CTAs per row: as many as bring the launch to two on every SM, up to SM_CLUSTER, none of them with less than 4096 logits.
static int sample_cluster(long long rows, int vocab) {
  int c = 1;
  while (c < SM_CLUSTER && (vocab > c * SM_WARPS * SM_STEP * SM_STEPS || (rows * c < 2 * sm_count() && vocab > c * 4096))) c *= 2;
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
  const auto kernel = is_fp32 ? sample_rows_kernel<float> : sample_rows_kernel<__nv_bfloat16>;
  static bool attr_set[64][2] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63][is_fp32 ? 1 : 0]) {
    MLF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleSmem)));
    attr_set[dev & 63][is_fp32 ? 1 : 0] = true;
  }
  MLF_CHECK_CUDA(launch_pdl_cluster(kernel, dim3((unsigned)(rows * C)), dim3(SM_THREADS), sizeof(SampleSmem), (unsigned)C,
                                    reinterpret_cast<cudaStream_t>(stream), p));
  count_launch();
  return 0;
}
