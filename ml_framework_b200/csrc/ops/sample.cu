// The next tokens from logits and given random numbers: temperature, top-k, top-p and min-p of each row.
//
// With m the largest logit, T the temperature and w_i = exp((x_i - m) / T), in the order of x (the larger first, of equal ones the
// lower index): the first k tokens are kept; of these the shortest prefix whose weights reach top_p of theirs; of these the
// tokens with w_i >= min_p; the first one in any case. The token is the first one, by index, at which the running sum of the kept
// weights is above u times their total. T < 2^-90: the largest logit, of equal ones the lowest index. T > 2^90
// counts as 2^90 (beyond either, the differences of logits that matter, or the second float of log2(e) / T, are no normal fp32 numbers).
// NaN counts as -inf, a subnormal logit as 0.
//
// Weights are integers, w_i rounded to 2^-40, from an exponential that is good to about 2^-30, 2^-28 at worst: x - m and the product with
// log2(e) / T are carried in two floats, 2^(j/32) comes from a table and the rest from a polynomial. Sums of integers do not depend on
// their order, so that a row gives the same token in any batch and with any number of CTAs. What is lost is the rounding
// of each weight, alike for equal ones: a border between two tokens lies within 2^-28 + vocab 2^-41 of the total from where the
// definition has it (2^20 logits 28 T below one large one sum to 2^-20 where the definition has 0.76 of that).
//
// A cluster of CTAs takes a row, and each lane keeps its logits in shared memory where four steps of 256 a warp are enough; rows of
// more are read again in every pass, from the caches, and their lanes' maxima of eight neighbours are kept instead. A pass costs
// its arithmetic and an exchange through distributed shared memory.
// (1) Largest logit, and mean and variance of a sample; logits further below the largest than 40 T, masked ones above all, are not in it
// and none beyond 29 T, which weigh nothing, is a candidate.
// (2) Where k limits the row, or (fp32 logits) a p under which few tokens are expected: the bins of equal width that hold the k (128)
// largest of the maxima of eight neighbours hold at least as many tokens, and hardly more. These go to a list in one CTA, where the
// token is decided: eight logits cost one comparison in both passes.
// (3) Where p alone limits it: bf16 logits are counted by their value, 16 binades of either sign, and a value's tokens have the same
// weight, so that 4096 weights give the total and the deciding value. fp32 logits under a p that keeps many: the weights of all
// of them in bins, and the deciding bin alone in the list.
// (4) Where a list is too long (many equal logits), or a bf16 row decided next to 0, the deciding value digit by digit over the row,
// 11 + 11 + 10 bits of the order-preserving integer of a float.
// (5) After (3), (4) or no limit: the token from sums of 256 neighbours.
//
// Bound by the chain of passes and exchanges for few rows and by the instructions of the weights (some 40 each), the atomics of the
// counts (some 16 clocks for 32 logits) and, with fp32 logits in (3), both for many; rows that take longest start first where not all
// run at once. us for 1 / 256 rows of 128256 bf16 logits (floor 0.04 / 10): largest logit 3 / 20, k = 50 with p 10 / 45, k = 1000
// 32 / 138, no limit 10 / 89, a p that keeps few 14 / 94, one that keeps thousands 20 / 138 - 156, rows of all kinds - / 80; of fp32 logits
// (floor 0.08 / 20) a p that keeps few 19 / 192, thousands 30 / 248.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <float.h>

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
constexpr int SM_STEPS = 32;                   // at most, per warp
constexpr int SM_BINS = 2048;
constexpr int SM_FINE = 4096;                   // bins of one bf16 value each: 16 binades of either sign
constexpr int SM_GROUPS = 64;                  // sums of neighbouring bins that CTAs exchange
constexpr int SM_COARSE = 512;                 // bins of the maxima
constexpr int SM_LIST = 2048;                  // tokens that a list takes
constexpr int SM_FEW = 128;                    // tokens that a p alone is expected to keep, where they are listed
constexpr int SM_CLUSTER = 8;                  // CTAs per row, at most
constexpr int SM_ORDER = 1024;                 // rows that a launch can put in order
constexpr int SM_ONE = 40;                     // log2 of the weight of the largest logit

struct SampleParams {
  const void* logits;
  long long ld;
  int rows, vocab, steps, vec, longest_first;
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
  union {
    u64 list[2 * SM_LIST];                     // every CTA has a part of it in rank 0
    struct {
      u64 part[SM_LIST];
      alignas(16) unsigned lo[SM_BINS];        // weights of the bins
      alignas(16) unsigned hi[SM_BINS];
    };
    alignas(16) unsigned fine[SM_FINE];        // counts of bf16 values
  };
  union {
    alignas(16) unsigned cnt[SM_BINS];         // counts of the bins
    u64 step[SM_WARPS * SM_STEPS];             // sums of 256 logits' values
    ulonglong2 pair[SM_THREADS];               // tokens of the list with their weights
  };
  u64 slot[10][3][SM_CLUSTER];                  // one set per exchange of a launch: values of every CTA
  u64 last;
  u64 warp[SM_WARPS];
  u64 res[5];
  alignas(16) u64 group[SM_GROUPS * SM_CLUSTER];
  unsigned exp2[32];
  int n_local, row;
  alignas(16) uint4 held[1];                   // SM_HELD steps of logits, or the maxima of all steps, as far as the launch goes
};

// Order-preserving integer of a float that is not NaN; -0 and subnormal numbers are 0.
__device__ __forceinline__ unsigned sm_key(float x) {
  const unsigned u = __float_as_uint(__fadd_rn(x, 0.f));
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sm_value(unsigned key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ u64 sm_entry(float x, int i) { return (u64)(~sm_key(x)) << 32 | (unsigned)i; }      // ascending: the order of the tokens
__device__ __forceinline__ float sm_entry_value(u64 e) { return sm_value(~(unsigned)(e >> 32)); }

// x - m as the sum of two floats. Logits that were rounded to bf16 (8 bits): exact in one where the two are within 2^16 of each other,
// the second is their difference's rounding where m is the larger. Where x is, the rounding would be lost, 2^-24 of x: a
// largest logit so near 0 that a logit with a weight can be 2^16 times as large is left out, m = 0, and every weight is exp(largest / T)
// times as large. Others: always exact.
template <bool BF16>
struct SampleWeight {
  float m, ch, cl;                             // 32 log2(e) / T in two floats
  float above;                                 // fp32: only logits above this weigh anything: -inf, beside infinite ones the largest finite number
  const unsigned* table;                       // 2^(j / 32) in units of 2^-31, one of the 32 banks each: any lanes read at once
  __device__ __forceinline__ u64 operator()(float x) const {     // NaN and -inf: 0
    // bf16: the callers pass no NaN, and the largest number is too far below FLT_MAX to weigh anything beside it
    x = BF16 || x > above ? fminf(x, FLT_MAX) : -INFINITY;
    const float s = __fsub_rn(x, m), t = __fadd_rn(s, m);
    const float r = BF16 ? __fsub_rn(x, t) : __fadd_rn(__fsub_rn(x, __fsub_rn(s, __fsub_rn(s, x))), -__fadd_rn(m, __fsub_rn(s, x)));
    const float p = fmaxf(__fmul_rn(s, ch), -2000.f);                               // 32nds of the exponent; 2^-62 is none
    const float e = __fmaf_rn(r, ch, __fmaf_rn(s, cl, __fmaf_rn(s, ch, -p)));
    const float big = __fadd_rn(p, 12582912.f);                                     // the next integer, in the low bits
    const float f = __fadd_rn(__fsub_rn(p, __fsub_rn(big, 12582912.f)), e);
    // 2^(f / 32) - 1, |f| <= 1 / 2: the series to f^3, with the middle of its fourth term in the second; off by 2^-32 at most
    const float q = __fmul_rn(f, __fmaf_rn(f, __fmaf_rn(f, 1.6938529e-06f, 2.3459933e-04f), 2.1660849e-02f));
    const int j = __float_as_int(big);                                              // 0x4b400000 + 32 exponent + 32nds
    const unsigned tj = table[j & 31];
    const unsigned w = tj + (unsigned)__float2int_rn(__fmul_rn(q, (float)tj));
    const int up = (j >> 5) + (SM_ONE - 31 - (0x4b400000 >> 5));                    // shift left, or right with rounding: the upper word of a product
    unsigned one;
    asm("shl.b32 %0, 1, %1;" : "=r"(one) : "r"(32 + up));                           // 0 where that is negative
    return up >= 0 ? (u64)w << up : ((u64)w * one + 0x80000000ull) >> 32;
  }
};
static_assert(SM_ONE <= 41, "right shifts of 32 bits at most");

// Sum over a warp of numbers below 2^44, in two halves of 22 bits.
__device__ __forceinline__ u64 sm_warp_sum(u64 v) {
  const unsigned lo = __reduce_add_sync(0xffffffffu, (unsigned)v & 0x3fffffu), hi = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 22));
  return ((u64)hi << 22) + lo;
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

// Threads for each of n <= SM_THREADS tokens of a list: a power of two up to eight.
__device__ __forceinline__ int sm_parts(int n) { return n <= SM_THREADS / 8 ? 8 : n <= SM_THREADS / 4 ? 4 : n <= SM_THREADS / 2 ? 2 : 1; }

// Ascending sort of n entries (a power of two from 128 to SM_LIST) in shared memory, by bitonic merges: what lies within 128 neighbours
// in a warp's registers, the rest with a barrier each (1024 entries: 6 of 55 steps).
__device__ __forceinline__ void sm_sort(u64* a, int n) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int k = 128; k <= n; k <<= 1) {
    for (int j = k >> 1; j >= 128; j >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += SM_THREADS) {
        const int i = 2 * t - (t & (j - 1));
        const u64 x = a[i], y = a[i + j];
        if ((x > y) == ((i & k) == 0)) { a[i] = y; a[i + j] = x; }
      }
    }
    __syncthreads();
    if (warp * 128 >= n) continue;             // a warp's 128, four a lane
    u64* own = a + warp * 128 + lane * 4;
    u64 v[4] = {own[0], own[1], own[2], own[3]};
    for (int k2 = k == 128 ? 2 : k; k2 <= k; k2 <<= 1)
#pragma unroll
      for (int j = 64; j > 0; j >>= 1) {
        if (j >= k2) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = warp * 128 + lane * 4 + q;
          if (j >= 4) {
            const u64 o = __shfl_xor_sync(0xffffffffu, v[q], j / 4);
            v[q] = ((i & j) == 0) == ((i & k2) == 0) ? min(v[q], o) : max(v[q], o);
          } else if ((q & j) == 0) {
            const u64 x = v[q], y = v[q | j];
            const bool up = (i & k2) == 0;
            v[q] = up ? min(x, y) : max(x, y);
            v[q | j] = up ? max(x, y) : min(x, y);
          }
        }
      }
    own[0] = v[0]; own[1] = v[1]; own[2] = v[2]; own[3] = v[3];
  }
  __syncthreads();
}
static_assert(SM_LIST <= SM_WARPS * 128, "a warp for every 128 entries");

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
  float* maxima;                               // else: this lane's largest logit of step 0, 512 lanes a step

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
    unpack(w, x);
  }
  __device__ __forceinline__ static void unpack(const unsigned (&w)[WORDS], float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = __uint_as_float(sizeof(T) == 4 ? w[j % WORDS] : j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  }
  // f(step, logits) over all steps, the next ones on their way
  template <typename F>
  __device__ __forceinline__ void each_words(F f) const {
    unsigned w[WORDS];
    if (steps > 0) words(0, w);
#pragma unroll 1
    for (int st = 0; st < steps; ++st) {
      unsigned now[WORDS];
#pragma unroll
      for (int j = 0; j < WORDS; ++j) now[j] = w[j];
      if (st + 1 < steps) words(st + 1, w);
      f(st, now);
    }
  }
  template <typename F>
  __device__ __forceinline__ void each_values(F f) const {
    each_words([&](int st, const unsigned (&w)[WORDS]) {
      float x[8];
      unpack(w, x);
      f(st, x);
    });
  }
  // the largest of a lane's eight logits; NaN only where all are
  __device__ __forceinline__ static float maximum(const unsigned (&w)[WORDS]) {
    if (sizeof(T) == 2) {
      const __nv_bfloat162 h = __hmax2(__hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]), *reinterpret_cast<const __nv_bfloat162*>(&w[1])),
                                       __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w[2]), *reinterpret_cast<const __nv_bfloat162*>(&w[3])));
      return fmaxf(__low2float(h), __high2float(h));
    }
    float v = __uint_as_float(w[0]);
#pragma unroll
    for (int j = 1; j < WORDS; ++j) v = fmaxf(v, __uint_as_float(w[j]));
    return v;
  }
  __device__ __forceinline__ float maximum(int step) const {
    if (!HELD) return maxima[step * SM_THREADS];
    unsigned w[WORDS];
    words(step, w);
    return maximum(w);
  }
  // The first pass: f(step, maximum) with the maxima noted; four steps' loads at a time.
  template <typename F>
  __device__ __forceinline__ void first_pass(F f) const {
    if (HELD) {
      each([&](int st) { f(st, maximum(st)); });
      return;
    }
    constexpr int AHEAD = 4;
    for (int st = 0; st < steps; st += AHEAD) {
      unsigned w[AHEAD][WORDS];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (st + j < steps) fetch(st + j, w[j]);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (st + j < steps) {
          const float v = maximum(w[j]);
          maxima[(st + j) * SM_THREADS] = v;
          f(st + j, v);
        }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int st = 0; st < steps; ++st) f(st);
  }
};

struct SampleSplit { unsigned bin; u64 cnt, w, target; };   // the deciding bin (SM_BINS: none), what lies above it, what was looked for

// First bin at which the cluster's running count (by_weight: weight) reaches target(weights of all), or all there is where that is
// less (all_there). Every CTA tells the others the sums of 64 groups of its bins (`group`: 64 x SM_CLUSTER values of counts, then of
// weights, as far as they are asked for) and its `here`, whose sum is handed to target; the deciding group's bins are then
// read from every CTA. One exchange, and a sixteenth of what reading all bins of all CTAs moved.
template <typename F>
__device__ __forceinline__ SampleSplit sm_find(cg::cluster_group& cl, SampleSmem& s, u64* group, u64* slot, int C, int rank, bool counts, bool by_weight, u64 here,
                                               F target_of, bool all_there, unsigned* in_bin) {
  constexpr int PER = SM_BINS / SM_THREADS, GROUP = SM_BINS / SM_GROUPS;      // bins of a thread, of a group
  static_assert(PER * SM_THREADS == SM_BINS && GROUP == 32 && GROUP / PER == SM_CLUSTER, "a lane of a group for every CTA, a lane for every bin");
  const int tid = threadIdx.x, lane = tid & 31;
  u64* group_w = group + (counts ? SM_GROUPS * SM_CLUSTER : 0);
  __syncthreads();                             // this CTA's bins are complete
  u64 sum_c = 0, sum_w = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (counts) sum_c += s.cnt[tid * PER + j];
    sum_w += (u64)s.hi[tid * PER + j] << 32 | s.lo[tid * PER + j];
  }
#pragma unroll
  for (int o = 1; o < GROUP / PER; o <<= 1) {
    sum_c += __shfl_xor_sync(0xffffffffu, sum_c, o);
    sum_w += __shfl_xor_sync(0xffffffffu, sum_w, o);
  }
  const int g = tid / (GROUP / PER), q0 = tid % (GROUP / PER);          // GROUP / PER = 8 lanes of a group: one CTA each
  if (q0 < C) {
    if (counts) cl.map_shared_rank(group, q0)[g * SM_CLUSTER + rank] = sum_c;
    cl.map_shared_rank(group_w, q0)[g * SM_CLUSTER + rank] = sum_w;
  }
  if (tid < C) cl.map_shared_rank(slot, tid)[rank] = here;
  cl.sync();
  u64 all = 0;
  for (int i = 0; i < C; ++i) all += slot[i];
  u64 target = target_of(all);
  if (tid < 32) {
    // two groups a lane, then one bin a lane
    u64 c[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
      for (int i = 0; i < C; ++i) {
        if (counts) c[j] += group[(2 * lane + j) * SM_CLUSTER + i];
        w[j] += group_w[(2 * lane + j) * SM_CLUSTER + i];
      }
    const u64 end_c = sm_warp_scan(c[0] + c[1]), end_w = sm_warp_scan(w[0] + w[1]);
    if (all_there && !by_weight) target = min(target, __shfl_sync(0xffffffffu, end_c, 31));
    u64 bc = end_c - c[0] - c[1], bw = end_w - w[0] - w[1];
    int mine = -1;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u64 b = by_weight ? bw : bc, a = by_weight ? w[j] : c[j];
      if (mine < 0) {
        if (a > 0 && b < target && b + a >= target) mine = 2 * lane + j;
        else { bc += c[j]; bw += w[j]; }
      }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, mine >= 0);
    if (hit == 0) {
      if (lane == 0) { s.res[0] = SM_BINS; s.res[1] = s.res[2] = s.res[3] = 0; }
    } else {
      const int owner = __ffs(hit) - 1;
      const int bin = __shfl_sync(0xffffffffu, mine, owner) * GROUP + lane;
      bc = __shfl_sync(0xffffffffu, bc, owner);
      bw = __shfl_sync(0xffffffffu, bw, owner);
      u64 n = 0, v = 0;
      for (int i = 0; i < C; ++i) {
        if (counts) n += cl.map_shared_rank(s.cnt, i)[bin];
        v += (u64)cl.map_shared_rank(s.hi, i)[bin] << 32 | cl.map_shared_rank(s.lo, i)[bin];
      }
      bc += sm_warp_scan(n) - n;
      bw += sm_warp_scan(v) - v;
      const u64 b = by_weight ? bw : bc, a = by_weight ? v : n;
      if (a > 0 && b < target && b + a >= target) { s.res[0] = bin; s.res[1] = bc; s.res[2] = bw; s.res[3] = n; }
    }
    if (lane == 0) s.res[4] = target;
  }
  __syncthreads();
  SampleSplit out;
  out.bin = (unsigned)s.res[0];
  out.cnt = s.res[1];
  out.w = s.res[2];
  out.target = s.res[4];
  *in_bin = (unsigned)s.res[3];
  return out;
}

// The same by counts in SM_COARSE bins, one a thread, which every CTA reads from all (after an exchange).
__device__ __forceinline__ SampleSplit sm_find_coarse(cg::cluster_group& cl, SampleSmem& s, int C, u64 target) {
  u64 n = 0, all;
  for (int i = 0; i < C; ++i) n += cl.map_shared_rank(s.cnt, i)[threadIdx.x];
  if (threadIdx.x == 0) s.res[0] = SM_COARSE;
  const u64 before = sm_block_scan(n, s, &all);
  if (n > 0 && before < target && before + n >= target) s.res[0] = threadIdx.x;
  __syncthreads();
  SampleSplit out;
  out.bin = (unsigned)s.res[0];
  return out;
}
static_assert(SM_COARSE == SM_THREADS, "one bin a thread");

// One weight into a bin: 64 bits from two native 32-bit atomics, whatever their order.
__device__ __forceinline__ void sm_add(SampleSmem& s, int b, u64 w) {
  const unsigned lo = (unsigned)w, hi = (unsigned)(w >> 32);
  const unsigned old = atomicAdd(&s.lo[b], lo);
  const unsigned up = hi + (old + lo < old ? 1u : 0u);
  if (up) atomicAdd(&s.hi[b], up);
}

// The q-th row where those that take longest come first: a p alone (0), no limit (1), a k or min_p alone (2), the largest logit (3).
// Up to SM_ORDER rows; every CTA looks at all of them. 256 rows of 128256 logits: of all kinds 100 us in their order, 80 so; of one
// kind 2 - 7 us more.
__device__ __forceinline__ int sm_longest_first(const SampleParams& p, SampleSmem& s, int q) {
  constexpr int PER = SM_ORDER / SM_THREADS, EACH = 4 * PER * SM_WARPS / 32;
  int* counts = reinterpret_cast<int*>(s.group);            // [class][run of 512 rows][warp]
  static_assert(4 * PER * SM_WARPS * 4 <= sizeof(s.group) && EACH % 4 == 0, "a few counts a lane");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int kind[PER], before[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int r = j * SM_THREADS + tid, at = min(r, p.rows - 1);
    const float temp = p.temperature[at], top_p = p.top_p ? p.top_p[at] : 1.f, min_p = p.min_p ? p.min_p[at] : 0.f;
    const int k = p.top_k ? p.top_k[at] : 0;
    kind[j] = r >= p.rows ? 4 : !(temp >= 0x1p-90f) ? 3 : k > 0 && k < p.vocab ? 2 : top_p < 1.f ? 0 : min_p > 0.f ? 2 : 1;
    before[j] = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned all = __ballot_sync(0xffffffffu, kind[j] == c);
      if (lane == 0) counts[(c * PER + j) * SM_WARPS + warp] = __popc(all);
      if (kind[j] == c) before[j] = __popc(all & ((1u << lane) - 1u));
    }
  }
  __syncthreads();
  // every warp sums them up for itself
  int n[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; i += 4) {
    const int4 v = reinterpret_cast<const int4*>(counts)[(lane * EACH + i) / 4];
    n[i] = v.x; n[i + 1] = v.y; n[i + 2] = v.z; n[i + 3] = v.w;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) { const int c = n[i]; n[i] = sum; sum += c; }
  int first = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, first, o);
    if (lane >= o) first += t;
  }
  first -= sum;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = (min(kind[j], 3) * PER + j) * SM_WARPS + warp;
    int place = before[j] + __shfl_sync(0xffffffffu, first, i / EACH);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int t = __shfl_sync(0xffffffffu, n[e], i / EACH);
      place += e == i % EACH ? t : 0;
    }
    if (kind[j] < 4 && place == q) s.row = j * SM_THREADS + tid;
  }
  __syncthreads();
  return s.row;
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
  if (tid == 0) s.n_local = 0;
  for (int i = tid; i < SM_COARSE; i += SM_THREADS) s.cnt[i] = 0;
  if (sizeof(T) == 2)
    for (int i = tid; i < SM_FINE / 4; i += SM_THREADS) reinterpret_cast<uint4*>(s.fine)[i] = make_uint4(0u, 0u, 0u, 0u);
  pdl_wait();
  const int r = p.longest_first ? sm_longest_first(p, s, blockIdx.x / C) : blockIdx.x / C;
  SampleRow<T, HELD> row;
  row.row = reinterpret_cast<const T*>(p.logits) + (long long)r * p.ld;
  row.vocab = p.vocab;
  row.first = (rank * SM_WARPS + warp) * p.steps * SM_STEP;
  row.steps = max(0, min(p.steps, (p.vocab - row.first + SM_STEP - 1) / SM_STEP));
  row.vec = p.vec;
  row.held = s.held + tid;
  row.maxima = reinterpret_cast<float*>(s.held) + tid;
  row.hold();
  const float given = p.temperature[r], temp = given > 0x1p90f ? 0x1p90f : given, top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f, u = p.u[r];
  const int top_k = p.top_k ? p.top_k[r] : 0;
  const bool greedy = !(temp >= 0x1p-90f) || min_p > 1.f;          // the first token of the order alone

  // ---- (1) the largest logit, with its first index where that is the answer; mean and variance of the first step's logits, as far as the
  // largest (of the warp, then of the CTA, then of all) does not make them masked ones
  const float masked = 40.f * temp;
  float best = -INFINITY, sum = 0.f, square = 0.f;
  int best_st = 0, n_sum = 0;
  row.first_pass([&](int st, float v) {
    if (v > best) { best = v; best_st = st; }
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
    if (row.steps > 0) {
      float x[8];
      row.values(0, x);
      const float from = fmaxf(sm_value((unsigned)(top >> 32)) - masked, -0x1p60f);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x[j] > from) { sum += x[j]; square += x[j] * x[j]; ++n_sum; }
    }
    n_sum = __reduce_add_sync(0xffffffffu, n_sum);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      square += __shfl_xor_sync(0xffffffffu, square, o);
    }
  }
  if (lane == 0) {
    s.group[warp] = top;
    s.group[SM_WARPS + warp] = (u64)__float_as_uint(sum) << 32 | __float_as_uint(square);
    s.group[2 * SM_WARPS + warp] = (u64)n_sum;
  }
  __syncthreads();
  cl.barrier_wait();
  // largest logit (and index) of up to 32 parts, a part a lane; sums over the parts that are not masked beside it. The sums in lane 0.
  auto combine = [&](u64& t, float& f, float& g, unsigned& n, int parts) {
    const unsigned hi = (unsigned)(t >> 32), most = __reduce_max_sync(0xffffffffu, hi);
    t = (u64)most << 32 | __reduce_max_sync(0xffffffffu, hi == most ? (unsigned)t : 0u);
    if (greedy) return;
    const bool in = sm_value(hi) >= sm_value(most) - masked;          // an empty lane: NaN
    n = __reduce_add_sync(0xffffffffu, in ? n : 0u);
    f = in ? f : 0.f;
    g = in ? g : 0.f;
#pragma unroll
    for (int o = SM_WARPS / 2; o > 0; o >>= 1)
      if (o < parts) {
        f += __shfl_xor_sync(0xffffffffu, f, o);
        g += __shfl_xor_sync(0xffffffffu, g, o);
      }
  };
  u64 fg = 0;
  if (warp == 0) {
    top = lane < SM_WARPS ? s.group[lane] : 0ull;
    fg = lane < SM_WARPS ? s.group[SM_WARPS + lane] : 0ull;
    unsigned n = lane < SM_WARPS ? (unsigned)s.group[2 * SM_WARPS + lane] : 0u;
    sum = __uint_as_float((unsigned)(fg >> 32));
    square = __uint_as_float((unsigned)fg);
    combine(top, sum, square, n, SM_WARPS);
    if (lane < C) {                            // lane i tells CTA i: all lanes below 16 have the sums
      u64* to = cl.map_shared_rank(&s.slot[0][0][0], lane);
      to[rank] = top;
      to[SM_CLUSTER + rank] = (u64)__float_as_uint(sum) << 32 | __float_as_uint(square);
      to[2 * SM_CLUSTER + rank] = n;
    }
  }
  cl.sync();
  top = lane < C ? s.slot[0][0][lane] : 0ull;
  fg = lane < C ? s.slot[0][1][lane] : 0ull;
  unsigned n_all = lane < C ? (unsigned)s.slot[0][2][lane] : 0u;
  float mean = __uint_as_float((unsigned)(fg >> 32)), var = __uint_as_float((unsigned)fg);
  combine(top, mean, var, n_all, SM_CLUSTER);
  const float m = sm_value((unsigned)(top >> 32));
  if (m == -INFINITY || greedy) {
    if (rank == 0 && tid == 0) {
      p.tokens[r] = m == -INFINITY ? 0 : (long long)(unsigned)~(unsigned)top;
      if (p.logprobs) p.logprobs[r] = m == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  mean = __shfl_sync(0xffffffffu, mean, 0);
  var = __shfl_sync(0xffffffffu, var, 0);
  const float n_mean = (float)n_all;
  // what lies further below the largest logit weighs 2^-41 of it at most, nothing: it is in no list and in no bin's range
  const float nothing = fmaxf(fminf(m, FLT_MAX) - 29.f * temp, -FLT_MAX);
  mean = n_mean > 0.f ? fmaxf(__fdiv_rn(mean, n_mean), nothing) : nothing;
  var = n_mean > 0.f ? fmaxf(__fdiv_rn(var, n_mean) - mean * mean, 0.f) : 0.f;
  SampleWeight<sizeof(T) == 2> weight;
  const double scale = 32. * 1.4426950408889634074 / (double)temp;
  // bf16: above 2^-11 T nothing down to 29 T below it is 2^16 times as large
  weight.m = sizeof(T) == 2 && fabsf(m) < 0x1p-11f * temp ? 0.f : fminf(m, FLT_MAX);
  weight.above = m == INFINITY ? FLT_MAX : -INFINITY;
  weight.ch = (float)scale;
  weight.cl = (float)(scale - (double)weight.ch);
  weight.table = s.exp2;
  auto finish = [&](long long token, float x, u64 total) {  // one thread of the row
    p.tokens[r] = token;
    if (p.logprobs) {
      const double lw = ((double)fminf(x, FLT_MAX) - (double)weight.m) / (double)temp;
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
  // ---- (5) the first index at which the running sum of value(logit, index) reaches target(total): found(index, logit, total) in one thread.
  // Logits below `floor_x` have none: steps whose maxima all are below it cost one comparison.
  auto locate = [&](float floor_x, auto value, auto target, auto found) {
    auto wanted = [&](int st) { return st < row.steps && __any_sync(0xffffffffu, row.maximum(st) >= floor_x); };
    unsigned w[SampleRow<T, HELD>::WORDS];
    bool now = wanted(0);
    if (now) row.words(0, w);
#pragma unroll 1
    for (int st = 0; st < row.steps; ++st) {
      u64 v = 0;
      if (now) {
        float x[8];
        row.unpack(w, x);
        now = wanted(st + 1);
        if (now) row.words(st + 1, w);         // the next ones on their way
        const int i = row.index(st);
#pragma unroll
        for (int j = 0; j < 8; ++j) v += value(x[j], i + j);
        v = sm_warp_sum(v);
      } else {
        now = wanted(st + 1);
        if (now) row.words(st + 1, w);
      }
      if (lane == 0) s.step[warp * p.steps + st] = v;
    }
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
      float at_x = x[0];
#pragma unroll
      for (int q = 0; q < 7; ++q) {
        from += e[q];
        if (from < t) { j = q + 1; at_x = x[q + 1]; }
      }
      found(i + j, at_x, a.x);
    }
  };

  if (need_k || need_p) {
    u64 w_all = 0, target_p = ~0ull;
    float per;
    int n_bins;
    auto bins = [&](int n, float width) {
      n_bins = n;
      per = __fdiv_rn((float)(n - 1), width);
      if (!(per > 0.f && per < 3e38f)) per = 0.f;
    };
    auto bin_of = [&](float x) {                            // what is below the range: the last one; the order of the logits
      const float f = __fmul_rn(__fsub_rn(m, x), per);
      return f < (float)(n_bins - 1) ? (int)f : n_bins - 1;
    };
    auto block_sum = [&](u64 here) {
      u64 t;
      sm_block_scan(here, s, &t);
      return t;
    };
    auto reach = [&](u64 all) {
      w_all = all;
      return target_p = max(1ull, sm_reach(top_p, all));
    };
    // The list: tokens that wanted() names, in rank 0; how many, or 0 where they do not fit. room: entries of a CTA's part.
    int room = 0;
    auto gather = [&](auto wanted) {
      u64* to = cl.map_shared_rank(s.list, 0) + rank * room;
      row.each([&](int st) {
        if (!wanted(row.maximum(st), true)) return;
        float x[8];
        row.values(st, x);
        const int i = row.index(st);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (x[j] >= nothing && wanted(x[j], false)) {
            const int at = atomicAdd(&s.n_local, 1);
            if (at < room) to[at] = sm_entry(x[j], i + j);
          }
      });
      __syncthreads();
      if (tid < C) cl.map_shared_rank(&s.slot[ex][0][0], tid)[rank] = (u64)s.n_local;
      cl.sync();
      int n = 0, most = 0;
      for (int i = 0; i < C; ++i) {
        const int c = (int)s.slot[ex][0][i];
        n += c;
        most = max(most, c);
      }
      if (tid == 0) s.n_local = 0;
      ++ex;
      return n <= SM_LIST && most <= room ? n : 0;
    };
    auto entry = [&](int i) {                               // rank 0: the i-th of the list, across the CTAs' parts
      int q = 0;
      for (; q < C - 1; ++q) {
        const int c = (int)s.slot[ex - 1][0][q];
        if (i < c) break;
        i -= c;
      }
      return s.list[q * room + i];
    };
    bool open = true;
    u64 n_class = 0, n_take = 0;                            // tokens with the deciding logit, and how many of them are kept
    // p alone: a normal distribution with this mean and variance has V exp((mean - m) / T + var / 2 T^2) of the largest logit's weight, and
    // z standard deviations above the mean 128 tokens, below which all but the upper tail beyond z - sigma / T of that weight
    // lies. Where that is more than p leaves out, 128 tokens will not do. Only the way depends on it, not the token.
    bool flat = false;
    if (sizeof(T) == 4 && !need_k && p.vocab > SM_LIST) {
      const float inv_t = __fdiv_rn(1.f, temp), t = sqrtf(2.f * __logf((float)p.vocab / SM_FEW));
      const float z = t - (2.30753f + 0.27061f * t) / (1.f + t * (0.99229f + 0.04481f * t));      // Hastings' approximation of the normal quantile
      const float bulk = __expf(__logf((float)p.vocab) + ((mean - m) + 0.5f * var * inv_t) * inv_t);
      flat = bulk * normcdff(z - sqrtf(var) * inv_t) > (1.f - top_p) * (bulk + 2.f);
    }
    if (sizeof(T) == 2 && !need_k) {
      // ---- (3) for bf16
      const float low = fmaxf(mean - 4.f * sqrtf(var), nothing);
      const int e_top = max(max((int)(__float_as_uint(m) >> 23 & 255u), (int)(__float_as_uint(low) >> 23 & 255u)), 16);
      const int most = e_top << 7 | 127;                    // magnitudes (15 bits) from here down: SM_FINE / 2 of them, no subnormal one
      u64 w_small = 0, w_low = 0;                           // weights of what is nearer to 0 than the bins, and of what lies below them
      row.each_words([&](int st, const unsigned (&w)[SampleRow<T, HELD>::WORDS]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned b = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
          const int mag = (int)(b & 0x7fffu), d = most - mag;
          if ((unsigned)d < SM_FINE / 2 && mag <= 0x7f80) {
            atomicAdd(&s.fine[b & 0x8000u ? SM_FINE - 1 - d : d], 1u);
          } else if (__uint_as_float(b << 16) >= nothing) { // no NaN either
            const u64 v = weight(__uint_as_float(b << 16));
            if (d < 0) w_low += v;
            else w_small += v;
          }
        }
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        w_small += __shfl_xor_sync(0xffffffffu, w_small, o);
        w_low += __shfl_xor_sync(0xffffffffu, w_low, o);
      }
      if (lane == 0) {
        s.group[warp] = w_small;
        s.group[SM_WARPS + warp] = w_low;
      }
      __syncthreads();
      if (tid < C) {
        w_small = w_low = 0;
#pragma unroll
        for (int i = 0; i < SM_WARPS; ++i) {
          w_small += s.group[i];
          w_low += s.group[SM_WARPS + i];
        }
        u64* to = cl.map_shared_rank(&s.slot[ex][0][0], tid);
        to[rank] = w_small;
        to[SM_CLUSTER + rank] = w_low;
      }
      cl.sync();
      w_small = w_low = 0;
      for (int i = 0; i < C; ++i) {
        w_small += s.slot[ex][0][i];
        w_low += s.slot[ex][1][i];
      }
      ++ex;
      // every CTA takes its share of the bins from all, `per` of them a thread in the order of the logits; what is near 0 stands before the
      // first negative one
      constexpr int MOST = SM_FINE / SM_THREADS;
      const int per = MOST / C, base = (rank * SM_THREADS + tid) * per;
      unsigned n[MOST];
#pragma unroll
      for (int i = 0; i < MOST; ++i) n[i] = cl.map_shared_rank(s.fine, i / per)[base + i % per];
#pragma unroll
      for (int o = MOST / 2; o > 0; o >>= 1)
        if (per <= o)
#pragma unroll
          for (int i = 0; i < o; ++i) { n[i] += n[i + o]; n[i + o] = 0; }
      auto value_of = [&](int bin) {
        return __uint_as_float(bin < SM_FINE / 2 ? (unsigned)(most - bin) << 16 : 0x80000000u | (unsigned)(most - (SM_FINE - 1 - bin)) << 16);
      };
      u64 w[MOST], mine = base == SM_FINE / 2 ? w_small : 0ull, here;
#pragma unroll
      for (int j = 0; j < MOST; ++j) {
        w[j] = n[j] > 0 ? weight(value_of(base + j)) : 0ull;
        mine += n[j] * w[j];
      }
      u64 before = sm_block_scan(mine, s, &here) + (base == SM_FINE / 2 ? w_small : 0ull);
      u64 (*const found)[SM_CLUSTER] = s.slot[ex + 1];      // of the deciding bin: logit, tokens, how many of them are kept
      if (tid == 0) found[1][0] = 0;
      const ulonglong2 sums = exchange_sum(here);
      before += sums.y;
      const u64 target = reach(sums.x + w_low);
      ++ex;
#pragma unroll
      for (int j = 0; j < MOST; ++j) {
        const u64 a = n[j] * w[j];
        if (a > 0 && before < target && before + a >= target)
          for (int q = 0; q < C; ++q) {
            u64* to = cl.map_shared_rank(&found[0][0], q);
            to[0] = __float_as_uint(value_of(base + j));
            to[SM_CLUSTER] = n[j];
            to[2 * SM_CLUSTER] = (target - before + w[j] - 1) / w[j];
          }
        before += a;
      }
      cl.sync();
      n_class = found[1][0];
      if (n_class > 0) {                                    // else near 0, or below the bins: (4)
        last_x = __uint_as_float((unsigned)found[0][0]);
        n_take = found[2][0];
        open = false;
      }
    } else if (!flat) {
      // ---- (2)
      bins(SM_COARSE, m - mean);
      u64 w_here = 0;
      row.each([&](int st) {
        const float v = row.maximum(st);
        const int b = bin_of(v);
        if (v >= nothing && b < SM_COARSE - 1) atomicAdd(&s.cnt[b], 1u);
        if (!need_k) {
          float x[8];
          row.values(st, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) w_here += weight(x[j]);
        }
      });
      if (need_k) cl.sync();
      else reach(exchange_sum(block_sum(w_here)).x);
      const SampleSplit sp = sm_find_coarse(cl, s, C, need_k ? (u64)top_k : (u64)SM_FEW);
      const int upto = sp.bin < SM_COARSE ? (int)sp.bin : SM_COARSE - 1;           // fewer in the bins: everything
      room = min(SM_LIST, 2 * SM_LIST / C);
      const int n = gather([&](float x, bool) { return x >= nothing && bin_of(x) <= upto; });
      if (n > 0) {
        if (rank == 0) {
          const int n_k = need_k ? min(top_k, n) : n;
          u64 target = target_p;
          bool enough = true;
          if (n <= SM_THREADS) {
            // a token for every one to eight threads: what comes before it is counted and summed directly
            const int parts = sm_parts(n), t = tid / parts, part = tid % parts;
            u64 mine = ~0ull, w = 0, before = 0;
            int ahead = 0;
            if (tid < n) {
              const u64 e = entry(tid);
              s.pair[tid] = make_ulonglong2(e, weight(sm_entry_value(e)));
            }
            __syncthreads();
            if (t < n) {
              mine = s.pair[t].x;
              w = s.pair[t].y;
              for (int j = part; j < n; j += parts) {
                const ulonglong2 o = s.pair[j];
                if (o.x < mine) { ++ahead; before += o.y; }
              }
            }
            for (int o = 1; o < parts; o <<= 1) {
              ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
              before += __shfl_xor_sync(0xffffffffu, before, o);
            }
            if (need_p) {
              u64 all;
              sm_block_scan(t < n && part == 0 && ahead < n_k ? w : 0ull, s, &all);
              if (need_k) target = sm_reach(top_p, all);
              enough = all >= target;
            }
            // kept: what begins below the target, is among the first k and not below min_p; the first token always
            const bool in = t < n && ahead < n_k && (ahead == 0 || ((!need_p || before < target) && sm_entry_value(mine) >= least));
            __syncthreads();
            if (t < n && part == 0) s.pair[t].y = in ? w : 0ull;
            __syncthreads();
            u64 all = 0;
            before = 0;
            if (t < n)
              for (int j = part; j < n; j += parts) {
                const ulonglong2 o = s.pair[j];
                all += o.y;
                before += (unsigned)o.x < (unsigned)mine ? o.y : 0;
              }
            for (int o = 1; o < parts; o <<= 1) {
              all += __shfl_xor_sync(0xffffffffu, all, o);
              before += __shfl_xor_sync(0xffffffffu, before, o);
            }
            if (in && part == 0 && enough) {
              const u64 goal = sm_above(u, all);
              if (before < goal && before + w >= goal) finish((long long)(unsigned)mine, sm_entry_value(mine), all);
            }
          } else {
            constexpr int PER = SM_LIST / SM_THREADS;
            int pow2 = 2 * SM_THREADS;
            while (pow2 < n) pow2 <<= 1;
            u64 e[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) e[j] = tid + j * SM_THREADS < n ? entry(tid + j * SM_THREADS) : ~0ull;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; ++j)
              if (tid + j * SM_THREADS < pow2) s.list[tid + j * SM_THREADS] = e[j];
            sm_sort(s.list, pow2);
            const int each = pow2 / SM_THREADS;
            u64 w[PER], mine = 0, all;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const int i = tid * each + j;
              w[j] = j < each && i < n_k ? weight(sm_entry_value(s.list[i])) : 0ull;
              mine += w[j];
            }
            u64 before = sm_block_scan(mine, s, &all);
            if (need_k && need_p) target = sm_reach(top_p, all);
            enough = !need_p || all >= target;
            u64 kept = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const int i = tid * each + j;
              if (j < each && i < n_k && (i == 0 || ((!need_p || before < target) && sm_entry_value(s.list[i]) >= least))) ++kept;
              before += w[j];
            }
            u64 n_kept;
            sm_block_scan(kept, s, &n_kept);
            if (enough) {
              const int nk = (int)n_kept;
              u64* by_index = s.list + SM_LIST;             // the same by index
              int pow2k = 128;
              while (pow2k < nk) pow2k <<= 1;
              for (int i = tid; i < pow2k; i += SM_THREADS) {
                const u64 x = s.list[i];
                by_index[i] = i < nk ? x << 32 | x >> 32 : ~0ull;
              }
              sm_sort(by_index, pow2k);
              const int each_k = (pow2k + SM_THREADS - 1) / SM_THREADS;
              mine = 0;
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                const int i = tid * each_k + j;
                w[j] = j < each_k && i < nk ? weight(sm_value(~(unsigned)by_index[i])) : 0ull;
                mine += w[j];
              }
              before = sm_block_scan(mine, s, &all);
              const u64 t = sm_above(u, all);
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                const int i = tid * each_k + j;
                if (before < t && before + w[j] >= t) finish((long long)(by_index[i] >> 32), sm_value(~(unsigned)by_index[i]), all);
                before += w[j];
              }
            }
          }
          if (!need_k && tid < C) *cl.map_shared_rank(&s.last, tid) = enough ? 1ull : 0ull;
        }
        if (need_k) return;
        cl.sync();
        open = s.last == 0;
        if (!open) return;
      }
    }
    if (sizeof(T) == 4 && !need_k && open) {
      // ---- (3) for fp32: down to where a third of what p leaves out is expected below; where that misses the deciding value, as far below
      // the mean as half of what the largest logit is above it
      const float inv_t = __fdiv_rn(1.f, temp);
      const float deep = m - (mean + var * inv_t + sqrtf(var) * normcdfinvf(fmaxf(1.f - top_p, 1e-6f) * 0.33f));
      SampleSplit sp;
      unsigned in_bin;
      bool known = !flat;                      // the sum of all weights
      for (int go = 0; go < 2; ++go) {
        if (go > 0) cl.sync();                 // the others have read the bins
        for (int i = tid; i < SM_BINS; i += SM_THREADS) s.lo[i] = s.hi[i] = 0;
        __syncthreads();
        bins(SM_BINS, go == 0 ? deep : 1.5f * (m - mean));
        u64 w_here = 0;
        row.each_values([&](int st, const float (&x)[8]) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int b = bin_of(x[j]);
            if (b >= SM_BINS - 1 && known) continue;
            const u64 w = weight(x[j]);
            if (b < SM_BINS - 1) sm_add(s, b, w);
            w_here += w;
          }
        });
        const u64 target = target_p;
        const bool fresh = !known;
        sp = sm_find(cl, s, s.group, s.slot[ex++][0], C, rank, false, true, block_sum(w_here), [&](u64 all) { return fresh ? reach(all) : target; }, false, &in_bin);
        known = true;
        if (sp.bin < SM_BINS) break;
      }
      if (sp.bin < SM_BINS) {
        room = SM_LIST / C;
        const int n = gather([&](float x, bool any) { return any ? bin_of(x) <= (int)sp.bin : bin_of(x) == (int)sp.bin; });
        if (n > 0) {
          // the last token that p keeps: the one at which the running weight reaches the target
          if (rank == 0) {
            constexpr int PER = SM_LIST / SM_THREADS;
            auto last_one = [&](u64 e) {
              for (int q = 0; q < C; ++q) *cl.map_shared_rank(&s.last, q) = e;
            };
            if (n <= SM_THREADS) {
              const int parts = sm_parts(n), t = tid / parts, part = tid % parts;
              u64 mine = ~0ull, w = 0, before = 0;
              if (tid < n) {
                const u64 e = entry(tid);
                s.pair[tid] = make_ulonglong2(e, weight(sm_entry_value(e)));
              }
              __syncthreads();
              if (t < n) {
                mine = s.pair[t].x;
                w = s.pair[t].y;
                for (int j = part; j < n; j += parts) {
                  const ulonglong2 o = s.pair[j];
                  if (o.x < mine) before += o.y;
                }
              }
              for (int o = 1; o < parts; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
              before += sp.w;
              if (t < n && part == 0 && before < target_p && before + w >= target_p) last_one(mine);
            } else {
              int pow2 = 2 * SM_THREADS;
              while (pow2 < n) pow2 <<= 1;
              u64 e[PER];
#pragma unroll
              for (int j = 0; j < PER; ++j) e[j] = tid + j * SM_THREADS < n ? entry(tid + j * SM_THREADS) : ~0ull;
              __syncthreads();
#pragma unroll
              for (int j = 0; j < PER; ++j)
                if (tid + j * SM_THREADS < pow2) s.list[tid + j * SM_THREADS] = e[j];
              sm_sort(s.list, pow2);
              const int each = pow2 / SM_THREADS;
              u64 w[PER], mine = 0, all;
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                const int i = tid * each + j;
                w[j] = j < each && i < n ? weight(sm_entry_value(s.list[i])) : 0ull;
                mine += w[j];
              }
              u64 before = sp.w + sm_block_scan(mine, s, &all);
#pragma unroll
              for (int j = 0; j < PER; ++j) {
                if (before < target_p && before + w[j] >= target_p) last_one(s.list[tid * each + j]);
                before += w[j];
              }
            }
          }
          cl.sync();
          last_x = sm_entry_value(s.last);
          last_i = (int)(unsigned)s.last;
          open = false;
        }
      }
    }
    if (open) {
      // ---- (4)
      auto decide = [&](bool by_weight, u64 target, u64* n_class, u64* n_above, u64* w_above) {
        unsigned prefix = 0;
        *n_above = *w_above = 0;
        int done = 0;
        for (int level = 0; level < 3; ++level) {
          const int bits = level < 2 ? 11 : 10, shift = level == 0 ? 21 : level == 1 ? 10 : 0;
          cl.sync();                           // the others have read the bins
          for (int i = tid; i < SM_BINS; i += SM_THREADS) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
          __syncthreads();
          row.each_values([&](int st, const float (&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const unsigned key = sm_key(x[j]);
              if (!(x[j] > -INFINITY) || (done > 0 && key >> (32 - done) != prefix)) continue;
              const int b = (1 << bits) - 1 - (int)((key >> shift) & ((1u << bits) - 1));
              atomicAdd(&s.cnt[b], 1u);
              if (need_p) sm_add(s, b, weight(x[j]));
            }
          });
          unsigned in_class;
          const u64 goal = target;
          const SampleSplit d = sm_find(cl, s, s.part, s.slot[9][0], C, rank, true, by_weight, 0ull, [&](u64) { return goal; }, level == 0, &in_class);
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
      u64 n_above, w_above, w_total = w_all;
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
    }
    if (n_take < n_class) {                    // some of the tokens with this logit: those of the lowest indices
      locate(last_x, [&](float x, int) { return x == last_x ? 1ull : 0ull; }, [&](u64) { return n_take; },
             [&](int i, float, u64) {
               for (int q = 0; q < C; ++q) *cl.map_shared_rank(&s.last, q) = (u64)i;
             });
      cl.sync();
      last_i = (int)s.last;
    }
  }
  if (least > last_x) {
    last_x = least;
    last_i = 0x7fffffff;
  }
  // behind last_i only logits above last_x: not less than the next normal number; none above infinity
  const float next_x = last_x == INFINITY ? __int_as_float(0x7fffffff) : last_x == 0.f ? FLT_MIN : sm_value(sm_key(last_x) + 1);
  locate(last_x, [&](float x, int i) { return weight(x >= (i <= last_i ? last_x : next_x) ? x : -INFINITY); }, [&](u64 total) { return sm_above(u, total); },
         [&](int i, float x, u64 total) { finish(i, x, total); });
}

}  // namespace mlf

using namespace mlf;

// CTAs per row: as many as a warp's steps need, none with less than 4096 logits; beyond that, more of them shorten the rows whose p keeps
// most of a flat distribution, which take four times as long as one with a small k, and cost every row their exchanges.
// us at 128256 bf16 logits with 1 / 2 / 4 CTAs: 256 rows of k = 50 34 / 44 / 64, without limits 88 / 89 / 102, of all kinds 147 / 80 / 95;
// with 1 / 2 / 4 / 8, 33 rows of 50257 fp32 logits, k = 50 22 / 20 / 17 / 22, of all kinds 73 / 49 / 39 / 31 (two CTAs fit an SM, but
// clusters of eight only 32 times). So four CTAs for every SM, and clusters of eight where all run at once.
static int sample_cluster(long long rows, int vocab) {
  int c = 1;
  while (c < SM_CLUSTER && (vocab > c * SM_WARPS * SM_STEP * SM_STEPS ||
                            (vocab > c * 4096 && (2 * c < SM_CLUSTER ? rows * 2 * c <= 4 * sm_count() : rows * 2 * c * 4 <= 7 * sm_count()))))
    c *= 2;
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
  p.longest_first = rows * C > 2 * sm_count() && rows <= SM_ORDER;
  p.u = u; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
  p.tokens = tokens; p.logprobs = logprobs;
  const bool held = p.steps <= SM_HELD;
  const auto kernel = is_fp32 ? (held ? sample_rows_kernel<float, true> : sample_rows_kernel<float, false>)
                              : (held ? sample_rows_kernel<__nv_bfloat16, true> : sample_rows_kernel<__nv_bfloat16, false>);
  // for the most steps, held or noted: one size for every launch of a kernel
  const size_t smem = sizeof(SampleSmem) + (held ? (size_t)SM_HELD * SM_THREADS * 8 * (is_fp32 ? 4 : 2) : (size_t)SM_STEPS * SM_THREADS * sizeof(float));
  static bool attr_set[64][4] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  bool& set = attr_set[dev & 63][(is_fp32 ? 2 : 0) + (held ? 1 : 0)];
  if (!set) {
    MLF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    set = true;
  }
  MLF_CHECK_CUDA(launch_pdl_cluster(kernel, dim3((unsigned)(rows * C)), dim3(SM_THREADS), smem, dim3((unsigned)C),
                                    reinterpret_cast<cudaStream_t>(stream), p));
  count_launch();
  return 0;
}
