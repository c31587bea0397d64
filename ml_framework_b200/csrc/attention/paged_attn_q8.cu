// Decode attention over a paged 8-bit cache (layout and scales: kv_q8.cuh): one query token per sequence,
//
//   o_h = sum_t p_t v_t,  p = softmax_t(scale q_h . k_t),  k_t = s_K(block of t) K[t],  v_t = s_V(block of t) V[t],  t < len.
//
// Bound by HBM: a cached token and KV head is 256 bytes and 4 * 128 multiply-adds per query head. What has to fit beside the
// loads is the conversion of every byte, so numbers go to f16 pairs (exact for both types, one instruction for two e4m3) and
// both products run on warp-level m16n8k16 tensor-core tiles with the cache as the 16-row operand:
//   S^T (16 tokens x 8 heads) = K (16 x 128) Q^T,   O^T (128 x 8 heads) += V^T (128 x 16) P^T.
// Both sums run in an order of our choice, and so do the rows of O^T: a lane takes 16 consecutive bytes of a row wherever the
// tile layout asks for some of its columns, with the query's columns permuted alike, so that cached bytes go from global
// memory to the lane that multiplies them without a transposition (V^T pairs two tokens' bytes with a byte permutation).
//
// The scales stay out of the products: s_K multiplies a token's scores, and s_V enters the exponent, w_t = p_t s_V(t) =
// 2^15 exp2(x_t + log2 s_V(t) - M) with M the running maximum of that sum: whatever the scales, the weights that are rounded to
// f16 are at most 2^15, and those down to 2^-29 of the largest are exact to 2^-11, smaller ones to 2^-40 of the largest. The
// softmax's own sum is sum_t w_t / s_V(t), in fp32.
// The query is brought to f16 by a power of two per head that puts its largest element into [2^7, 2^8): exact for elements down
// to 2^-21 of the largest, whose bf16 significands f16 holds whole.
//
// A CTA's warps take the pairs of tiles of its run in turn, and each keeps the next pair in flight. Where a tile of 16 tokens lies in
// one block (blocks of a multiple of 16), TMA fetches it, one box of 16 rows of 128 bytes for the keys and one for the values, and
// the warp waits at a barrier of its own; asynchronous 16-byte copies by the lanes, which the other block sizes take, read at most
// 5.0 TB/s without any arithmetic and 4.4 with it where the boxes give 5.7 (4 x 60001 tokens of 8 heads: 117 us and 86, floor 75).
// The box's rows are swizzled: the 16-byte column x of row r lies at column x ^ (r & 7), so that a lane that takes columns 2 c and
// 2 c + 1 of key rows g and g + 8, and column g of four value rows, shares no bank with the seven that read at the same time.
//
// Few sequences are split over CTAs, which merge through distributed shared memory where they all run at once. Other figures (us,
// floor): 1 x 700 5.3 (0.2: the chain length - table - tile - softmax and the merge), 13 x 2500 18 (9.3), 64 x 576 16 (8.9: one round of
// CTAs, half of it their first loads), 24 x 900 of 40 heads 34 (26: 1.6 rounds), 600 x 900
// 185 (169).
#include <cooperative_groups.h>

#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../common/rope.cuh"
#include "../mlf_api.h"
#include "kv_q8.cuh"

namespace mlf {

namespace cg = cooperative_groups;

constexpr int DQ_WARPS = 4;                                  // at most
constexpr int DQ_TILE = 16;                                  // tokens
constexpr int DQ_PAIR = 2;                                   // tiles that a warp works on at once
constexpr int DQ_STAGES = 2;                                 // pairs in flight per warp
constexpr int DQ_TILE_BYTES = 2 * DQ_TILE * Q8_D + 128;      // keys, values, 16 + 16 scales
constexpr int DQ_STAGE_BYTES = DQ_PAIR * DQ_TILE_BYTES;
constexpr int DQ_SMEM = DQ_WARPS * DQ_STAGES * DQ_STAGE_BYTES;
constexpr int DQ_BOX_STAGE = DQ_PAIR * 2 * DQ_TILE * Q8_D;   // of the TMA form: scales stay in registers
constexpr int dq_box_smem(int warps) { return warps * DQ_STAGES * DQ_BOX_STAGE + 1024; }
constexpr float DQ_UP = 15.f;                                // log2 of the largest weight
constexpr int DQ_CLUSTER = 8;                                // splits that a cluster merges
constexpr int DQ_RED = Q8_D + 2;                             // floats of a partial result: maximum, sum, output

struct DecodeQ8Params {
  const __nv_bfloat16* q;         // [B, Hq, 128], row pitch ldq elements
  long long ldq;
  uint8_t* cache;
  float* scale;
  const int* block_table;         // [B, max_blocks]
  const int* seq_lens;            // [B]
  __nv_bfloat16* out;             // [B, Hq, 128]
  float* ws;                      // [B, Hkv, splits, G, 130] (m, l, o[128]): splits that a second kernel merges
  int B, Hq, Hkv, G, block_size, bs_shift, max_blocks, num_blocks, splits;   // bs_shift: log2(block_size) or -1
  unsigned unit;                  // tokens that a split is a multiple of
  float scale_log2;
  int* err;
  // packed form: unrotated heads of packed QKV rows; the newest token goes to slots[b]
  const __nv_bfloat16* k_new;
  const __nv_bfloat16* v_new;
  const long long* slots;
  float theta;
  int early;
};

__device__ __forceinline__ void dq_copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void dq_copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void dq_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void dq_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// D(16x8, fp32) += A(16x16, f16, row) B(16x8, f16, col)
__device__ __forceinline__ void dq_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned dq_transpose(unsigned a) {    // an 8 x 8 matrix of f16, a row's pair per lane
  unsigned d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ unsigned dq_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}

// Without a token the sum is 0 and so is the output; a NaN among the scores is one of the output too.
__device__ __forceinline__ __nv_bfloat16 dq_quotient(float o, float l) { return __float2bfloat16(l == 0.f ? 0.f : o / l); }

// The newest token's key (side 0: rotated) or value, in 8 bits: a warp, four elements a lane. Its block's scale is settled as a
// cache write would (a block's first row starts it anew; a larger scale rounds the held rows again), and the row is written;
// a row without a slot has a scale of its own. Returns the four bytes and the scale that they stand in.
template <int FMT>
__device__ __forceinline__ unsigned q8_append_row(const DecodeQ8Params& p, float (&x)[4], int hkv, int side, long long slot, float& now) {
  const int lane = threadIdx.x & 31;
  float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  now = q8_scale_for<FMT>(amax);
  uint8_t* dst = nullptr;
  if (slot >= 0) {
    const long long blk = slot / p.block_size;
    if (blk >= p.num_blocks) {
      if (lane == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    } else {
      const int off = (int)(slot - blk * p.block_size);
      const long long pitch = (long long)p.Hkv * Q8_D;
      uint8_t* rows = p.cache + ((blk * 2 + side) * p.block_size * p.Hkv + hkv) * Q8_D + lane * 4;
      float* sc = p.scale + (blk * 2 + side) * p.Hkv + hkv;
      dst = rows + off * pitch;
      if (off > 0) {
        const float before = *sc;
        if (before < now) {
          const float ratio = before * __frcp_rn(now);
          for (int r = 0; r < p.block_size; ++r) {
            if (r == off) continue;
            unsigned* w = reinterpret_cast<unsigned*>(rows + r * pitch);
            *w = q8_shrink4<FMT>(*w, ratio);
          }
        }
        now = fmaxf(before, now);
      }
      __syncwarp();                // every lane has read the old scale
      if (lane == 0) *sc = now;
    }
  }
  const float inv = __frcp_rn(now);
  const unsigned w = q8_power_of_two(now) ? q8_pack4<FMT>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv) : q8_divide4<FMT>(x[0], x[1], x[2], x[3], now);
  if (dst != nullptr) *reinterpret_cast<unsigned*>(dst) = w;
  return w;
}

// NT: tiles of eight query heads (the group's heads, zero-padded).
// WHOLE: blocks of a multiple of 16 tokens, so that a tile lies in one. W: warps of a CTA.
template <int FMT, int NT, bool ROPE, bool WHOLE, int W>
__global__ void __launch_bounds__(W * 32, NT == 1 ? 12 / W : 2)
paged_decode_q8_kernel(const DecodeQ8Params p, const __grid_constant__ CUtensorMap tm) {
  extern __shared__ __align__(128) uint8_t dq_raw[];
  uint8_t* dq_smem = WHOLE ? dq_raw + (1024 - (smem_u32(dq_raw) & 1023)) % 1024 : dq_raw;      // swizzled boxes start on 1024 bytes
  __shared__ __align__(8) uint64_t s_full[W * DQ_STAGES];
  __shared__ int s_abort;
  __shared__ __align__(16) uint8_t s_new[2][Q8_D];
  __shared__ float s_new_scale[2];
  __shared__ float2 s_cs[ROPE ? Q8_D / 2 : 1];
  // the heads of a sequence run side by side: their 128 bytes of a token are neighbours in memory (4800 CTAs of 900 tokens 246 us with the
  // sequences side by side, 177 so)
  const int b = blockIdx.x / p.Hkv, hkv = blockIdx.x - b * p.Hkv, sp = blockIdx.z;
  pdl_trigger();
  if (WHOLE) {
    if (threadIdx.x == 0) {
      s_abort = 0;
      tma_prefetch_desc(&tm);
    }
    if (threadIdx.x < W * DQ_STAGES) mbar_init(smem_u32(&s_full[threadIdx.x]), 1);
    mbar_fence_init();
    __syncthreads();
  }
  // Lengths, table and cached rows may be read ahead of the kernels before this one where those do not write them.
  const bool early = ROPE && p.early != 0;
  if (!early) pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  int len = p.seq_lens[b];
  const long long cap = (long long)p.max_blocks * p.block_size;
  if (len < 0 || len > cap) {                  // beyond what the table's row can describe: clamped and reported
    if (tid == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    len = len < 0 ? 0 : (int)cap;
  }
  // a split is a whole number of blocks, so that a block whose scale grows with its newest row is read by one CTA alone
  // (a unit is below 2^31, and a split behind the last token may begin beyond 2^32)
  const unsigned per = ((unsigned)(len + p.splits - 1) / (unsigned)p.splits + p.unit - 1) / p.unit * p.unit;
  const int t_lo = (int)min((unsigned long long)len, (unsigned long long)sp * per), t_hi = (int)min((unsigned)len, (unsigned)t_lo + per);
  float* ws = p.ws ? p.ws + (((long long)b * p.Hkv + hkv) * p.splits + sp) * p.G * DQ_RED : nullptr;
  // behind the warps' partial results in shared memory: this CTA's, for the others of its cluster
  float* mine_out = reinterpret_cast<float*>(dq_smem) + W * p.G * DQ_RED;
  // The splits of a sequence and KV head are the CTAs of a cluster: each merges a part of the output from all of them.
  auto merge_cluster = [&]() {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    for (int i = sp * (W * 32) + tid; i < p.G * Q8_D; i += p.splits * (W * 32)) {
      const int at = i / Q8_D * DQ_RED, d = i % Q8_D;
      float m[DQ_CLUSTER], M = -INFINITY, L = 0.f, acc = 0.f;
#pragma unroll
      for (int q = 0; q < DQ_CLUSTER; ++q) {
        m[q] = q < p.splits ? cl.map_shared_rank(mine_out, q)[at] : -INFINITY;
        M = fmaxf(M, m[q]);
      }
      const float M_use = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int q = 0; q < DQ_CLUSTER; ++q)
        if (q < p.splits) {
          const float* r = cl.map_shared_rank(mine_out, q) + at;
          const float f = exp2f(m[q] - M_use);
          L += f * r[1];
          acc += f * r[2 + d];
        }
      p.out[((long long)b * p.Hq + hkv * p.G) * Q8_D + i] = dq_quotient(acc, L);
    }
    cl.sync();                                 // nobody leaves while its results are read
  };
  if (t_lo >= t_hi) {
    if (early) pdl_wait();
    if (ws) {
      for (int i = tid; i < p.G * DQ_RED; i += (W * 32)) ws[i] = i % DQ_RED == 0 ? -INFINITY : 0.f;
    } else if (p.splits > 1) {
      for (int i = tid; i < p.G * DQ_RED; i += (W * 32)) mine_out[i] = i % DQ_RED == 0 ? -INFINITY : 0.f;
      merge_cluster();
    } else {
      for (int i = tid; i < p.G * Q8_D; i += (W * 32)) p.out[((long long)b * p.Hq + hkv * p.G) * Q8_D + i] = __float2bfloat16(0.f);
    }
    return;
  }
  const int* bt = p.block_table + (long long)b * p.max_blocks;
  const long long v_off = (long long)p.block_size * p.Hkv * Q8_D, blk_bytes = 2 * v_off;
  constexpr int SPAN = DQ_PAIR * DQ_TILE;
  const int pairs = (t_hi - t_lo + SPAN - 1) / SPAN;
  const int mine = pairs > warp ? (pairs - warp + W - 1) / W : 0;      // pairs of tiles warp, warp + 4, ...
  constexpr int STAGE = WHOLE ? DQ_BOX_STAGE : DQ_STAGE_BYTES, TILE_BYTES = STAGE / DQ_PAIR;
  uint8_t* ring_p = dq_smem + warp * DQ_STAGES * STAGE;
  const uint32_t ring = smem_u32(ring_p), full = smem_u32(&s_full[warp * DQ_STAGES]);
  const bool has_new = ROPE && t_hi == len;
  // tiles that reach into the newest token's block wait until that token is written
  const int held_back = has_new ? (len - 1) / p.block_size * p.block_size : 0x7fffffff;

  const long long row_bytes = (long long)p.Hkv * Q8_D;
  auto block_of = [&](int t) { return p.bs_shift >= 0 ? t >> p.bs_shift : t / p.block_size; };
  auto checked = [&](int page) {
    if (page >= 0 && page < p.num_blocks) return page;
    atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return 0;
  };
  // WHOLE: the blocks of 16 pairs of tiles of this warp and their scales, a tile a lane; scales of the 16 pairs before stay in use for a while
  int pages = 0, pages_from = -1;
  float scales[2][2];
  scales[0][0] = scales[0][1] = scales[1][0] = scales[1][1] = 1.f;
  auto issue = [&](int i) {                    // this warp's i-th pair
    const int first = t_lo + (warp + i * W) * SPAN;
    const uint32_t st = ring + (i % DQ_STAGES) * STAGE;
    if constexpr (WHOLE) {
      if ((i & ~15) != pages_from) {
        pages_from = i & ~15;
        const int t = t_lo + (warp + (pages_from + (lane >> 1)) * W) * SPAN + (lane & 1) * DQ_TILE;
        pages = t < t_hi ? checked(bt[block_of(t)]) : 0;
        const float* sc = p.scale + (long long)pages * 2 * p.Hkv + hkv;
        const float sk = t < t_hi ? sc[0] : 1.f, sv = t < t_hi ? sc[p.Hkv] : 1.f;
        if ((i >> 4) & 1) { scales[1][0] = sk; scales[1][1] = sv; }
        else { scales[0][0] = sk; scales[0][1] = sv; }
      }
      const int page0 = __shfl_sync(0xffffffffu, pages, 2 * (i & 15)), page1 = __shfl_sync(0xffffffffu, pages, 2 * (i & 15) + 1);
      if (elect_one()) {
        const uint32_t bar = full + 8 * (i % DQ_STAGES);
        const bool two = first + DQ_TILE < t_hi;
        mbar_expect_tx(bar, two ? STAGE : TILE_BYTES);
#pragma unroll
        for (int h = 0; h < DQ_PAIR; ++h) {
          if (h == 1 && !two) break;
          const int t0 = first + h * DQ_TILE, row = (h ? page1 : page0) * 2 * p.block_size + t0 - block_of(t0) * p.block_size;
          tma_load_2d(st + h * TILE_BYTES, &tm, hkv * Q8_D, row, bar);
          tma_load_2d(st + h * TILE_BYTES + DQ_TILE * Q8_D, &tm, hkv * Q8_D, row + p.block_size, bar);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < DQ_PAIR; ++h) {
        const uint32_t to = st + h * TILE_BYTES;
        const int t = first + h * DQ_TILE + (lane & 15), tt = t < t_hi ? t : t_lo;
        const int blk = block_of(tt), at = t < t_hi ? t - blk * p.block_size : -1;
        const int page = checked(bt[blk]);
        dq_copy4(to + 2 * DQ_TILE * Q8_D + lane * 4, p.scale + ((long long)page * 2 + (lane >> 4)) * p.Hkv + hkv, at >= 0 ? 4 : 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {            // rows g and g + 8 of the keys, 16-byte columns 2c and 2c + 1
          const int pg = __shfl_sync(0xffffffffu, page, g + 8 * j), r = __shfl_sync(0xffffffffu, at, g + 8 * j);
          const uint8_t* src = p.cache + pg * blk_bytes + max(r, 0) * row_bytes + hkv * Q8_D + c * 32;
          dq_copy16(to + (j * 2) * 512 + lane * 16, src, r >= 0 ? 16 : 0);
          dq_copy16(to + (j * 2 + 1) * 512 + lane * 16, src + 16, r >= 0 ? 16 : 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {            // rows 2c, 2c + 1, 2c + 8, 2c + 9 of the values, column g
          const int tr = 2 * c + (j & 1) + 8 * (j >> 1);
          const int pg = __shfl_sync(0xffffffffu, page, tr), r = __shfl_sync(0xffffffffu, at, tr);
          dq_copy16(to + DQ_TILE * Q8_D + j * 512 + lane * 16, p.cache + pg * blk_bytes + v_off + max(r, 0) * row_bytes + hkv * Q8_D + g * 16, r >= 0 ? 16 : 0);
        }
      }
    }
  };
  // where this lane's 16 bytes lie in a tile: keys, half 0 / 1 of its columns in row g + 8 j; values, the j-th of its rows
  auto key_at = [&](int half, int j) {
    return WHOLE ? (g + 8 * j) * Q8_D + (((2 * c + half) ^ g) << 4) : (2 * j + half) * 512 + lane * 16;
  };
  auto value_at = [&](int j) {
    const int row = 2 * c + (j & 1) + 8 * (j >> 1);
    return DQ_TILE * Q8_D + (WHOLE ? row * Q8_D + ((g ^ (row & 7)) << 4) : j * 512 + lane * 16);
  };
  auto late = [&](int i) { return has_new && t_lo + (warp + i * W) * SPAN + SPAN > held_back; };
#pragma unroll
  for (int i = 0; i < DQ_STAGES; ++i) {
    if (i < mine && !late(i)) issue(i);
    if (!WHOLE) dq_commit();
  }
  if (ROPE) {
    if (tid < Q8_D / 2) s_cs[tid] = rope_cos_sin((float)(len - 1), __logf(p.theta), rope_exponent<Q8_D>(tid));
    __syncthreads();
  }
  if (early) pdl_wait();
  long long slot = -1;
  if (has_new) {
    slot = p.slots[b];
    if (warp < 2) {
      const __nv_bfloat16* src = (warp ? p.v_new : p.k_new) + (long long)b * p.ldq + (long long)hkv * Q8_D + lane * 4;
      const uint2 own = *reinterpret_cast<const uint2*>(src);
      float2 u = unpack_bf16x2(own.x), v = unpack_bf16x2(own.y);
      float x[4] = {u.x, u.y, v.x, v.y};
      if (warp == 0) {                         // rotated and rounded to bf16, as a cache write takes it
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float other = __shfl_xor_sync(0xffffffffu, x[j], 16);
          float lo = lane < 16 ? x[j] : other, hi = lane < 16 ? other : x[j];
          rope_rotate(lo, hi, s_cs[(lane & 15) * 4 + j]);
          x[j] = __bfloat162float(__float2bfloat16(lane < 16 ? lo : hi));
        }
      }
      float now;
      const unsigned w = q8_append_row<FMT>(p, x, hkv, warp, slot, now);
      *reinterpret_cast<unsigned*>(&s_new[warp][lane * 4]) = w;
      if (lane == 0) s_new_scale[warp] = now;
      __threadfence();                         // the copies below read past the L1, or through TMA
      if (WHOLE) fence_proxy_async_all();
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DQ_STAGES; ++i)
      if (i < mine && late(i)) issue(i);
    if (!WHOLE) dq_commit();
  }

  // Q^T as the B operand: head n = g of each tile of eight, the 32 elements that this lane's pieces of a key row hold
  unsigned qb[NT][8][2];
  float qf[NT][2];                             // of heads 2c and 2c + 1: power of two taken out, softmax scale, log2 e
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int head = n * 8 + g;
    float x[32];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // rows are 4-byte aligned at least
        float2 a = make_float2(0.f, 0.f), e = a;
        if (head < p.G) {
          const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + (long long)b * p.ldq + (long long)(hkv * p.G + head) * Q8_D + c * 32 + h * 16 + j * 4);
          a = unpack_bf16x2(src[0]);
          e = unpack_bf16x2(src[1]);
        }
        x[h * 16 + j * 4] = a.x; x[h * 16 + j * 4 + 1] = a.y; x[h * 16 + j * 4 + 2] = e.x; x[h * 16 + j * 4 + 3] = e.y;
      }
    if (ROPE) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {           // the pair of column 32 c + j is 64 further, two lanes of the four on
        const float other = __shfl_xor_sync(0xffffffffu, x[j], 2);
        float lo = c < 2 ? x[j] : other, hi = c < 2 ? other : x[j];
        rope_rotate(lo, hi, s_cs[(c & 1) * 32 + j]);
        x[j] = __bfloat162float(__float2bfloat16(c < 2 ? lo : hi));
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) amax = fmaxf(amax, fabsf(x[j]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    int e = (int)(__float_as_uint(amax) >> 23) - 127;          // largest element in [2^e, 2^(e+1))
    e = max(-100, min(120, e));
    const float up = __uint_as_float((unsigned)(127 + 7 - e) << 23), down = __uint_as_float((unsigned)(127 - 7 + e) << 23);
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      qb[n][ks][0] = dq_half2(x[ks * 4] * up, x[ks * 4 + 1] * up);
      qb[n][ks][1] = dq_half2(x[ks * 4 + 2] * up, x[ks * 4 + 3] * up);
    }
    qf[n][0] = __shfl_sync(0xffffffffu, down, 8 * c) * p.scale_log2;         // the lane of head 2c, then of 2c + 1
    qf[n][1] = __shfl_sync(0xffffffffu, down, 8 * c + 4) * p.scale_log2;
  }

  float o[NT][8][4];
  float m_run[NT][2], m_use[NT][2], l_run[NT][2];   // of heads 2c, 2c + 1: maximum, what weights are relative to, sum (of this lane's tokens)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int mt = 0; mt < 8; ++mt) o[n][mt][0] = o[n][mt][1] = o[n][mt][2] = o[n][mt][3] = 0.f;
    m_run[n][0] = m_run[n][1] = -INFINITY;
    m_use[n][0] = m_use[n][1] = l_run[n][0] = l_run[n][1] = 0.f;
  }

  for (int i = 0; i < mine; ++i) {
    if (WHOLE) {
      if (!mbar_wait_warp(full + 8 * (i % DQ_STAGES), (i / DQ_STAGES) & 1, &s_abort, p.err, ERR_WAIT_ATTN)) break;
    } else {
      if (has_new && late(i)) dq_wait<0>();    // its group is not the i-th one
      else dq_wait<DQ_STAGES - 1>();
      __syncwarp();                            // the scales are other lanes' copies
    }
    uint8_t* stage = ring_p + (i % DQ_STAGES) * STAGE;
    // two tiles side by side: the products of one hide the latencies of the other's
    float s[DQ_PAIR][NT][4], iv[DQ_PAIR][2];
    float ks[DQ_PAIR][2], lv[DQ_PAIR][2];
    bool in[DQ_PAIR][2];
#pragma unroll
    for (int h = 0; h < DQ_PAIR; ++h) {
      uint8_t* st = stage + h * TILE_BYTES;
      const int t0 = t_lo + (warp + i * W) * SPAN + h * DQ_TILE;
      float vs[2];
      if (WHOLE) {
        const bool odd = (i >> 4) & 1;
        ks[h][0] = __shfl_sync(0xffffffffu, odd ? scales[1][0] : scales[0][0], 2 * (i & 15) + h);
        vs[0] = __shfl_sync(0xffffffffu, odd ? scales[1][1] : scales[0][1], 2 * (i & 15) + h);
        if (has_new && late(i) && t0 < t_hi) {                 // as the newest token left them
          const float* sc = p.scale + (long long)checked(bt[block_of(t0)]) * 2 * p.Hkv + hkv;
          ks[h][0] = sc[0];
          vs[0] = sc[p.Hkv];
        }
        ks[h][1] = ks[h][0];
        vs[1] = vs[0];
      } else {
        const float* sc = reinterpret_cast<const float*>(st + 2 * DQ_TILE * Q8_D);
        ks[h][0] = sc[g]; ks[h][1] = sc[g + 8];
        vs[0] = sc[16 + g]; vs[1] = sc[16 + g + 8];
      }
      if (ROPE && slot < 0 && has_new && len - 1 >= t0 && len - 1 < t0 + DQ_TILE) {   // a newest token that is nowhere in the cache
        const int r = len - 1 - t0;
        if ((r & 7) == g) {
          *reinterpret_cast<uint4*>(st + key_at(0, r >> 3)) = *reinterpret_cast<const uint4*>(&s_new[0][c * 32]);
          *reinterpret_cast<uint4*>(st + key_at(1, r >> 3)) = *reinterpret_cast<const uint4*>(&s_new[0][c * 32 + 16]);
          if (r < 8) { ks[h][0] = s_new_scale[0]; vs[0] = s_new_scale[1]; }
          else { ks[h][1] = s_new_scale[0]; vs[1] = s_new_scale[1]; }
        }
        if (((r & 7) >> 1) == c) *reinterpret_cast<uint4*>(st + value_at((r & 1) + 2 * (r >> 3))) = *reinterpret_cast<const uint4*>(&s_new[1][g * 16]);
        if (WHOLE) fence_proxy_async_smem();   // before the next box lands here
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        in[h][e] = t0 + g + 8 * e < t_hi;
        // a block of zeros (or one that was never written) may have any scale: 2^-60 stands for what is smaller
        vs[e] = fminf(fmaxf(vs[e], 8.6736174e-19f), 1.1529215e18f);
        lv[h][e] = __log2f(vs[e]);
        iv[h][e] = __fdividef(1.f, vs[e]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)       // 64 of the key's 128 columns
#pragma unroll
      for (int h = 0; h < DQ_PAIR; ++h) {
        const uint8_t* st = stage + h * TILE_BYTES;
        const uint4 a = *reinterpret_cast<const uint4*>(st + key_at(half, 0)), e = *reinterpret_cast<const uint4*>(st + key_at(half, 1));
        const unsigned aw[4] = {a.x, a.y, a.z, a.w}, ew[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          unsigned a0, a2, a1, a3;
          q8_unpack4<FMT>(aw[j], a0, a2);
          q8_unpack4<FMT>(ew[j], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) dq_mma(s[h][n], a0, a1, a2, a3, qb[n][half * 4 + j][0], qb[n][half * 4 + j][1]);
        }
      }
    unsigned pb[DQ_PAIR][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int h = 0; h < DQ_PAIR; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {          // tokens g (0, 1) and g + 8 (2, 3), heads 2c and 2c + 1
          s[h][n][e] = in[h][e >> 1] ? fmaf(s[h][n][e] * qf[n][e & 1], ks[h][e >> 1], lv[h][e >> 1]) : -INFINITY;
          mx[e & 1] = fmaxf(mx[e & 1], s[h][n][e]);
        }
      // a new maximum is met in few tiles: only then are the lanes asked for theirs and the sums brought to it
      if (__any_sync(0xffffffffu, mx[0] > m_run[n][0] || mx[1] > m_run[n][1])) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
          const float m_new = fmaxf(m_run[n][e], mx[e]);
          m_use[n][e] = m_new == -INFINITY ? 0.f : m_new - DQ_UP;
          alpha[e] = exp2f(m_run[n][e] - DQ_UP - m_use[n][e]);
          m_run[n][e] = m_new;
          l_run[n][e] *= alpha[e];
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          o[n][mt][0] *= alpha[0]; o[n][mt][1] *= alpha[1];
          o[n][mt][2] *= alpha[0]; o[n][mt][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int h = 0; h < DQ_PAIR; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][n][e] = exp2f(s[h][n][e] - m_use[n][e & 1]);
          l_run[n][e & 1] += s[h][n][e] * iv[h][e >> 1];
        }
        // rows are tokens here and columns in the next product
        pb[h][n][0] = dq_transpose(dq_half2(s[h][n][0], s[h][n][1]));
        pb[h][n][1] = dq_transpose(dq_half2(s[h][n][2], s[h][n][3]));
      }
    }
#pragma unroll
    for (int h = 0; h < DQ_PAIR; ++h) {
      const uint8_t* st = stage + h * TILE_BYTES;
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(st + value_at(j));
      const int left = t_hi - (t_lo + (warp + i * W) * SPAN + h * DQ_TILE);
      if (WHOLE && left < DQ_TILE) {           // rows behind the sequence hold anything, and 0 times a NaN is one
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (2 * c + (j & 1) + 8 * (j >> 1) >= left) v[j] = make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {            // rows 16 g + 4 j .. + 3 of O^T
        const unsigned t0w = (&v[0].x)[j], t1w = (&v[1].x)[j], t8w = (&v[2].x)[j], t9w = (&v[3].x)[j];
#pragma unroll
        for (int q = 0; q < 2; ++q) {          // two tokens' bytes side by side: rows 4 j + 2 q, 4 j + 2 q + 1
          unsigned a0, a1, a2, a3;
          q8_unpack4<FMT>(__byte_perm(t0w, t1w, q ? 0x7362 : 0x5140), a0, a1);
          q8_unpack4<FMT>(__byte_perm(t8w, t9w, q ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) dq_mma(o[n][j * 2 + q], a0, a1, a2, a3, pb[h][n][0], pb[h][n][1]);
        }
      }
    }
    __syncwarp();                              // this stage has been read
    if (i + DQ_STAGES < mine) issue(i + DQ_STAGES);
    if (!WHOLE) dq_commit();
  }
  if (!WHOLE) dq_wait<0>();
  __syncthreads();                             // the rings are free
  if (WHOLE && s_abort) {                      // a wait ran out: boxes still under way get time to land first
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) __nanosleep(1000);
    __syncthreads();
  }
  // ---- merge the four warps: red[warp][head][m, l, o[128]]
  float* red = reinterpret_cast<float*>(dq_smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[n][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int head = n * 8 + 2 * c + e;
      if (head < p.G) {
        float* r = red + ((long long)warp * p.G + head) * DQ_RED;
        if (g == 0) { r[0] = m_run[n][e]; r[1] = l; }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt) {
          r[2 + g * 16 + 2 * mt] = o[n][mt][e];
          r[2 + g * 16 + 2 * mt + 1] = o[n][mt][2 + e];
        }
      }
    }
  __syncthreads();
  for (int i = tid; i < p.G * Q8_D; i += (W * 32)) {
    const int h = i / Q8_D, d = i % Q8_D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, red[(w * p.G + h) * DQ_RED]);
    const float M_use = M == -INFINITY ? 0.f : M;
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* r = red + (w * p.G + h) * DQ_RED;
      const float f = exp2f(r[0] - M_use);     // a warp without tokens has m = -inf, l = 0, o = 0
      acc += f * r[2 + d];
      l += f * r[1];
    }
    if (p.splits > 1) {
      float* to = (ws ? ws : mine_out) + h * DQ_RED;
      to[2 + d] = acc;
      if (d == 0) { to[0] = M; to[1] = l; }
    } else {
      p.out[((long long)b * p.Hq + hkv * p.G + h) * Q8_D + d] = dq_quotient(acc, l);
    }
  }
  if (p.splits > 1 && ws == nullptr) merge_cluster();
}
static_assert((2 + 1) * 8 * DQ_RED * 4 <= 2 * DQ_STAGES * DQ_BOX_STAGE && (DQ_WARPS + 1) * 16 * DQ_RED * 4 <= DQ_WARPS * DQ_STAGES * DQ_BOX_STAGE,
              "partial results of 8 heads (of 16: four warps) fit the rings");

// out = sum_s exp2(m_s - M) o_s / sum_s exp2(m_s - M) l_s over the splits of a sequence and head. The splits' factors first, one a
// thread, so that the loop over their outputs has nothing but loads in it, eight at a time.
__global__ void __launch_bounds__(Q8_D)
paged_decode_q8_merge_kernel(const float* ws, __nv_bfloat16* out, int Hq, int Hkv, int G, int splits) {
  __shared__ float s_f[Q8_D], s_max[Q8_D / 32], s_sum[Q8_D / 32];
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x / Hq, h = blockIdx.x % Hq, d = threadIdx.x;
  const float* base = ws + (((long long)b * Hkv + h / G) * splits * G + h % G) * DQ_RED;
  const long long sstride = (long long)G * DQ_RED;
  float M = -INFINITY, L = 0.f, o = 0.f;       // relative to the maximum so far
  for (int s0 = 0; s0 < splits; s0 += Q8_D) {
    const int n = min(Q8_D, splits - s0);
    const float m = d < n ? base[(s0 + d) * sstride] : -INFINITY, l = d < n ? base[(s0 + d) * sstride + 1] : 0.f;
    float mx = m;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
    __syncthreads();
    if ((d & 31) == 0) s_max[d >> 5] = mx;
    __syncthreads();
    const float M_new = fmaxf(fmaxf(M, fmaxf(s_max[0], s_max[1])), fmaxf(s_max[2], s_max[3]));
    const float M_use = M_new == -INFINITY ? 0.f : M_new, back = exp2f(M - M_use), f = exp2f(m - M_use);
    float sum = f * l;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if ((d & 31) == 0) s_sum[d >> 5] = sum;
    s_f[d] = f;
    __syncthreads();
    L = L * back + (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    o *= back;
    M = M_new;
    const float* at = base + s0 * sstride + 2 + d;
    int s = 0;
    for (; s + 8 <= n; s += 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = at[(s + k) * sstride];
#pragma unroll
      for (int k = 0; k < 8; ++k) o += s_f[s + k] * x[k];
    }
    for (; s < n; ++s) o += s_f[s] * at[s * sstride];
  }
  out[(long long)blockIdx.x * Q8_D + d] = dq_quotient(o, L);
}
static_assert(Q8_D == 128, "four warps");

}  // namespace mlf

using namespace mlf;

// One query token per sequence over an 8-bit cache. Without slots: q [B, Hq, 128], row pitch ldq. With slots (the packed form): q is
// the QKV product [B, (Hq + 2 Hkv) * 128], not yet rotated; the newest token of a sequence, the last of its seq_lens, is rotated at
// position seq_lens - 1, written to its slot (< 0: not written) as mlf_kv_write_q8 would and attended to like the cached ones.
// max_seq_len: an upper bound of seq_lens, for the launch's shape alone. fmt: 0 e4m3, 1 int8. ws: B * Hq * splits * 130 floats (ws_elems: what is there) for splits that a second kernel merges; without it
// up to 8 are merged by clusters of the launch, which is faster where all of them are resident at once (a 4-split launch of 24 x
// 900 tokens of 40 heads, nine rounds: 67 us, 49 with ws). inputs_static: as for mlf_paged_decode_rope.
MLF_API int mlf_paged_decode_q8(const void* q, long long ldq, void* cache, float* scale, int fmt, const int* block_table, const int* seq_lens,
                                const long long* slots, void* out, float* ws, long long ws_elems, int B, int Hq, int Hkv, int block_size, int max_blocks,
                                int num_blocks, int max_seq_len, int splits, float softmax_scale, float theta, int inputs_static, uint64_t stream) {
  if (B <= 0) return 0;
  MLF_REQUIRE(fmt == Q8_E4M3 || fmt == Q8_INT8, "paged_decode_q8: format %d", fmt);
  MLF_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "paged_decode_q8: bad head counts %d, %d", Hq, Hkv);
  const int G = Hq / Hkv;
  MLF_REQUIRE(G <= 16, "paged_decode_q8: group size %d not supported (1 to 16)", G);
  MLF_REQUIRE(block_size > 0 && max_blocks > 0 && num_blocks > 0 && splits > 0, "paged_decode_q8: bad sizes");
  MLF_REQUIRE((long long)max_blocks * block_size < (1LL << 31) - (1 << 20), "paged_decode_q8: block table of %d x %d tokens", max_blocks, block_size);
  MLF_REQUIRE((long long)B * Hq < (1LL << 31) && splits <= 65535, "paged_decode_q8: grid");
  MLF_REQUIRE((splits <= DQ_CLUSTER && ws == nullptr) || (ws != nullptr && ws_elems >= (long long)B * Hq * splits * DQ_RED), "paged_decode_q8: workspace too small for %d splits", splits);
  MLF_REQUIRE((reinterpret_cast<uintptr_t>(cache) & 15) == 0, "paged_decode_q8: the cache must be 16-byte aligned");
  const bool rope = slots != nullptr;
  MLF_REQUIRE(rope ? ldq % 4 == 0 && (reinterpret_cast<uintptr_t>(q) & 7) == 0 && theta > 0.f : ldq % 2 == 0 && (reinterpret_cast<uintptr_t>(q) & 3) == 0,
              "paged_decode_q8: query rows must be %d-byte aligned", rope ? 8 : 4);
  DecodeQ8Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.ldq = ldq;
  p.cache = static_cast<uint8_t*>(cache);
  p.scale = scale;
  p.block_table = block_table; p.seq_lens = seq_lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  const bool second = splits > 1 && ws != nullptr;     // a kernel of its own merges the splits
  p.ws = second ? ws : nullptr;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.block_size = block_size; p.max_blocks = max_blocks; p.num_blocks = num_blocks;
  p.splits = splits;
  p.unit = block_size * ((64 + block_size - 1) / block_size);
  p.bs_shift = -1;
  for (int sh = 0; sh < 31; ++sh) if ((1 << sh) == block_size) p.bs_shift = sh;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.err = device_status_word();
  p.k_new = rope ? p.q + (long long)Hq * Q8_D : nullptr;
  p.v_new = rope ? p.k_new + (long long)Hkv * Q8_D : nullptr;
  p.slots = slots;
  p.theta = theta;
  p.early = inputs_static;
  const long long cache_rows = 2LL * num_blocks * block_size;
  const bool whole = block_size % DQ_TILE == 0 && cache_rows < (1LL << 31);
  // Warps of a CTA (a warp's ring is 16 KB): three CTAs of four fit an SM, four of three, six of two. With up to eight heads the form whose
  // rounds have the fewest places; of equal ones, and for short sequences in more than a round, the one with the fewest warps. us
  // with 4 / 3 / 2 warps (places an SM in brackets): 480 CTAs of 900 tokens 31 / 24 / 31 (6, 4, 6), 720 37 / 43 / 34 (6, 8, 6), 960 47 /
  // 46 / 54 (9, 8, 12), 1280 55 / 63 / 62 (9, 12, 12), 1600 69 / 68 / 66 (12, 12, 12), 2000 83 / 87 / 90 (15, 16, 18); 1280 of 300 30 / 30
  // / 28, 2000 of 300 46 / 41 / 39, 4800 of 300 92 / 80 / 74.
  const long long ctas = (long long)B * Hkv * splits, sms = sm_count();
  auto places = [&](int per_sm) { return (ctas + sms * per_sm - 1) / (sms * per_sm) * per_sm; };
  int warps = 4;
  if (whole && G <= 8) {
    if (places(4) <= places(3)) warps = 3;
    if (places(6) <= places(7 - warps) || (ctas > 6 * sms && max_seq_len <= 400LL * splits)) warps = 2;
  }
  const int smem = whole ? dq_box_smem(warps) : DQ_SMEM;
  CUtensorMap tm = {};
  if (whole) {
    const int rc = make_tmap_2d(&tm, cache, 1, (uint64_t)Hkv * Q8_D, (uint64_t)cache_rows, (uint64_t)Hkv * Q8_D, Q8_D, DQ_TILE, true);
    if (rc) return rc;
  }
#define DQ_ROPE(FMT, NT, WHOLE, W) {paged_decode_q8_kernel<FMT, NT, false, WHOLE, W>, paged_decode_q8_kernel<FMT, NT, true, WHOLE, W>}
#define DQ_KERNELS(FMT) {DQ_ROPE(FMT, 1, false, 4), DQ_ROPE(FMT, 2, false, 4), DQ_ROPE(FMT, 2, true, 4), DQ_ROPE(FMT, 1, true, 4), DQ_ROPE(FMT, 1, true, 3), DQ_ROPE(FMT, 1, true, 2)}
  void (*const kernels[2][6][2])(DecodeQ8Params, CUtensorMap) = {DQ_KERNELS(Q8_E4M3), DQ_KERNELS(Q8_INT8)};
#undef DQ_KERNELS
#undef DQ_ROPE
  const int form = !whole ? (G > 8 ? 1 : 0) : G > 8 ? 2 : 7 - warps;
  const auto kernel = kernels[fmt][form][rope ? 1 : 0];
  static bool attr_set[64][24] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  bool& set = attr_set[dev & 63][(fmt * 6 + form) * 2 + (rope ? 1 : 0)];
  if (!set) {
    MLF_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    set = true;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  MLF_CHECK_CUDA(launch_pdl_cluster(kernel, dim3((unsigned)(B * Hkv), 1, splits), dim3(warps * 32), smem, dim3(1, 1, second ? 1 : splits), st, p, tm));
  count_launch();
  if (second) {
    MLF_CHECK_CUDA(launch_pdl(paged_decode_q8_merge_kernel, dim3((unsigned)(B * Hq)), dim3(Q8_D), 0, st, (const float*)ws, p.out, Hq, Hkv, G, splits));
    count_launch();
  }
  return 0;
}
