// Writes to a paged 8-bit cache and the way back to bf16 (layout and scales: kv_q8.cuh).
//
// A block and head has one scale, so the rows of a call that fall into one block belong together: one warp takes a block's rows of
// one head and side, finds their largest magnitude, settles the scale and rounds. A call that writes a block's first row starts
// the block anew; otherwise the scale is the larger of the old one and the new rows' own, and where it grows the rows that the
// block held are rounded to it. Which rows of a block a call writes: up to 256 tokens, a warp looks through all their slots. For more,
// q8_map_kernel notes for each slot which token goes there; the map is read back only where the slot it stands at names the same
// token, so that it needs no clearing: entries of earlier calls, or of nothing at all, point at tokens of other slots.
//
// Bound by HBM in long calls (a row is read in 16 bits and written in 8), by the chain of loads slots - map - slots - rows in short ones.
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../mlf_api.h"
#include "kv_q8.cuh"

namespace mlf {

constexpr int QW_WARPS = 8;
constexpr int QW_GROUP = 16;                  // tokens whose blocks a CTA looks at: in a prompt's order about one block
constexpr int QW_FEW = 256;                   // tokens that need no map

struct Q8WriteParams {
  uint8_t* cache;
  float* scale;
  const __nv_bfloat16 *k, *v;
  const long long* slots;
  int* map;                                   // [num_blocks * block_size], null up to QW_FEW tokens
  long long T, ldk, ldv;
  int Hkv, block_size, num_blocks, group;
  int* err;
};

__global__ void __launch_bounds__(256) q8_map_kernel(const Q8WriteParams p) {
  pdl_trigger();
  pdl_wait();
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t >= p.T) return;
  const long long slot = p.slots[t];
  if (slot < 0) return;
  if (slot >= (long long)p.num_blocks * p.block_size) {
    atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return;
  }
  p.map[slot] = (int)t;                       // a slot that is given twice keeps one of its tokens
}

// Lanes 0 .. 15: the token that this call writes to slot first + lane, the lowest of them without a map, or -1 (also for the
// `count` rows' end). `found`: 16 ints of this warp.
__device__ __forceinline__ int q8_tokens_at(const Q8WriteParams& p, long long first, int count, int* found) {
  const int lane = threadIdx.x & 31;
  if (p.map != nullptr) {
    if (lane >= count) return -1;
    const int t = p.map[first + lane];
    return t >= 0 && t < p.T && p.slots[t] == first + lane ? t : -1;
  }
  __syncwarp();
  if (lane < 16) found[lane] = 0x7fffffff;
  __syncwarp();
  for (int t = lane; t < p.T; t += 32) {
    const long long at = p.slots[t] - first;
    if (at >= 0 && at < count) atomicMin(&found[at], t);
  }
  __syncwarp();
  const int t = lane < count ? found[lane] : 0x7fffffff;
  return t == 0x7fffffff ? -1 : t;
}

// known: the tokens of the block's first 16 rows, by row
template <int FMT>
__device__ __forceinline__ void q8_write_rows(const Q8WriteParams& p, int blk, int h, int side, const int* known, int* found) {
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const long long first = (long long)blk * p.block_size;
  const __nv_bfloat16* src = (side ? p.v : p.k) + (long long)h * Q8_D + col;
  const long long ld = side ? p.ldv : p.ldk;
  uint8_t* dst = p.cache + (((long long)blk * 2 + side) * p.block_size * p.Hkv + h) * Q8_D + col;
  float* scale = p.scale + ((long long)blk * 2 + side) * p.Hkv + h;
  const int chunks = (p.block_size + 15) / 16;
  uint4 x[8];
  int tok = -1;                               // lanes 0..15: the token of row chunk * 16 + lane
  auto load = [&](int c) {
    tok = c == 0 ? (lane < 16 ? known[lane] : -1) : q8_tokens_at(p, first + c * 16, min(16, p.block_size - c * 16), found);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = __shfl_sync(0xffffffffu, tok, 2 * i + half);
      x[i] = t >= 0 ? *reinterpret_cast<const uint4*>(src + t * ld) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const float held_scale = *scale;
  float amax = 0.f;
  bool anew = false;
  for (int c = 0; c < chunks; ++c) {
    load(c);
    if (c == 0) anew = __shfl_sync(0xffffffffu, tok, 0) >= 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack_bf16x2(w[j]);
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const float fit = q8_scale_for<FMT>(amax), before = anew ? 0.f : held_scale;
  const float now = fmaxf(before, fit);
  const float inv = __frcp_rn(now), ratio = before * inv;     // exact for powers of two
  const bool shrink = !anew && before < now;
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = c * 16 + 2 * i + half;
      const int t = __shfl_sync(0xffffffffu, tok, 2 * i + half);
      if (row >= p.block_size) continue;
      uint2* to = reinterpret_cast<uint2*>(dst + (long long)row * p.Hkv * Q8_D);
      if (t >= 0) {
        const float2 a = unpack_bf16x2(x[i].x), b = unpack_bf16x2(x[i].y), e = unpack_bf16x2(x[i].z), f = unpack_bf16x2(x[i].w);
        *to = make_uint2(q8_pack4<FMT>(a.x * inv, a.y * inv, b.x * inv, b.y * inv), q8_pack4<FMT>(e.x * inv, e.y * inv, f.x * inv, f.y * inv));
      } else if (shrink) {
        const uint2 held = *to;
        *to = make_uint2(q8_shrink4<FMT>(held.x, ratio), q8_shrink4<FMT>(held.y, ratio));
      }
    }
  }
  if (lane == 0) *scale = now;
}

// A CTA finds, among `group` tokens, those that are the first of their block's rows in this call, and writes those blocks; the
// heads and sides are split over blockIdx.y.
template <int FMT>
__global__ void __launch_bounds__(QW_WARPS * 32) q8_write_kernel(const Q8WriteParams p) {
  __shared__ int s_blk[QW_GROUP], s_tok[QW_GROUP][16], s_found[QW_WARPS][16];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < p.group; i += QW_WARPS) {
    const long long t = (long long)blockIdx.x * p.group + i;
    int blk = -1, tok = -1;
    if (t < p.T) {
      const long long slot = p.slots[t];
      if (slot >= (long long)p.num_blocks * p.block_size) {
        if (p.map == nullptr && lane == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
      } else if (slot >= 0) {
        blk = (int)(slot / p.block_size);
        // this token takes the block if it is the first, by row, of those that the call writes there
        const int off = (int)(slot - (long long)blk * p.block_size);
        const long long first = (long long)blk * p.block_size;
        for (int c = 0; c * 16 <= off && blk >= 0; ++c) {
          const int at = q8_tokens_at(p, first + c * 16, min(16, p.block_size - c * 16), s_found[warp]);
          if (c == 0) tok = at;
          const unsigned there = __ballot_sync(0xffffffffu, at >= 0);
          if (there != 0) {
            const int row = __ffs(there) - 1;
            if (c * 16 + row != off || __shfl_sync(0xffffffffu, at, row) != (int)t) blk = -1;
            else break;
          }
        }
      }
    }
    if (lane == 0) s_blk[i] = blk;
    if (lane < 16) s_tok[i][lane] = tok;
  }
  __syncthreads();
  const int units = 2 * p.Hkv;
  for (int i = 0; i < p.group; ++i) {
    if (s_blk[i] < 0) continue;
    for (int u = blockIdx.y * QW_WARPS + warp; u < units; u += gridDim.y * QW_WARPS) q8_write_rows<FMT>(p, s_blk[i], u >> 1, u & 1, s_tok[i], s_found[warp]);
  }
}

// out_k / out_v [len, Hkv, 128] bf16 <- pages of one sequence; a thread takes 16 numbers of a key and of the value.
template <int FMT>
__global__ void __launch_bounds__(256)
q8_gather_kernel(const uint8_t* cache, const float* scale, const int* block_table, int len, int Hkv, int block_size, int num_blocks,
                 __nv_bfloat16* out_k, __nv_bfloat16* out_v, int* err) {   // len <= table entries * block_size (checked by the launcher)
  pdl_trigger();
  pdl_wait();
  const int vec_per_tok = Hkv * (Q8_D / 16);
  const long long total = (long long)len * vec_per_tok;
  const long long side = (long long)block_size * Hkv * Q8_D;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const int t = (int)(i / vec_per_tok), c = (int)(i - (long long)t * vec_per_tok) * 16;
    int blk = block_table[t / block_size];
    if (blk < 0 || blk >= num_blocks) { atomicCAS(err, 0, ERR_BAD_INDEX); blk = 0; }
    const uint8_t* src = cache + 2 * side * blk + (long long)(t % block_size) * Hkv * Q8_D + c;
    const float* s = scale + (long long)blk * 2 * Hkv + c / Q8_D;
    const uint4 k = *reinterpret_cast<const uint4*>(src), v = *reinterpret_cast<const uint4*>(src + side);
    const float sk = s[0], sv = s[Hkv];
    const unsigned kw[4] = {k.x, k.y, k.z, k.w}, vw[4] = {v.x, v.y, v.z, v.w};
    unsigned ok[8], ov[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 a = q8_floats<FMT>(kw[j]), b = q8_floats<FMT>(vw[j]);
      ok[2 * j] = pack_bf16x2(a.x * sk, a.y * sk);
      ok[2 * j + 1] = pack_bf16x2(a.z * sk, a.w * sk);
      ov[2 * j] = pack_bf16x2(b.x * sv, b.y * sv);
      ov[2 * j + 1] = pack_bf16x2(b.z * sv, b.w * sv);
    }
    uint4* dk = reinterpret_cast<uint4*>(out_k + (long long)t * Hkv * Q8_D + c);
    uint4* dv = reinterpret_cast<uint4*>(out_v + (long long)t * Hkv * Q8_D + c);
    dk[0] = make_uint4(ok[0], ok[1], ok[2], ok[3]);
    dk[1] = make_uint4(ok[4], ok[5], ok[6], ok[7]);
    dv[0] = make_uint4(ov[0], ov[1], ov[2], ov[3]);
    dv[1] = make_uint4(ov[4], ov[5], ov[6], ov[7]);
  }
}

}  // namespace mlf

using namespace mlf;

// k, v [T, Hkv, 128] bf16 (row pitch ldk / ldv, 16-byte aligned rows) into slots[T] = block * block_size + offset (< 0 skips).
// map: num_blocks * block_size ints of scratch, any contents; not needed for up to 256 tokens. fmt: 0 e4m3, 1 int8.
MLF_API int mlf_kv_write_q8(void* cache, float* scale, int fmt, const void* k, const void* v, const long long* slots, int* map, long long T,
                            int Hkv, int block_size, int num_blocks, long long ldk, long long ldv, uint64_t stream) {
  if (T <= 0) return 0;
  MLF_REQUIRE(fmt == Q8_E4M3 || fmt == Q8_INT8, "kv_write_q8: format %d", fmt);
  MLF_REQUIRE(Hkv > 0 && block_size > 0 && num_blocks > 0 && T < (1LL << 31), "kv_write_q8: bad sizes");
  MLF_REQUIRE(ldk % 8 == 0 && ldv % 8 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(cache)) & 15) == 0,
              "kv_write_q8: rows and cache must be 16-byte aligned");
  Q8WriteParams p;
  p.cache = static_cast<uint8_t*>(cache);
  p.scale = scale;
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.slots = slots;
  p.map = T > QW_FEW ? map : nullptr;
  MLF_REQUIRE(T <= QW_FEW || map != nullptr, "kv_write_q8: %lld tokens need a map", T);
  p.T = T; p.ldk = ldk; p.ldv = ldv;
  p.Hkv = Hkv; p.block_size = block_size; p.num_blocks = num_blocks;
  p.group = T > QW_FEW ? QW_GROUP : 1;        // few tokens: often one to a block, and too few CTAs otherwise
  p.err = device_status_word();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.map != nullptr) MLF_CHECK_CUDA(launch_pdl(q8_map_kernel, dim3((unsigned)((T + 255) / 256)), dim3(256), 0, st, p));
  const dim3 grid((unsigned)((T + p.group - 1) / p.group), (unsigned)((2 * Hkv + QW_WARPS - 1) / QW_WARPS));
  const auto kernel = fmt == Q8_E4M3 ? q8_write_kernel<Q8_E4M3> : q8_write_kernel<Q8_INT8>;
  MLF_CHECK_CUDA(launch_pdl(kernel, grid, dim3(QW_WARPS * 32), 0, st, p));
  count_launch(p.map != nullptr ? 2 : 1);
  return 0;
}

MLF_API int mlf_kv_gather_q8(const void* cache, const float* scale, int fmt, const int* block_table, int table_len, int len, int Hkv,
                             int block_size, int num_blocks, void* out_k, void* out_v, uint64_t stream) {
  if (len <= 0) return 0;
  MLF_REQUIRE(fmt == Q8_E4M3 || fmt == Q8_INT8, "kv_gather_q8: format %d", fmt);
  MLF_REQUIRE(Hkv > 0 && block_size > 0 && num_blocks > 0, "kv_gather_q8: bad sizes");
  MLF_REQUIRE((long long)len <= (long long)table_len * block_size, "kv_gather_q8: %d tokens need more than the %d block-table entries given", len,
              table_len);
  MLF_REQUIRE((reinterpret_cast<uintptr_t>(cache) & 15) == 0, "kv_gather_q8: the cache must be 16-byte aligned");
  long long g = ((long long)len * Hkv * (Q8_D / 16) + 255) / 256;
  const long long cap = (long long)sm_count() * 8;
  if (g > cap) g = cap;
  const auto kernel = fmt == Q8_E4M3 ? q8_gather_kernel<Q8_E4M3> : q8_gather_kernel<Q8_INT8>;
  MLF_CHECK_CUDA(launch_pdl(kernel, dim3((unsigned)g), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(cache), scale,
                            block_table, len, Hkv, block_size, num_blocks, static_cast<__nv_bfloat16*>(out_k), static_cast<__nv_bfloat16*>(out_v),
                            device_status_word()));
  count_launch();
  return 0;
}
