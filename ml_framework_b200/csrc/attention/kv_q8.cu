// Writes to a paged 8-bit cache and the way back to bf16 (layout and scales: kv_q8.cuh).
//
// A block and head has one scale, so the rows of a call that fall into one block belong together: one warp takes a block's rows of
// one head and side, finds their largest magnitude, settles the scale and rounds. A call that writes a block's first row starts
// the block anew; otherwise the scale is the larger of the old one and the new rows' own, and where it grows the rows that the
// block held are rounded to it. Which rows of a block a call writes: up to 2048 tokens, a CTA looks through all slots of the call
// (16 KB, from the L2). For more, or blocks of more than 64 rows, q8_map_kernel notes for each slot which token goes there; the map is
// read back only where the slot it stands at names the same token, so that it needs no clearing: entries of earlier calls, or of
// nothing at all, point at tokens of other slots.
//
// Bound by HBM in long calls (a row is read in 16 bits and written in 8), by the chain of loads slots - rows (slots - map - slots -
// rows) in short ones. us with rows, cache and scales in HBM (floor at 6.54 TB/s): 37 tokens of 8 heads 4.6 (0.03), 1111 7 (1.0), 2048 9 (1.9), behind
// 1111 others 11, 8192 17 (7.7), 32768 49 (31), 4096 of 40 heads 32 (19).
// The way back, q8_gather_kernel: 3159 tokens of 8 heads 5.5 (3.0), 8192 10 (7.7), 32768 34 (31).
#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../mlf_api.h"
#include "kv_q8.cuh"

namespace mlf {

constexpr int QW_WARPS = 8;
constexpr int QW_GROUP = 16;                  // tokens whose blocks a CTA looks at: in a prompt's order about one block
constexpr int QW_FEW = 2048;                  // tokens, and rows of a block, that need no map
constexpr int QW_ROWS = 64;

struct Q8WriteParams {
  uint8_t* cache;
  float* scale;
  const __nv_bfloat16 *k, *v;
  const long long* slots;
  int* map;                                   // [num_blocks * block_size]; null: every CTA looks through the slots
  long long T;
  int ldk, ldv, Hkv, block_size, bs_shift, num_blocks, group;       // bs_shift: log2(block_size) or -1
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

// slot / block_size: a division of 64 bits takes as long as a load
__device__ __forceinline__ int q8_block(const Q8WriteParams& p, long long slot) {
  if (p.bs_shift >= 0) return (int)(slot >> p.bs_shift);
  return slot <= 0x7fffffff ? (int)((unsigned)slot / (unsigned)p.block_size) : (int)(slot / p.block_size);
}

// The token that the map has for `slot`, or -1.
__device__ __forceinline__ int q8_token_at(const Q8WriteParams& p, long long slot) {
  const int t = p.map[slot];
  return t >= 0 && t < p.T && p.slots[t] == slot ? t : -1;
}

// Eight bf16 numbers times inv in 8 bits. plain: no NaN, and none beyond the format.
template <int FMT>
__device__ __noinline__ uint2 q8_pack_any(uint4 x, float inv) {
  const float2 a = unpack_bf16x2(x.x), b = unpack_bf16x2(x.y), e = unpack_bf16x2(x.z), f = unpack_bf16x2(x.w);
  return make_uint2(q8_pack4<FMT>(a.x * inv, a.y * inv, b.x * inv, b.y * inv), q8_pack4<FMT>(e.x * inv, e.y * inv, f.x * inv, f.y * inv));
}
template <int FMT>
__device__ __forceinline__ uint2 q8_pack8(uint4 x, float inv, bool plain) {
  if (FMT == Q8_E4M3) {                       // the conversion minds NaN and the largest numbers itself
    const float2 a = unpack_bf16x2(x.x), b = unpack_bf16x2(x.y), e = unpack_bf16x2(x.z), f = unpack_bf16x2(x.w);
    return make_uint2(q8_pack4<FMT>(a.x * inv, a.y * inv, b.x * inv, b.y * inv), q8_pack4<FMT>(e.x * inv, e.y * inv, f.x * inv, f.y * inv));
  }
  if (!plain) return q8_pack_any<FMT>(x, inv);
  // rounded by adding 1.5 * 2^23: the integer is the low byte of the sum (one instruction for a conversion's two, at four times its rate)
  const unsigned w[4] = {x.x, x.y, x.z, x.w};
  unsigned lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(w[j]);
    lo[j] = __byte_perm(__float_as_uint(__fmaf_rn(f.x, inv, 12582912.f)), __float_as_uint(__fmaf_rn(f.y, inv, 12582912.f)), 0x0040);
  }
  return make_uint2(__byte_perm(lo[0], lo[1], 0x5410), __byte_perm(lo[2], lo[3], 0x5410));
}
template <int FMT>
__device__ __noinline__ void q8_shrink8(uint2* at, float ratio) {
  const uint2 held = *at;
  *at = make_uint2(q8_shrink4<FMT>(held.x, ratio), q8_shrink4<FMT>(held.y, ratio));
}

// A block's rows of one head and side. known: the tokens of its rows (-1: not written by this call), the first 16 of them with a map.
// True where the block keeps a scale that is no power of two: nothing is written, its rows are left to q8_write_divided.
template <int FMT, bool MAP>
__device__ __forceinline__ bool q8_write_rows(const Q8WriteParams& p, int blk, int h, int side, const int* known) {
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const long long first = (long long)blk * p.block_size, pitch = (long long)p.Hkv * Q8_D;
  const __nv_bfloat16* src = (side ? p.v : p.k) + (long long)h * Q8_D + col;
  const int ld = side ? p.ldv : p.ldk;
  uint8_t* dst = p.cache + (((long long)blk * 2 + side) * p.block_size * p.Hkv + h) * Q8_D + col + half * pitch;
  float* scale = p.scale + ((long long)blk * 2 + side) * p.Hkv + h;
  const int chunks = (p.block_size + 15) / 16;
  uint4 x[8];
  int tok = -1;                               // lanes 0..15: the token of row chunk * 16 + lane
  bool whole = false;                         // every row of the chunk is written: no row decides anything by itself
  auto load = [&](int c) {
    const int row = c * 16 + lane;
    tok = -1;
    if (lane < 16 && row < p.block_size) tok = !MAP || c == 0 ? known[row] : q8_token_at(p, first + row);
    whole = __all_sync(0xffffffffu, lane >= 16 || tok >= 0);
    if (whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4*>(src + (long long)__shfl_sync(0xffffffffu, tok, 2 * i + half) * ld);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = __shfl_sync(0xffffffffu, tok, 2 * i + half);
      x[i] = t >= 0 ? *reinterpret_cast<const uint4*>(src + (long long)t * ld) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const float held_scale = *scale;
  // the largest magnitude, by its bits (a NaN's are above all others')
  __nv_bfloat162 most = __float2bfloat162_rn(0.f), numbers = most;              // with NaN, and without
  bool anew = false;
  for (int c = 0; c < chunks; ++c) {
    load(c);
    if (c == 0) anew = __shfl_sync(0xffffffffu, tok, 0) >= 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned w[4] = {x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu, x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        most = __hmax2_nan(most, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
        numbers = __hmax2(numbers, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
      }
    }
  }
  const unsigned with_nan = __reduce_max_sync(0xffffffffu, max(__float_as_uint(__low2float(most)), __float_as_uint(__high2float(most))));
  const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, max(__float_as_uint(__low2float(numbers)), __float_as_uint(__high2float(numbers)))));
  const float fit = q8_scale_for<FMT>(amax), before = anew ? 0.f : held_scale;
  const float now = fmaxf(before, fit);
  if (!q8_power_of_two(now)) return true;
  const float inv = __frcp_rn(now), ratio = before * inv;     // exact for powers of two
  const bool shrink = !anew && before < now, plain = with_nan <= 0x7f800000u && amax * inv <= 127.f;
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) load(c);
    uint8_t* to = dst + c * 16 * pitch;
    if (whole && (FMT == Q8_E4M3 || plain)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        *reinterpret_cast<uint2*>(to) = q8_pack8<FMT>(x[i], inv, true);
        to += 2 * pitch;
      }
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = __shfl_sync(0xffffffffu, tok, 2 * i + half);
      if (t >= 0) *reinterpret_cast<uint2*>(to) = q8_pack8<FMT>(x[i], inv, plain);
      else if (shrink && c * 16 + 2 * i + half < p.block_size) q8_shrink8<FMT>(reinterpret_cast<uint2*>(to), ratio);
      to += 2 * pitch;
    }
  }
  if (lane == 0) *scale = now;
  return false;
}
// A row at a time and read again, behind the other units: the way that calls take holds no registers for it.
template <int FMT, bool MAP>
__device__ __forceinline__ void q8_write_divided(const Q8WriteParams& p, int blk, int h, int side, const int* known, float scale) {
  const int half = (threadIdx.x & 31) >> 4, col = (threadIdx.x & 15) * 8;
  const __nv_bfloat16* src = (side ? p.v : p.k) + (long long)h * Q8_D + col;
  uint8_t* dst = p.cache + (((long long)blk * 2 + side) * p.block_size * p.Hkv + h) * Q8_D + col;
#pragma unroll 1
  for (int row = half; row < p.block_size; row += 2) {
    const int t = !MAP || row < 16 ? known[row] : q8_token_at(p, (long long)blk * p.block_size + row);
    if (t < 0) continue;
    const uint4 x = *reinterpret_cast<const uint4*>(src + (long long)t * (side ? p.ldv : p.ldk));
    const float2 a = unpack_bf16x2(x.x), b = unpack_bf16x2(x.y), e = unpack_bf16x2(x.z), f = unpack_bf16x2(x.w);
    *reinterpret_cast<uint2*>(dst + (long long)row * p.Hkv * Q8_D) =
        make_uint2(q8_divide4<FMT>(a.x, a.y, b.x, b.y, scale), q8_divide4<FMT>(e.x, e.y, f.x, f.y, scale));
  }
}

// Three CTAs on an SM without a map, four with one: registers against loads in flight (us with three / four: 37 tokens of 8 heads 4.1 / 5.1,
// 1111 6.2 / 7.8, 8192 19.6 / 17.4, 4096 of 40 heads 39 / 33).
// A CTA looks at the blocks of `group` tokens and writes those whose first row, of the rows that the call writes there, one of these
// tokens is; the heads and sides are split over blockIdx.y.
template <int FMT, bool MAP>
__global__ void __launch_bounds__(QW_WARPS * 32, MAP ? 4 : 3) q8_write_kernel(const Q8WriteParams p) {
  __shared__ int s_blk[QW_GROUP], s_tok[QW_GROUP][QW_ROWS], s_blocks;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long from = (long long)blockIdx.x * p.group, end = (long long)p.num_blocks * p.block_size;
  // the blocks of the group, each once
  if (warp == 0) {
    const long long slot = lane < p.group && from + lane < p.T ? p.slots[from + lane] : -1;
    if (slot >= end) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    const int blk = slot >= 0 && slot < end ? q8_block(p, slot) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, blk);          // every lane takes part
    const bool once = blk >= 0 && __ffs(same) - 1 == lane;
    const unsigned all = __ballot_sync(0xffffffffu, once);
    if (once) s_blk[__popc(all & ((1u << lane) - 1u))] = blk;
    if (lane == 0) s_blocks = __popc(all);
  }
  if (!MAP)
    for (int i = tid; i < QW_GROUP * QW_ROWS; i += QW_WARPS * 32) (&s_tok[0][0])[i] = 0x7fffffff;
  __syncthreads();
  const int n = s_blocks;
  if (!MAP) {
    // every token of the call that goes to one of them
    constexpr int EACH = QW_FEW / (QW_WARPS * 32);
    long long slots[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int t = tid + j * QW_WARPS * 32;
      slots[j] = t < p.T ? p.slots[t] : -1;
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if (slots[j] < 0 || slots[j] >= end) continue;
      const int blk = q8_block(p, slots[j]);
      for (int i = 0; i < n; ++i)      // a slot that is given twice: the lower token
        if (s_blk[i] == blk) atomicMin(&s_tok[i][slots[j] - (long long)blk * p.block_size], tid + j * QW_WARPS * 32);
    }
    __syncthreads();
  }
  // the tokens of a block's rows (with a map, of the first 16), and the first one of them, whose CTA writes the block
  for (int i = warp; i < n; i += QW_WARPS) {
    int first = -1;
    for (int r0 = 0; r0 < p.block_size && (first < 0 || !MAP); r0 += 32) {
      const int r = r0 + lane;
      int t = -1;
      if (r < p.block_size) t = !MAP ? s_tok[i][r] : q8_token_at(p, (long long)s_blk[i] * p.block_size + r);
      if (t == 0x7fffffff) t = -1;
      const unsigned there = __ballot_sync(0xffffffffu, t >= 0);
      if (first < 0 && there != 0) first = __shfl_sync(0xffffffffu, t, __ffs(there) - 1);
      if (r < p.block_size && (!MAP || r < 16)) s_tok[i][r] = t;
    }
    __syncwarp();
    if (lane == 0 && (first < from || first >= from + p.group)) s_blk[i] = -1;                         // another CTA's
  }
  __syncthreads();
  const int units = 2 * p.Hkv;
  bool left = false;
  for (int i = 0; i < n; ++i) {
    if (s_blk[i] < 0) continue;
    for (int u = blockIdx.y * QW_WARPS + warp; u < units; u += gridDim.y * QW_WARPS) left |= q8_write_rows<FMT, MAP>(p, s_blk[i], u >> 1, u & 1, s_tok[i]);
  }
  if (!left) return;
  __syncwarp();                                // the scales that grew are lane 0's to write
  for (int i = 0; i < s_blocks; ++i) {
    if (s_blk[i] < 0) continue;
    for (int u = blockIdx.y * QW_WARPS + (threadIdx.x >> 5); u < 2 * p.Hkv; u += gridDim.y * QW_WARPS) {
      const float scale = p.scale[((long long)s_blk[i] * 2 + (u & 1)) * p.Hkv + (u >> 1)];
      if (!q8_power_of_two(scale)) q8_write_divided<FMT, MAP>(p, s_blk[i], u >> 1, u & 1, s_tok[i], scale);
    }
  }
}
static_assert(QW_GROUP <= 32, "a lane for every token of a group");

// out_k / out_v [len, Hkv, 128] bf16 <- pages of one sequence; sixteen threads a token and head, eight numbers of its key and of its
// value each (16 bytes out: with sixteen numbers a thread, every store left half of its sectors to the next one), of PAIRS such
// pairs at a time: one, or two from 64 K on (us with 1 / 2 / 4 a thread, with divisions for the shifts: 37 tokens of 8 heads 1.7 / 2.1 / 3.2, 3159 5.7 / 6.7 / 8.5, 8192
// 11.3 / 11.1 / 13.4, 32768 39 / 36 / 41).
template <int FMT, int PAIRS>
__global__ void __launch_bounds__(256)
q8_gather_kernel(const uint8_t* cache, const float* scale, const int* block_table, unsigned pairs, int Hkv, int block_size, int hkv_shift, int bs_shift,
                 int num_blocks, __nv_bfloat16* out_k, __nv_bfloat16* out_v, int* err) {   // tokens <= table entries * block_size (checked by the launcher)
  pdl_trigger();
  pdl_wait();
  const long long side = (long long)block_size * Hkv * Q8_D;
  const unsigned first = blockIdx.x * (16 * PAIRS) + (threadIdx.x >> 4), c = (threadIdx.x & 15) * 8;
  auto token_of = [&](unsigned i) { return hkv_shift >= 0 ? i >> hkv_shift : i / (unsigned)Hkv; };
  auto entry_of = [&](unsigned t) { return bs_shift >= 0 ? t >> bs_shift : t / (unsigned)block_size; };
  uint2 k[PAIRS], v[PAIRS];
  float sk[PAIRS], sv[PAIRS];
  int blk[PAIRS];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    const unsigned i = first + 16 * e;
    blk[e] = i < pairs ? block_table[entry_of(token_of(i))] : 0;
  }
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) bad = bad || blk[e] < 0 || blk[e] >= num_blocks;
  if (bad) atomicCAS(err, 0, ERR_BAD_INDEX);
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    const unsigned i = first + 16 * e;
    if (i < pairs) {
      const unsigned t = token_of(i), h = i - t * Hkv, b = entry_of(t);
      if (blk[e] < 0 || blk[e] >= num_blocks) blk[e] = 0;
      const uint8_t* src = cache + 2 * side * blk[e] + ((long long)(t - b * block_size) * Hkv + h) * Q8_D + c;
      const float* s = scale + (long long)blk[e] * 2 * Hkv + h;
      k[e] = *reinterpret_cast<const uint2*>(src);
      v[e] = *reinterpret_cast<const uint2*>(src + side);
      sk[e] = s[0];
      sv[e] = s[Hkv];
    }
  }
#pragma unroll
  for (int e = 0; e < PAIRS; ++e) {
    const unsigned i = first + 16 * e;
    if (i >= pairs) continue;
    auto put = [&](uint2 q, float f, __nv_bfloat16* out) {
      const float4 a = q8_floats<FMT>(q.x), b = q8_floats<FMT>(q.y);
      *reinterpret_cast<uint4*>(out + (long long)i * Q8_D + c) =
          make_uint4(pack_bf16x2(a.x * f, a.y * f), pack_bf16x2(a.z * f, a.w * f), pack_bf16x2(b.x * f, b.y * f), pack_bf16x2(b.z * f, b.w * f));
    };
    put(k[e], sk[e], out_k);
    put(v[e], sv[e], out_v);
  }
}

// log2 of a power of two, else -1
static int shift_of(int n) {
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == n) return sh;
  return -1;
}

}  // namespace mlf

using namespace mlf;

// k, v [T, Hkv, 128] bf16 (row pitch ldk / ldv, 16-byte aligned rows) into slots[T] = block * block_size + offset (< 0 skips).
// map: num_blocks * block_size ints of scratch, any contents; not needed for up to 2048 tokens and blocks of 64. fmt: 0 e4m3, 1 int8.
MLF_API int mlf_kv_write_q8(void* cache, float* scale, int fmt, const void* k, const void* v, const long long* slots, int* map, long long T,
                            int Hkv, int block_size, int num_blocks, long long ldk, long long ldv, uint64_t stream) {
  if (T <= 0) return 0;
  MLF_REQUIRE(fmt == Q8_E4M3 || fmt == Q8_INT8, "kv_write_q8: format %d", fmt);
  MLF_REQUIRE(Hkv > 0 && block_size > 0 && num_blocks > 0 && T < (1LL << 31), "kv_write_q8: bad sizes");
  MLF_REQUIRE(ldk >= 0 && ldv >= 0 && ldk < (1LL << 31) && ldv < (1LL << 31), "kv_write_q8: rows %lld and %lld elements apart", ldk, ldv);
  MLF_REQUIRE(ldk % 8 == 0 && ldv % 8 == 0 && ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(cache)) & 15) == 0,
              "kv_write_q8: rows and cache must be 16-byte aligned");
  Q8WriteParams p;
  p.cache = static_cast<uint8_t*>(cache);
  p.scale = scale;
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.slots = slots;
  p.bs_shift = shift_of(block_size);
  const bool few = T <= QW_FEW && block_size <= QW_ROWS;
  MLF_REQUIRE(few || map != nullptr, "kv_write_q8: %lld tokens into blocks of %d need a map", T, block_size);
  p.map = few ? nullptr : map;
  p.T = T; p.ldk = (int)ldk; p.ldv = (int)ldv;
  p.Hkv = Hkv; p.block_size = block_size; p.num_blocks = num_blocks;
  p.group = T > 256 ? QW_GROUP : 1;           // few tokens: often one to a block, and too few CTAs otherwise
  p.err = device_status_word();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.map != nullptr) MLF_CHECK_CUDA(launch_pdl(q8_map_kernel, dim3((unsigned)((T + 255) / 256)), dim3(256), 0, st, p));
  // a CTA finds its blocks once for all heads that it takes: about as many of them as fit, four to an SM
  const long long x = (T + p.group - 1) / p.group, most = (2 * Hkv + QW_WARPS - 1) / QW_WARPS, fill = 4LL * sm_count() / x > 0 ? 4LL * sm_count() / x : 1;
  const dim3 grid((unsigned)x, (unsigned)(fill < most ? fill : most));
  const auto kernel = fmt == Q8_E4M3 ? (few ? q8_write_kernel<Q8_E4M3, false> : q8_write_kernel<Q8_E4M3, true>)
                                     : (few ? q8_write_kernel<Q8_INT8, false> : q8_write_kernel<Q8_INT8, true>);
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
  MLF_REQUIRE((long long)len * Hkv < (1LL << 31), "kv_gather_q8: %d tokens of %d heads", len, Hkv);
  const unsigned pairs = (unsigned)len * (unsigned)Hkv, each = pairs >= 65536 ? 2 : 1, g = (pairs + 16 * each - 1) / (16 * each);
  const auto kernel = fmt == Q8_E4M3 ? (each == 1 ? q8_gather_kernel<Q8_E4M3, 1> : q8_gather_kernel<Q8_E4M3, 2>)
                                     : (each == 1 ? q8_gather_kernel<Q8_INT8, 1> : q8_gather_kernel<Q8_INT8, 2>);
  MLF_CHECK_CUDA(launch_pdl(kernel, dim3(g), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(cache), scale,
                            block_table, pairs, Hkv, block_size, shift_of(Hkv), shift_of(block_size), num_blocks, static_cast<__nv_bfloat16*>(out_k),
                            static_cast<__nv_bfloat16*>(out_v), device_status_word()));
  count_launch();
  return 0;
}
