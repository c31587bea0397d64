// Copies of whole cache blocks, over all layers of a cache in one launch: the copy-on-write of forked sequences that diverge
// and the moves of a compaction (bookkeeping in serving/block_manager.cpp). dst block <- src block, for every tensor and pair.
//
// Bound by HBM: a copied byte is read once and written once. The tensors' addresses and the pairs, which the host knows, are
// kernel parameters: nothing is uploaded ahead of the launch, and a captured launch keeps its own. 700 blocks of 64 KB in 8 layers
// 115 us (6.4 TB/s), one in each of 32 layers 1.8.
#include <string.h>

#include <new>
#include <vector>

#include "../common/host.h"
#include "../common/ptx.cuh"
#include "../mlf_api.h"

namespace mlf {

constexpr int CB_TENSORS = 64;
constexpr int CB_PAIRS = 384;                 // with the tensors just below the 4 KB of parameters that every driver takes
constexpr int CB_THREADS = 256;
constexpr int CB_VECS = 4;                    // 16-byte loads in flight per thread

struct CopyBlocksParams {
  char* base[CB_TENSORS];
  unsigned bytes[CB_TENSORS];                 // of one block
  int2 pairs[CB_PAIRS];                       // (src, dst)
};

template <typename V>
__device__ __forceinline__ void copy_chunk(char* dst, const char* src, unsigned n) {   // n bytes, a multiple of sizeof(V)
  const unsigned vecs = n / sizeof(V);
  for (unsigned i0 = threadIdx.x; i0 < vecs; i0 += CB_THREADS * CB_VECS) {
    V r[CB_VECS];
#pragma unroll
    for (int j = 0; j < CB_VECS; ++j)
      if (i0 + j * CB_THREADS < vecs) r[j] = reinterpret_cast<const V*>(src)[i0 + j * CB_THREADS];
#pragma unroll
    for (int j = 0; j < CB_VECS; ++j)
      if (i0 + j * CB_THREADS < vecs) reinterpret_cast<V*>(dst)[i0 + j * CB_THREADS] = r[j];
  }
}

// grid (chunks of the largest block, pairs, tensors)
__global__ void __launch_bounds__(CB_THREADS)
copy_blocks_kernel(const __grid_constant__ CopyBlocksParams p, unsigned chunk) {
  pdl_trigger();
  pdl_wait();
  const unsigned bytes = p.bytes[blockIdx.z], at = blockIdx.x * chunk;
  if (at >= bytes) return;
  const int2 pr = p.pairs[blockIdx.y];
  char* base = p.base[blockIdx.z];
  const char* src = base + (long long)pr.x * bytes + at;
  char* dst = base + (long long)pr.y * bytes + at;
  const unsigned n = min(chunk, bytes - at);
  const unsigned low = (unsigned)(reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) | n;
  if ((low & 15) == 0) copy_chunk<uint4>(dst, src, n);
  else if ((low & 3) == 0) copy_chunk<unsigned>(dst, src, n);
  else copy_chunk<unsigned char>(dst, src, n);
}

}  // namespace mlf

using namespace mlf;

// bases / bytes: n_tensors tensors of num_blocks blocks each, and how large they are; pairs: n_pairs (src, dst) block numbers on the host. A block
// is written at most once and not read where it is written, so that the order of the copies does not matter.
MLF_API int mlf_kv_copy_blocks(void* const* bases, const long long* bytes, int n_tensors, const int* pairs, int n_pairs, int num_blocks,
                               uint64_t stream) {
  MLF_REQUIRE(n_tensors >= 0 && n_pairs >= 0 && num_blocks >= 0, "kv_copy_blocks: negative counts");
  if (n_tensors == 0 || n_pairs == 0) return 0;
  MLF_REQUIRE(num_blocks > 0, "kv_copy_blocks: no blocks");
  std::vector<unsigned char> role;
  try {
    role.assign(num_blocks, 0);
  } catch (const std::bad_alloc&) {
    MLF_REQUIRE(false, "kv_copy_blocks: out of host memory for %d blocks", num_blocks);
  }
  for (int i = 0; i < n_pairs; ++i) {
    const int s = pairs[2 * i], d = pairs[2 * i + 1];
    MLF_REQUIRE(s >= 0 && s < num_blocks && d >= 0 && d < num_blocks, "kv_copy_blocks: pair (%d, %d) is outside the cache's %d blocks", s, d, num_blocks);
    MLF_REQUIRE(!(role[d] & 2), "kv_copy_blocks: block %d is written twice", d);
    role[d] |= 2;
    role[s] |= 1;
  }
  for (int i = 0; i < n_pairs; ++i)
    MLF_REQUIRE(!(role[pairs[2 * i + 1]] & 1), "kv_copy_blocks: block %d is both read and written", pairs[2 * i + 1]);
  for (int t = 0; t < n_tensors; ++t)
    MLF_REQUIRE(bytes[t] > 0 && bytes[t] % num_blocks == 0 && bytes[t] / num_blocks < (1LL << 31), "kv_copy_blocks: %d blocks in %lld bytes", num_blocks, bytes[t]);
  const unsigned chunk = CB_THREADS * CB_VECS * 16;
  for (int t0 = 0; t0 < n_tensors; t0 += CB_TENSORS) {
    const int nt = n_tensors - t0 < CB_TENSORS ? n_tensors - t0 : CB_TENSORS;
    CopyBlocksParams p;
    long long most = 0;
    for (int t = 0; t < nt; ++t) {
      p.base[t] = static_cast<char*>(bases[t0 + t]);
      p.bytes[t] = (unsigned)(bytes[t0 + t] / num_blocks);
      most = most > p.bytes[t] ? most : p.bytes[t];
    }
    for (int i0 = 0; i0 < n_pairs; i0 += CB_PAIRS) {
      const int np = n_pairs - i0 < CB_PAIRS ? n_pairs - i0 : CB_PAIRS;
      memcpy(p.pairs, pairs + 2 * i0, (size_t)np * sizeof(int2));
      const dim3 grid((unsigned)((most + chunk - 1) / chunk), (unsigned)np, (unsigned)nt);
      MLF_CHECK_CUDA(launch_pdl(copy_blocks_kernel, grid, dim3(CB_THREADS), 0, reinterpret_cast<cudaStream_t>(stream), p, chunk));
      count_launch();
    }
  }
  return 0;
}
