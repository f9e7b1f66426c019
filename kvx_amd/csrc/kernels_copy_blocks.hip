// Block copies inside the caches of all layers (kvx_launch_copy_blocks).
//
// Data movement only: every byte of a block is read and written once, so the
// floor is 2 * block bytes * pairs * tensors over the HBM rate.  A dense block
// (any axis order) is one run of bytes, copied in 16-byte chunks; one launch
// covers K and V of up to kCopyTensors / 2 layers, whose bases travel as
// kernel arguments, so that a fork's few pages cost one launch instead of one
// for each layer.  Other blocks (padded axes, a block axis that is not
// outermost) are copied element by element through their strides.
//
// Measured, 64 tensors (32 layers) of 32 KiB blocks: 400 pairs 318 us (5.3 TB/s;
// a library copy of 2 GiB reaches 4.9), 2 pairs 3.4 us in the kernel and 10.7 us
// a call, which the host's walk over the layers takes; element by element (16
// padded tensors, 400 pairs) 346 us, 1.2 TB/s, where dense blocks take 80.
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "operators_internal.h"

namespace kvx {
namespace dev {
namespace {

constexpr int kCopyTensors = 96;  // 2.3 KB of kernel arguments
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;

struct CopyArgs {
  struct One {
    char *data;
    int64_t s_block;  // bytes
    int64_t num_blocks;
  } t[kCopyTensors];
  const void *pairs;
  int64_t block_bytes;
  int32_t tensors;
  int32_t parts;  // workgroups per block
  int32_t part;   // bytes of one of them
};

__device__ __forceinline__ int64_t id_at(const void *p, bool is64, int64_t i) {
  return is64 ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

template <int B, bool I64>
__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(CopyArgs a) {
  const int part = (int)(blockIdx.x % (uint32_t)a.parts);
  const uint32_t rest = blockIdx.x / (uint32_t)a.parts;
  const uint32_t tensor = rest % (uint32_t)a.tensors;
  const int64_t pair = rest / (uint32_t)a.tensors;
  const CopyArgs::One t = a.t[tensor];
  const int64_t src = id_at(a.pairs, I64, 2 * pair), dst = id_at(a.pairs, I64, 2 * pair + 1);
  if (src < 0 || dst < 0 || src >= t.num_blocks || dst >= t.num_blocks || src == dst) return;
  const int64_t at = (int64_t)part * a.part;
  const int64_t n = min((int64_t)a.part, a.block_bytes - at);
  const char *from = t.data + src * t.s_block + at;
  char *to = t.data + dst * t.s_block + at;
  constexpr int64_t kStep = (int64_t)kCopyThreads * B;
  int64_t i = (int64_t)threadIdx.x * B;
  for (; i + (kCopyUnroll - 1) * kStep < n; i += kCopyUnroll * kStep) {
    Raw<B> r[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) r[u] = ld<B, true>(from + i + u * kStep);
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u) st<B, true>(to + i + u * kStep, r[u]);
  }
  for (; i < n; i += kStep) st<B, true>(to + i, ld<B, true>(from + i));
}

struct StridedCopyArgs {
  char *data;
  const void *pairs;
  int64_t num_blocks;
  int64_t per_block;  // elements
  GeomBytes g;
  int32_t heads;
  int32_t head_dim;
  int32_t parts;
};

template <int E, bool I64>
__global__ void __launch_bounds__(kCopyThreads) copy_strided_kernel(StridedCopyArgs a) {
  const int64_t pair = blockIdx.x / (uint32_t)a.parts;
  const int64_t src = id_at(a.pairs, I64, 2 * pair), dst = id_at(a.pairs, I64, 2 * pair + 1);
  if (src < 0 || dst < 0 || src >= a.num_blocks || dst >= a.num_blocks || src == dst) return;
  const int64_t step = (int64_t)a.parts * kCopyThreads;
  for (int64_t e = (int64_t)(blockIdx.x % (uint32_t)a.parts) * kCopyThreads + threadIdx.x;
       e < a.per_block; e += step) {
    const int64_t d = e % a.head_dim, row = e / a.head_dim;
    const int64_t off = (row / a.heads) * a.g.s_off + (row % a.heads) * a.g.s_head +
                        (d / a.g.pack) * a.g.s_piece + (d % a.g.pack) * a.g.s_inner;
    st<E>(a.data + dst * a.g.s_block + off, ld<E>(a.data + src * a.g.s_block + off));
  }
}

// Bytes of a block whose elements fill one run of addresses from its first
// on, else 0: every axis in order of its stride steps by the size of those
// inside it.
int64_t dense_block_bytes(const CopyTensor &t) {
  struct Axis {
    int64_t n, s;
  } ax[4] = {{t.block_size, t.g.s_off}, {t.heads, t.g.s_head},
             {t.head_dim / t.g.pack, t.g.s_piece}, {t.g.pack, t.g.s_inner}};
  int64_t run = 1;
  bool used[4] = {};
  for (int k = 0; k < 4; ++k) {
    int next = -1;
    for (int i = 0; i < 4; ++i)
      if (!used[i] && (ax[i].n == 1 || ax[i].s == run)) {
        next = i;
        if (ax[i].n == 1) break;
      }
    if (next < 0) return 0;
    used[next] = true;
    run *= ax[next].n;
  }
  return run * t.esize;
}

template <int B>
void launch_copy(const CopyArgs &a, bool i64, int64_t grid, hipStream_t s) {
  if (i64)
    copy_blocks_kernel<B, true><<<dim3((uint32_t)grid), kCopyThreads, 0, s>>>(a);
  else
    copy_blocks_kernel<B, false><<<dim3((uint32_t)grid), kCopyThreads, 0, s>>>(a);
}

template <int E>
void launch_strided(const StridedCopyArgs &a, bool i64, int64_t grid, hipStream_t s) {
  if (i64)
    copy_strided_kernel<E, true><<<dim3((uint32_t)grid), kCopyThreads, 0, s>>>(a);
  else
    copy_strided_kernel<E, false><<<dim3((uint32_t)grid), kCopyThreads, 0, s>>>(a);
}

// Pairs per launch, so that the grid stays inside HIP's limit on work-items.
int64_t pairs_per_launch(int64_t per_pair) {
  const int64_t most = (int64_t)0xFFFFFFFF / kCopyThreads;
  return most / per_pair;
}

}  // namespace
}  // namespace dev

using namespace dev;

kvx_status_t enqueue_copy_blocks(const CopyTensor *tensors, int64_t count, const void *pairs,
                                 bool index_is64, int64_t pair_count, void *stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t pair_bytes = index_is64 ? 16 : 8;
  CopyArgs a{};
  uint64_t low = 0;  // low address and stride bits of the tensors collected
  auto flush = [&]() -> bool {
    if (a.tensors == 0) return true;
    low |= (uint64_t)a.block_bytes;
    const int width = low % 16 == 0 ? 16 : low % 4 == 0 ? 4 : low % 2 == 0 ? 2 : 1;
    // One pass of a workgroup's unrolled loop: 16 KiB of 16-byte chunks.
    a.part = kCopyThreads * kCopyUnroll * width;
    const int64_t parts = (a.block_bytes + a.part - 1) / a.part;
    if (parts > 0x7FFFFFFF / kCopyTensors) return false;
    a.parts = (int32_t)parts;
    const int64_t per_pair = parts * a.tensors, batch = pairs_per_launch(per_pair);
    if (batch == 0) return false;
    for (int64_t at = 0; at < pair_count; at += batch) {
      const int64_t n = pair_count - at < batch ? pair_count - at : batch;
      a.pairs = static_cast<const char *>(pairs) + at * pair_bytes;
      const int64_t grid = n * per_pair;
      if (width == 16) launch_copy<16>(a, index_is64, grid, s);
      else if (width == 4) launch_copy<4>(a, index_is64, grid, s);
      else if (width == 2) launch_copy<2>(a, index_is64, grid, s);
      else launch_copy<1>(a, index_is64, grid, s);
    }
    a.tensors = 0;
    low = 0;
    return true;
  };
  for (int64_t i = 0; i < count; ++i) {
    const CopyTensor &t = tensors[i];
    const int64_t bytes = dense_block_bytes(t);
    if (bytes > 0) {
      if (a.tensors == kCopyTensors || (a.tensors > 0 && bytes != a.block_bytes))
        if (!flush()) return KVX_STATUS_UNSUPPORTED;
      a.block_bytes = bytes;
      const int64_t step = t.num_blocks > 1 ? t.g.s_block * t.esize : 0;
      a.t[a.tensors++] = {t.data, step, t.num_blocks};
      low |= (uint64_t)(uintptr_t)t.data | (uint64_t)step;
      continue;
    }
    StridedCopyArgs b{};
    b.data = t.data;
    b.num_blocks = t.num_blocks;
    b.per_block = (int64_t)t.block_size * t.heads * t.head_dim;
    b.heads = t.heads;
    b.head_dim = t.head_dim;
    b.g = {t.g.s_block * t.esize, t.g.s_off * t.esize, t.g.s_head * t.esize,
           t.g.s_piece * t.esize, t.g.s_inner * t.esize, t.g.pack, 0};
    const int64_t want = (b.per_block + 4 * kCopyThreads - 1) / (4 * kCopyThreads);
    b.parts = (int32_t)(want < 1024 ? want : 1024);
    const int64_t batch = pairs_per_launch(b.parts);
    for (int64_t at = 0; at < pair_count; at += batch) {
      const int64_t n = pair_count - at < batch ? pair_count - at : batch;
      b.pairs = static_cast<const char *>(pairs) + at * pair_bytes;
      if (t.esize == 1) launch_strided<1>(b, index_is64, n * b.parts, s);
      else if (t.esize == 2) launch_strided<2>(b, index_is64, n * b.parts, s);
      else launch_strided<4>(b, index_is64, n * b.parts, s);
    }
  }
  if (!flush()) return KVX_STATUS_UNSUPPORTED;
  return hipGetLastError() == hipSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR;
}

}  // namespace kvx
