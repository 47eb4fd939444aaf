// dak_pages.cu - copying pages of a KV cache: forking and compacting sequences,
// and moving pages between HBM and pinned host memory.
//
// One launch copies every listed page in every slab (layer, K or V half) of the
// pools.  The list travels in the kernel's parameters, so a call needs no
// device buffer for it, can be captured into a graph, and its hazards can be
// refused on the host.  Bound by memory: each byte is read once and written
// once, 16 KB per CTA with all of a thread's loads before its stores.  397 pages
// of 70 KB in 16 slabs (885 MB): 135 us, 6.5 TB/s, the measured copy rate; 256
// pages from or to pinned host memory: 51 GB/s of a link whose copy engines reach
// 53 (in) and 56 (out).
#include <cstring>

#include "dak_common.cuh"
#include "dak_host.h"

namespace dak {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kPieceVecs = kCopyThreads * kCopyUnroll;  // 16 KB per CTA
constexpr int kMaxMoves = 3584;                         // 28 KB of the 32,764 parameter bytes
constexpr int kFewMoves = 120;                          // 1 KB of parameters: cheaper to launch
constexpr int kSomeMoves = 500;                         // 4 KB

template <int N>
struct CopyParams {
  uint4 *pool[2];             // device, host
  long long slab_stride[2];   // 16-byte vectors
  long long page_vecs;
  int pieces;                 // CTAs per page
  int moves, pdl;
  int32_t src[N], dst[N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
  pdl_enter(p.pdl);
  const long long page = blockIdx.x / p.pieces;
  const int piece = (int)(blockIdx.x - page * p.pieces);
  const long long slab = page / p.moves;
  const int m = (int)(page - slab * p.moves);
  const int a = p.src[m], b = p.dst[m];
  const uint4 *src = p.pool[a < 0] + slab * p.slab_stride[a < 0] + (a < 0 ? -1ll - a : a) * p.page_vecs;
  uint4 *dst = p.pool[b < 0] + slab * p.slab_stride[b < 0] + (b < 0 ? -1ll - b : b) * p.page_vecs;
  const long long v0 = (long long)piece * kPieceVecs + threadIdx.x;
  uint4 r[kCopyUnroll];
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i)
    if (v0 + i * kCopyThreads < p.page_vecs) r[i] = __ldcs(src + v0 + i * kCopyThreads);
#pragma unroll
  for (int i = 0; i < kCopyUnroll; ++i)
    if (v0 + i * kCopyThreads < p.page_vecs) __stcs(dst + v0 + i * kCopyThreads, r[i]);
  if (b < 0) __threadfence_system();
}

template <int N>
cudaError_t launch_copy(const void *pool_dev, const void *pool_host, long long dev_stride, long long host_stride,
                        long long page_bytes, int slabs, const int32_t *src, const int32_t *dst, int n, cudaStream_t s) {
  CopyParams<N> p;
  p.pool[0] = static_cast<uint4 *>(const_cast<void *>(pool_dev));
  p.pool[1] = static_cast<uint4 *>(const_cast<void *>(pool_host));
  p.slab_stride[0] = dev_stride / 16;
  p.slab_stride[1] = host_stride / 16;
  p.page_vecs = page_bytes / 16;
  p.pieces = (int)((p.page_vecs + kPieceVecs - 1) / kPieceVecs);
  p.moves = n;
  p.pdl = decode_pdl_enabled() ? 1 : 0;
  std::memcpy(p.src, src, sizeof(int32_t) * n);
  std::memcpy(p.dst, dst, sizeof(int32_t) * n);
  const long long grid = (long long)p.pieces * n * slabs;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  return launch_ex(copy_pages_kernel<N>, dim3((unsigned)grid), dim3(kCopyThreads), 0, s, 1, p.pdl != 0, p);
}

// Which of a list's entries were added: open addressing, at most half full.
class MoveSet {
 public:
  MoveSet(const int32_t *list, int n) : list_(list) {
    while ((2 << bits_) < 4 * n) ++bits_;
    std::memset(slots_, 0, sizeof(uint16_t) << bits_);
  }
  bool add(int i) {  // false: an equal entry is there
    uint16_t &s = slots_[find(list_[i])];
    if (s) return false;
    s = (uint16_t)(i + 1);
    return true;
  }
  bool has(int32_t v) const { return slots_[find(v)] != 0; }

 private:
  uint32_t find(int32_t v) const {
    const uint32_t mask = (1u << bits_) - 1;
    uint32_t at = ((uint32_t)v * 2654435769u) >> (32 - bits_);  // 2^32 over the golden ratio
    while (slots_[at] && list_[slots_[at] - 1] != v) at = (at + 1) & mask;
    return at;
  }
  const int32_t *list_;
  int bits_ = 4;
  uint16_t slots_[8192];
};
static_assert(2 * kMaxMoves <= 8192, "half full");

}  // namespace
}  // namespace dak

extern "C" int dak_copy_pages(void *pool_dev, int64_t dev_pages, void *pool_host, int64_t host_pages, int64_t page_bytes,
                              int slabs, int64_t dev_slab_stride, int64_t host_slab_stride, const int32_t *src,
                              const int32_t *dst, int n, void *stream) {
  using namespace dak;
  if (n < 0 || n > kMaxMoves) return fail(DAK_ERR_INVALID_ARG, "copy_pages: 0 to %d pages per call (got %d)", kMaxMoves, n);
  if (slabs <= 0 || page_bytes <= 0) return fail(DAK_ERR_INVALID_ARG, "copy_pages: slabs and page_bytes must be positive");
  if (dev_pages < 0 || host_pages < 0 || (dev_pages > 0) != (pool_dev != nullptr) ||
      (host_pages > 0) != (pool_host != nullptr))
    return fail(DAK_ERR_INVALID_ARG, "copy_pages: each tier needs a pool and a positive page count, or neither");
  if (n > 0 && (!src || !dst)) return fail(DAK_ERR_INVALID_ARG, "copy_pages: src and dst are required");
  if (page_bytes % 16 || dev_slab_stride % 16 || host_slab_stride % 16 ||
      ((reinterpret_cast<uintptr_t>(pool_dev) | reinterpret_cast<uintptr_t>(pool_host)) & 15u))
    return fail(DAK_ERR_ALIGNMENT, "copy_pages: pools, pages and slabs must be multiples of 16 bytes");
  if (slabs > 1 && ((pool_dev && dev_slab_stride / page_bytes < dev_pages) ||
                    (pool_host && host_slab_stride / page_bytes < host_pages)))
    return fail(DAK_ERR_INVALID_ARG, "copy_pages: slab stride below the pool's pages");
  // A page written by one copy must not be touched by another of the same
  // call: the copies run at the same time.
  for (int i = 0; i < n; ++i)
    for (int32_t v : {src[i], dst[i]}) {
      const int64_t idx = v < 0 ? -1ll - v : v;
      if (idx >= (v < 0 ? host_pages : dev_pages))
        return fail(DAK_ERR_INVALID_ARG, "copy_pages: entry %d is outside its pool", (int)v);
    }
  MoveSet written(dst, n);
  for (int i = 0; i < n; ++i)
    if (!written.add(i)) return fail(DAK_ERR_INVALID_ARG, "copy_pages: page %d is a destination twice", (int)dst[i]);
  for (int i = 0; i < n; ++i)
    if (written.has(src[i]))
      return fail(DAK_ERR_INVALID_ARG, "copy_pages: page %d is both a source and a destination", (int)src[i]);
  int st;
  if (pool_dev && (st = check_gpu_accessible(pool_dev, "pool_dev"))) return st;
  if (pool_host && (st = check_gpu_accessible(pool_host, "pool_host"))) return st;
  if (n == 0) return DAK_OK;
  auto s = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      n <= kFewMoves
          ? launch_copy<kFewMoves>(pool_dev, pool_host, dev_slab_stride, host_slab_stride, page_bytes, slabs, src, dst, n, s)
      : n <= kSomeMoves
          ? launch_copy<kSomeMoves>(pool_dev, pool_host, dev_slab_stride, host_slab_stride, page_bytes, slabs, src, dst, n, s)
          : launch_copy<kMaxMoves>(pool_dev, pool_host, dev_slab_stride, host_slab_stride, page_bytes, slabs, src, dst, n, s);
  return cuda_status(e, "copy_pages launch");
}
