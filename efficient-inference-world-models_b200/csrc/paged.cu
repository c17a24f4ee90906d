// Pages of a paged K/V cache: copies between pages for every layer at once.
#include <new>
#include <vector>

#include "launch.cuh"

namespace oasis {

int pages_check(const oasis_pages_t* p, const char* who) {
  if (!p || !p->k || !p->v) return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null pages");
  if (p->layers <= 0 || p->pages <= 0 || p->kv_heads <= 0 || p->page_tokens <= 0 || p->head_dim <= 0)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": page sizes must be positive");
  if (p->dtype != OASIS_DT_BF16 && p->dtype != OASIS_DT_FP16)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": pages are bf16 or fp16");
  if (!aligned16(p->k) || !aligned16(p->v))
    return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": page bases must be 16-byte aligned");
  const long long page = static_cast<long long>(p->kv_heads) * p->page_tokens * p->head_dim * 2;
  if (page % 16) return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": a page must be a multiple of 16 bytes");
  if (static_cast<long long>(p->pages) * p->page_tokens > 0x7fffffffLL)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": more than 2^31 - 1 token slots");
  return OASIS_OK;
}

// ----------------------------------------------------------------------------------
// Page copies.  One launch copies up to N pages for all layers, K and V: the page pairs
// travel as kernel parameters, so a captured launch needs no list in device memory and the
// caller's list is free when the call returns.  A page of one layer and tensor is one
// contiguous run; it is cut into pieces of kCopyPiece bytes, one per CTA.  CTAs of the same
// piece of successive pairs are neighbours, so a source copied to several forks comes from
// L2 after its first read.  Bound by HBM, every byte read once and written once: 1,500 pages of 16
// layers (3.1 GB) take 467 us, 6.7 TB/s; one page of 16 layers (2 MB) 2.0 us.
// The pointers are not __restrict__: that would let the sources be read through the read-only path, and
// with dependent launches the kernel that appends to the pages may still run when this one starts.
// ----------------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;                                     // 16-byte vectors per thread
constexpr long long kCopyPiece = kCopyThreads * kCopyVecs * 16;  // 32 KB

template <int N>
struct PagePairs {
  int32_t src[N], dst[N];
};

template <int N>
__global__ void __launch_bounds__(kCopyThreads)
    pages_copy_kernel(const __grid_constant__ PagePairs<N> pairs, int n, const uint8_t* sk, const uint8_t* sv,
                      uint8_t* dk, uint8_t* dv, int src_pages, int dst_pages, long long page_bytes, int pieces) {
  pdl_trigger();
  pdl_wait();
  // blockIdx.x = ((layer * 2 + tensor) * pieces + piece) * n + pair
  const long long unit = blockIdx.x;
  const int pair = static_cast<int>(unit % n);
  const long long rest = unit / n;
  const int piece = static_cast<int>(rest % pieces);
  const long long lt = rest / pieces;
  const long long layer = lt >> 1;
  const uint8_t* s = (lt & 1 ? sv : sk) + (layer * src_pages + pairs.src[pair]) * page_bytes;
  uint8_t* d = (lt & 1 ? dv : dk) + (layer * dst_pages + pairs.dst[pair]) * page_bytes;
  const long long base = piece * kCopyPiece + threadIdx.x * 16;
  uint4 v[kCopyVecs];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i) {
    const long long o = base + i * (kCopyThreads * 16);
    if (o < page_bytes) v[i] = *reinterpret_cast<const uint4*>(s + o);
  }
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i) {
    const long long o = base + i * (kCopyThreads * 16);
    if (o < page_bytes) *reinterpret_cast<uint4*>(d + o) = v[i];
  }
}

template <int N>
cudaError_t launch_pages_copy(const oasis_pages_t& s, const oasis_pages_t& d, const int32_t* src,
                              const int32_t* dst, int n, cudaStream_t stream) {
  PagePairs<N> pairs;
  for (int i = 0; i < n; ++i) {
    pairs.src[i] = src[i];
    pairs.dst[i] = dst[i];
  }
  const long long page = static_cast<long long>(s.kv_heads) * s.page_tokens * s.head_dim * 2;
  const int pieces = static_cast<int>((page + kCopyPiece - 1) / kCopyPiece);
  const long long units = 2LL * s.layers * pieces * n;
  return launch_pdl(pages_copy_kernel<N>, dim3(static_cast<unsigned>(units)), dim3(kCopyThreads), 0, stream,
                    pairs, n, static_cast<const uint8_t*>(s.k), static_cast<const uint8_t*>(s.v),
                    static_cast<uint8_t*>(d.k), static_cast<uint8_t*>(d.v), s.pages, d.pages, page, pieces);
}

}  // namespace oasis

extern "C" int oasis_pages_copy(const oasis_pages_t* src, const oasis_pages_t* dst, const int32_t* src_pages,
                                const int32_t* dst_pages, int n, cudaStream_t stream) {
  using namespace oasis;
  if (int st = pages_check(src, "oasis_pages_copy")) return st;
  if (int st = pages_check(dst, "oasis_pages_copy")) return st;
  if (src->layers != dst->layers || src->kv_heads != dst->kv_heads || src->page_tokens != dst->page_tokens ||
      src->head_dim != dst->head_dim || src->dtype != dst->dtype)
    return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: the caches' pages differ");
  if (n < 0 || (n > 0 && (!src_pages || !dst_pages)))
    return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: bad page lists");
  const bool same_k = src->k == dst->k, same_v = src->v == dst->v;
  const bool same = same_k && same_v;
  // another cache has to be other memory: overlapping pools are one cache seen at two bases
  const long long page = static_cast<long long>(src->kv_heads) * src->page_tokens * src->head_dim * 2;
  auto overlap = [&](const void* a, int na, const void* b, int nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + static_cast<uintptr_t>(page * src->layers * nb) &&
           y < x + static_cast<uintptr_t>(page * src->layers * na);
  };
  if (overlap(src->k, src->pages, dst->v, dst->pages) || overlap(src->v, src->pages, dst->k, dst->pages) ||
      (!same && (overlap(src->k, src->pages, dst->k, dst->pages) ||
                 overlap(src->v, src->pages, dst->v, dst->pages))) ||
      (same && src->pages != dst->pages))
    return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: the two caches overlap");
  try {
    std::vector<uint8_t> seen(static_cast<size_t>(dst->pages), 0);  // 1: a destination, 2: a source
    for (int i = 0; i < n; ++i) {
      if (src_pages[i] < 0 || src_pages[i] >= src->pages || dst_pages[i] < 0 || dst_pages[i] >= dst->pages)
        return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: page index out of range");
      if (seen[dst_pages[i]]++) return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: a destination is listed twice");
    }
    for (int i = 0; same && i < n; ++i)
      if (seen[src_pages[i]])
        return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: a page is both source and destination");
  } catch (const std::bad_alloc&) {
    return fail(OASIS_ERR_INVALID_ARG, "oasis_pages_copy: out of host memory");
  }
  // few pairs travel in 512 bytes of parameters, many in 16 KB (a launch copies all of
  // them, so a short list should not pay for a long one)
  constexpr int kFew = 64, kMany = 2048;
  const long long per_pair = 2LL * src->layers * ((page + kCopyPiece - 1) / kCopyPiece);
  if (per_pair > 0x7fffffffLL) return fail(OASIS_ERR_UNSUPPORTED, "oasis_pages_copy: pages too large");
  const int most = static_cast<int>(std::min<long long>(kMany, 0x7fffffffLL / per_pair));
  for (int i = 0; i < n;) {
    const int m = std::min(n - i, most);
    cudaError_t e = m <= kFew ? launch_pages_copy<kFew>(*src, *dst, src_pages + i, dst_pages + i, m, stream)
                              : launch_pages_copy<kMany>(*src, *dst, src_pages + i, dst_pages + i, m, stream);
    if (e != cudaSuccess) return cuda_status(e, "pages_copy_kernel");
    i += m;
  }
  return OASIS_OK;
}
