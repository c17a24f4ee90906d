// Attention over cache pages with a sliding window of frames and sink frames.
//
//   out = softmax(scale q K^T over the visible keys) V,  key j visible to position p iff
//   j < kv_len, j / F <= p / F and (W == 0 or p / F - j / F < W or j / F < S).
// The visible keys of a position are two runs: [0, sink_end) and [start, end).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "launch.cuh"

namespace oasis {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994): the integer divisions of a dozen rows are otherwise a
// microsecond before the first load.
struct FastDiv {
  int d;
  uint32_t mul, shift;
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((__umulhi(mul, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> shift);
  }
  __device__ __forceinline__ int mod(int n) const { return n - div(n) * d; }
};
inline FastDiv fast_div(int d) {
  uint32_t shift = 0;
  while ((1ull << shift) < static_cast<uint64_t>(d)) ++shift;
  return {d, static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}

struct WinArgs {
  const void* q;
  void* out;
  float* lse;
  long long q_ts, q_hs, o_ts, o_hs;
  const void *k, *v;
  int pages, kv_heads, page_tokens;
  FastDiv by_page, by_group, by_frame;
  const int32_t* table;
  int width;
  const int32_t *kv_len, *cu_q;
  int batch, tokens, heads, group;
  int window, sinks, frame;
  float scale_log2;  // scale * log2(e)
};

// Rows of the packed queries and cached tokens of sequence b, clamped to what exists.
struct WinSeq {
  int q0, n_q, kv;
};
__device__ __forceinline__ WinSeq win_seq(const WinArgs& a, int b) {
  WinSeq s;
  s.q0 = a.cu_q ? a.cu_q[b] : b;
  int q1 = a.cu_q ? a.cu_q[b + 1] : b + 1;
  s.q0 = max(0, min(s.q0, a.tokens));
  q1 = max(s.q0, min(q1, a.tokens));
  s.n_q = q1 - s.q0;
  s.kv = max(0, min(a.kv_len[b], a.width * a.page_tokens));
  return s;
}

constexpr int kWinSplits = 8;  // CTAs of a cluster, at most: the portable size

struct WinRange {
  int sink_end, start, end;  // visible: [0, sink_end) and [start, end); sink_end <= start
  __device__ __forceinline__ bool sees(int key) const {
    return key < end && (key >= start || key < sink_end);
  }
};
__device__ __forceinline__ WinRange win_range(const WinArgs& a, int pos, int kv) {
  WinRange r = {0, 0, 0};
  if (pos < 0) return r;  // more queries than cached tokens
  const int f = a.by_frame.div(pos);
  r.end = static_cast<int>(min(static_cast<long long>(f + 1) * a.frame, static_cast<long long>(kv)));
  if (a.window && f >= a.window) {
    r.start = (f - a.window + 1) * a.frame;
    r.sink_end = static_cast<int>(min(static_cast<long long>(a.sinks) * a.frame, static_cast<long long>(r.start)));
  }
  return r;
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

// Into the shared memory of a CTA of the cluster (a mapa_shared address).
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

// One query row by one warp, key after key with the running maximum and sum: each lane holds
// D / 32 dims.  Reads only what the row sees.  For the rows that the tiled kernels leave: those of a
// launch that was told of fewer, and those of a CTA with infinities or NaN in values that only some of
// its rows see.
template <typename T, int D>
__device__ __noinline__ void window_row(const WinArgs& a, int b, const WinSeq& s, int qi, int head, int lane) {
  constexpr int E = D / 32;
  const long long row = s.q0 + qi;
  const T* q = static_cast<const T*>(a.q) + row * a.q_ts + head * a.q_hs + lane * E;
  const WinRange r = win_range(a, s.kv - s.n_q + qi, s.kv);
  const int kvh = a.by_group.div(head);
  const int32_t* table = a.table + static_cast<long long>(b) * a.width;
  float qv[E], o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qv[i] = to_float(q[i]) * a.scale_log2;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const int hi = part ? r.end : r.sink_end;
#pragma unroll 1
    for (int key = part ? r.start : 0; key < hi; ++key) {
      const int page = table[a.by_page.div(key)];
      if (page < 0 || page >= a.pages) continue;
      const long long off =
          ((static_cast<long long>(page) * a.kv_heads + kvh) * a.page_tokens + a.by_page.mod(key)) * D + lane * E;
      const T* k = static_cast<const T*>(a.k) + off;
      const T* v = static_cast<const T*>(a.v) + off;
      float d = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) d = fmaf(qv[i], to_float(k[i]), d);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
      const float mn = fmaxf(m, d);
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float al = exp2f(m - base), p = exp2f(d - base);
      m = mn;
      l = l * al + p;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = fmaf(p, to_float(v[i]), o[i] * al);
    }
  }
  T* out = static_cast<T*>(a.out) + row * a.o_ts + head * a.o_hs + lane * E;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) out[i] = from_float<T>(l == 0.0f ? 0.0f : o[i] * inv);
  if (a.lse && lane == 0)
    a.lse[row * a.heads + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace oasis

#include "attn_window_tile.cuh"
#include "attn_window_few.cuh"

namespace oasis {

// Dynamic shared memory of a kernel above 48 KB, set once per device; `registers`: per thread, checked.
template <auto Kernel>
int allow_smem(int bytes, int registers, const char* what) {
  static std::atomic<uint64_t> done{0};  // one per kernel
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, what);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return OASIS_OK;
  if (registers) {  // what the kernel shares out anew is what the block starts with, or it waits for good
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, Kernel);
    if (e != cudaSuccess) return cuda_status(e, what);
    if (attr.numRegs != registers) return fail(OASIS_ERR_UNSUPPORTED, std::string(what) + ": built with other registers");
  }
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_status(e, what);
  done.fetch_or(bit, std::memory_order_release);
  return OASIS_OK;
}

// Rows of one page that a box of at most `most` rows can always take whole.
inline int page_box(int page_tokens, int most) {
  int r = 16;
  while (r < most && page_tokens % (2 * r) == 0) r *= 2;
  return r;
}

// The pages of one tensor as rows of D elements; boxes of 64 elements x box_rows.
int encode_page_rows(CUtensorMap* map, const void* base, const WinArgs& a, int d, int box_rows) {
  const long long dims[2] = {d, static_cast<long long>(a.pages) * a.kv_heads * a.page_tokens};
  const long long strides[1] = {static_cast<long long>(d) * 2};
  const int box[2] = {64, box_rows};
  return encode_bf16_sw128(map, base, 2, dims, strides, box);
}

// Keys of the longest sequence that a query can see under the window.
inline long long visible_keys(const WinArgs& a, int max_kv) {
  if (!a.window) return max_kv;
  return std::min<long long>(max_kv, (static_cast<long long>(a.window) + a.sinks) * a.frame);
}

// Clusters of `size` CTAs of a tile kernel that fit the device at once (a cluster lies within a GPC),
// asked once per device; 0 where the question fails.
template <typename T, int D>
int tile_clusters(int size) {
  static std::atomic<int> known[64][kWinSplits];  // + 1
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev < 64)
    if (const int k = known[dev][size - 1].load(std::memory_order_relaxed)) return k - 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(kWtThreads);
  cfg.dynamicSmemBytes = WtShape<D>::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, attn_window_tile_kernel<T, D>, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();
    n = 0;
  }
  if (dev < 64) known[dev][size - 1].store(n + 1, std::memory_order_relaxed);
  return n;
}

// CTAs of a cluster that share the keys of one pair of query tiles: the count of least estimated
// time, where a CTA costs its key tiles and about 3 more to begin and end, joining 2 more.
template <typename T, int D>
int tile_splits(long long pairs, long long keys) {
  const long long tiles = (keys + kWtKeys - 1) / kWtKeys;
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= kWinSplits; ++s) {
    const long long fit = tile_clusters<T, D>(s);
    if (fit <= 0) continue;
    const double cost = static_cast<double>((pairs + fit - 1) / fit) *
                        (static_cast<double>((tiles + s - 1) / s) + 3.0 + (s > 1 ? 2.0 : 0.0));
    if (least == 0.0 || cost < least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

// Whether the device takes clusters of kFewSplits CTAs of this kernel (more than the portable 8), asked
// once per device.
template <auto Kernel, int Threads>
bool wide_clusters() {
  static std::atomic<int> known[64];  // 1: no, 2: yes
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
  if (const int k = known[dev].load(std::memory_order_acquire)) return k == 2;
  int n = 0;
  bool fine = cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
  if (fine) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kFewSplits);
    cfg.blockDim = dim3(Threads);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kFewSplits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    fine = cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg) == cudaSuccess && n > 0;
  }
  if (!fine) (void)cudaGetLastError();
  known[dev].store(fine ? 2 : 1, std::memory_order_release);
  return fine;
}

template <typename T, int D, int NR, int NW>
int launch_attn_window_few(const WinArgs& a, long long base, long long steps, cudaStream_t stream) {
  // CTAs per (sequence, key head): six of 4 warps per SM, where three (D = 128) are resident at a time,
  // so that ragged sequences even out; a warp keeps a step of 16 keys at least.  32 ragged sequences of
  // 8 key heads: 151 us with 4, 164 with 2 or 8, 187 with 1.
  const long long want = std::min((6LL * num_sms() + base - 1) / base, (steps + NW - 1) / NW);
  constexpr auto kernel = attn_window_few_kernel<T, D, NR, NW>;
  const bool more = want > kWinSplits && base * kWinSplits * NW <= 256 && wide_clusters<kernel, NW * 32>();
  const long long most = more ? kFewSplits : kWinSplits;
  const int splits = static_cast<int>(std::max(1LL, std::min(want, most)));
  cudaError_t e = launch_pdl_cluster(kernel, dim3(splits * a.kv_heads, 1, a.batch), dim3(NW * 32), 0, stream, splits, a,
                                     splits);
  if (e != cudaSuccess) return cuda_status(e, "attn_window_few_kernel");
  return OASIS_OK;
}

template <typename T, int D>
int launch_attn_window(const WinArgs& a, int max_q, int max_kv, cudaStream_t stream) {
  const long long max_rows = static_cast<long long>(max_q) * a.group;
  // The few-rows kernel takes at most 16.  8 sequences of 4,096 tokens, 16 heads of 64: 16 rows 50 us there, 17
  // rows 53 here; 32 heads of 128 on 8 key heads: 16 rows 39 us there, 32 rows 37 here.
  if (max_rows > 16) {
    const int box = page_box(a.page_tokens, kWtKeys);
    CUtensorMap tk, tv;
    if (int st = encode_page_rows(&tk, a.k, a, D, box)) return st;
    if (int st = encode_page_rows(&tv, a.v, a, D, box)) return st;
    if (int st = allow_smem<attn_window_tile_kernel<T, D>>(WtShape<D>::kSmem, kWtRegs, "attn_window_tile_kernel")) return st;
    const int row_tiles = static_cast<int>((max_rows + 2 * kWtRows - 1) / (2 * kWtRows));
    const int splits = tile_splits<T, D>(static_cast<long long>(row_tiles) * a.kv_heads * a.batch, visible_keys(a, max_kv));
    if (static_cast<long long>(row_tiles) * a.kv_heads * splits > 0x7fffffffLL)
      return fail(OASIS_ERR_UNSUPPORTED, "oasis_attn_window: too many query rows");
    cudaError_t e = launch_pdl_cluster(attn_window_tile_kernel<T, D>, dim3(row_tiles * a.kv_heads * splits, 1, a.batch),
                                       dim3(kWtThreads), WtShape<D>::kSmem, stream, splits, a, tk, tv, box, row_tiles,
                                       splits);
    if (e != cudaSuccess) return cuda_status(e, "attn_window_tile_kernel");
    return OASIS_OK;
  }
  // Few pairs of a sequence and a key head: twice the warps per CTA (1 sequence of 16,000 tokens and 8 key
  // heads of 128: 22 us against 35), and clusters of up to 16 where those would still leave most SMs
  // without work (1 key head: 13 us against 20; with 8 key heads they take 26, clusters of 16 lying worse).
  const long long base = static_cast<long long>(a.batch) * a.kv_heads;
  const long long steps = (visible_keys(a, max_kv) + 15) / 16;
  const bool wide = base * 64 <= 12LL * num_sms() && steps >= 4 * kWinSplits;
  if (max_rows <= 8)
    return wide ? launch_attn_window_few<T, D, 8, 8>(a, base, steps, stream)
                : launch_attn_window_few<T, D, 8, 4>(a, base, steps, stream);
  if constexpr (D == 64)  // (the parts of 8 warps, 16 rows and 128 dims would not fit)
    if (wide) return launch_attn_window_few<T, D, 16, 8>(a, base, steps, stream);
  return launch_attn_window_few<T, D, 16, 4>(a, base, steps, stream);
}

}  // namespace oasis

extern "C" int oasis_attn_window(const oasis_attn_window_t* p, cudaStream_t stream) {
  using namespace oasis;
  const char* who = "oasis_attn_window";
  if (!p) return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null arguments");
  if (p->batch < 0 || p->tokens < 0 || p->heads <= 0 || p->kv_heads <= 0 || p->table_width <= 0 ||
      p->max_q < 0 || p->max_kv < 0)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": bad sizes");
  if (p->heads % p->kv_heads)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": heads must be a multiple of kv_heads");
  if (p->window < 0 || p->sinks < 0 || p->frame_tokens <= 0)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": window and sinks >= 0, frame_tokens >= 1");
  if (p->head_dim != 64 && p->head_dim != 128)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": head_dim must be 64 or 128");
  if (p->page_tokens % 16)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": page_tokens must be a multiple of 16");
  if (p->dtype != OASIS_DT_BF16 && p->dtype != OASIS_DT_FP16)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": bf16 or fp16");
  if (!(p->scale > 0.0f) || p->scale > 2.0e38f)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": scale must be positive and finite");
  if (p->batch > 65535 || p->heads > 65535)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": at most 65535 sequences and heads");
  if (static_cast<long long>(p->table_width) * p->page_tokens > 0x3fffffffLL)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": at most 2^30 - 1 tokens per sequence");
  if (static_cast<long long>(p->tokens) * (p->heads / p->kv_heads) > 0x7fffff00LL)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": more than 2^31 query rows per key head");
  if (!p->cu_q && p->tokens != p->batch)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": without cu_q there is one query per sequence");
  if (p->batch == 0 || p->tokens == 0) return OASIS_OK;
  if (!p->q || !p->out || !p->page_table || !p->kv_len)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null pointer");
  const oasis_pages_t pages = {const_cast<void*>(p->k), const_cast<void*>(p->v), 1, p->pages, p->kv_heads,
                               p->page_tokens, p->head_dim, p->dtype};
  if (int st = pages_check(&pages, who)) return st;
  if (static_cast<long long>(p->pages) * p->kv_heads * p->page_tokens > 0x7fffff00LL)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": more than 2^31 rows of pages");
  for (long long s : {p->q_token_stride, p->q_head_stride, p->out_token_stride, p->out_head_stride})
    if (s % 8) return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": strides must be multiples of 16 bytes");
  if (!aligned16(p->q) || !aligned16(p->out))
    return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": bases must be 16-byte aligned");
  WinArgs a = {};
  a.q = p->q, a.out = p->out, a.lse = p->lse;
  a.q_ts = p->q_token_stride, a.q_hs = p->q_head_stride;
  a.o_ts = p->out_token_stride, a.o_hs = p->out_head_stride;
  a.k = p->k, a.v = p->v;
  a.pages = p->pages, a.kv_heads = p->kv_heads, a.page_tokens = p->page_tokens;
  a.table = p->page_table, a.width = p->table_width;
  a.kv_len = p->kv_len, a.cu_q = p->cu_q;
  a.batch = p->batch, a.tokens = p->tokens, a.heads = p->heads, a.group = p->heads / p->kv_heads;
  // a frame longer than any sequence is one frame; more sinks than any sequence are all of it
  a.frame = std::min(p->frame_tokens, 0x3fffffff);
  a.window = p->window;
  a.sinks = p->sinks;
  a.by_page = fast_div(a.page_tokens), a.by_group = fast_div(a.group), a.by_frame = fast_div(a.frame);
  a.scale_log2 = p->scale * 1.4426950408889634f;
  const int capacity = p->table_width * p->page_tokens;
  const int max_q = !p->cu_q ? 1 : p->max_q > 0 ? std::min(p->max_q, p->tokens) : p->tokens;
  const int max_kv = p->max_kv > 0 ? std::min(p->max_kv, capacity) : capacity;
  if (p->dtype == OASIS_DT_BF16)
    return p->head_dim == 64 ? launch_attn_window<__nv_bfloat16, 64>(a, max_q, max_kv, stream)
                             : launch_attn_window<__nv_bfloat16, 128>(a, max_q, max_kv, stream);
  return p->head_dim == 64 ? launch_attn_window<__half, 64>(a, max_q, max_kv, stream)
                           : launch_attn_window<__half, 128>(a, max_q, max_kv, stream);
}
