// RMS norm of query and key heads with the rotation over several position axes, in one pass;
// optionally the append of keys and values into cache pages.
#include "launch.cuh"

namespace oasis {

// 8 consecutive elements of a row as fp32, and back with one rounding to nearest even.
template <typename T>
struct Vec8;
template <>
struct Vec8<__nv_bfloat16> {
  using raw = uint4;
  static __device__ __forceinline__ void unpack(const raw& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
  static __device__ __forceinline__ raw pack(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                      pack_bf16x2(x[6], x[7]));
  }
};
template <>
struct Vec8<__half> {
  using raw = uint4;
  static __device__ __forceinline__ void unpack(const raw& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ raw pack(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
struct alignas(16) Raw32 {
  float4 a, b;
};
template <>
struct Vec8<float> {
  using raw = Raw32;
  static __device__ __forceinline__ void unpack(const raw& r, float (&x)[8]) {
    x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w;
    x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
  }
  static __device__ __forceinline__ raw pack(const float (&x)[8]) {
    Raw32 r;
    r.a = make_float4(x[0], x[1], x[2], x[3]);
    r.b = make_float4(x[4], x[5], x[6], x[7]);
    return r;
  }
};

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;  // with slots: k_out / v_out are the pages
  long long q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs, ko_ts, ko_hs;
  int tokens, heads, kv_heads;
  float eps;
  const float *qw, *kw;
  const void* positions;
  int positions_64;
  const double* freqs;
  int axes, pair_end[OASIS_MAX_AXES];  // pairs of axis a: pair_end[a-1] .. pair_end[a]-1
  const int32_t* slots;
  int page_tokens;
  long long n_slots;  // pages * page_tokens
  int warps_per_token;
};

constexpr int kRopeWarps = 8;

// A head of D elements is spread over L = D / 8 lanes, 8 consecutive elements (16 or 32 bytes)
// each, so a warp takes 32 / L heads at a time and a mean of squares is log2(L) shuffles.  A CTA
// takes 8 / warps_per_token tokens.  It first computes the cos and sin of every rotated pair of
// its tokens into shared memory, one pair per thread: the angle is position * frequency in turns,
// reduced to [-1/2, 1/2] in fp64 (an fp32 angle of position 10^6 is off by 0.06 rad), then sincospi
// in fp32.  Each lane keeps the values of its own pairs in registers for all heads of the token.
// With the half-split pairing the other element of a pair sits in another lane, rot / 16 away, and
// comes by shuffle.  Bound by HBM (every byte read and written once).
template <typename T, int D, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(kRopeWarps * 32) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = D / 8;
  constexpr int HPI = 32 / L;  // heads per warp and iteration
  constexpr int NA = INTERLEAVED ? 4 : 8;
  using V = Vec8<T>;
  using raw = typename V::raw;
  __shared__ float2 s_cs[kRopeWarps][D / 2];
  pdl_trigger();
  pdl_wait();
  const int wpt = a.warps_per_token;
  const int tpc = kRopeWarps / wpt;  // tokens per CTA
  const long long tok0 = static_cast<long long>(blockIdx.x) * tpc;
  const int pairs = a.pair_end[a.axes - 1];
  for (int i = threadIdx.x; i < tpc * pairs; i += kRopeWarps * 32) {
    const int lt = i / pairs, p = i - lt * pairs;
    const long long t = tok0 + lt;
    if (t >= a.tokens) break;
    int ax = 0;
    while (p >= a.pair_end[ax]) ++ax;
    const long long at = t * a.axes + ax;
    const double pos = a.positions_64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                                      : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
    const double turns = pos * a.freqs[p] * 0.15915494309189533577;  // 1 / (2 pi)
    const float frac = static_cast<float>(turns - rint(turns));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    s_cs[lt][p] = make_float2(cs, sn);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lt = warp / wpt, part = warp - lt * wpt;
  const long long t = tok0 + lt;
  if (t >= a.tokens) return;
  const int j = lane % L, sub = lane / L;
  // this lane's pairs: cos / sin, identity beyond the rotated dims
  float cs[NA], sn[NA];
  int partner = lane;
  if (INTERLEAVED) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int p = 4 * j + i;
      const float2 c = p < pairs ? s_cs[lt][p] : make_float2(1.0f, 0.0f);
      cs[i] = c.x;
      sn[i] = c.y;
    }
  } else {
    // pairs % 8 == 0: a lane's 8 dims are all first halves, all second halves or none
    const int hl = pairs / 8;  // lanes of one half
    const bool first = j < hl, second = !first && j < 2 * hl;
    partner = first ? lane + hl : second ? lane - hl : lane;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      float2 c = make_float2(1.0f, 0.0f);
      if (first || second) c = s_cs[lt][(first ? j : j - hl) * 8 + i];
      cs[i] = c.x;
      sn[i] = first ? -c.y : c.y;  // first: a cos - b sin, second: b cos + a sin
    }
  }
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wq[i] = NORM && a.qw ? a.qw[j * 8 + i] : 1.0f;
    wk[i] = NORM && a.kw ? a.kw[j * 8 + i] : 1.0f;
  }
  long long slot_off = 0;  // element offset of head 0 of the token's slot in the pages
  long long slot_hs = 0;
  bool stored = true;
  if (a.slots) {
    const long long s = a.slots[t];
    stored = s >= 0 && s < a.n_slots;
    const long long page = s / a.page_tokens;
    slot_off = (page * a.kv_heads * a.page_tokens + (s - page * a.page_tokens)) * D;
    slot_hs = static_cast<long long>(a.page_tokens) * D;
  }
  const int rows = a.heads + a.kv_heads;
  const T* qp = static_cast<const T*>(a.q) + t * a.q_ts + j * 8;
  const T* kp = static_cast<const T*>(a.k) + t * a.k_ts + j * 8;
  T* qo = static_cast<T*>(a.q_out) + t * a.qo_ts + j * 8;
  T* ko = static_cast<T*>(a.k_out) + (a.slots ? slot_off : t * a.ko_ts) + j * 8;
  const long long ko_hs = a.slots ? slot_hs : a.ko_hs;
  constexpr int U = 4;  // row groups in flight
  for (int r0 = part * HPI * U; r0 < rows; r0 += wpt * HPI * U) {
    raw in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * HPI + sub;
      if (r < rows)
        in[u] = *reinterpret_cast<const raw*>(r < a.heads ? qp + r * a.q_hs : kp + (r - a.heads) * a.k_hs);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * HPI + sub;
      if (r0 + u * HPI >= rows) break;  // warp-uniform
      const bool is_q = r < a.heads;
      float x[8];
      if (r < rows) {
        V::unpack(in[u], x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
      }
      if (NORM) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rs = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * rs * (is_q ? wq[i] : wk[i]);
      }
      float y[8];
      if (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
          y[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
        }
        if (4 * j + 3 >= pairs) {  // pass-through dims keep their value, NaN neighbours or not
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * j + i >= pairs) {
              y[2 * i] = x[2 * i];
              y[2 * i + 1] = x[2 * i + 1];
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float other = __shfl_sync(0xffffffffu, x[i], partner);
          y[i] = partner == lane ? x[i] : x[i] * cs[i] + other * sn[i];
        }
      }
      if (r < rows) {
        if (is_q)
          *reinterpret_cast<raw*>(qo + r * a.qo_hs) = V::pack(y);
        else if (stored)
          *reinterpret_cast<raw*>(ko + (r - a.heads) * ko_hs) = V::pack(y);
      }
    }
  }
  if (a.slots && stored) {
    const T* vp = static_cast<const T*>(a.v) + t * a.v_ts + j * 8;
    T* vo = static_cast<T*>(a.v_out) + slot_off + j * 8;
    for (int r = part * HPI + sub; r < a.kv_heads; r += wpt * HPI)
      *reinterpret_cast<raw*>(vo + r * slot_hs) = *reinterpret_cast<const raw*>(vp + r * a.v_hs);
  }
}

template <typename T, int D>
cudaError_t launch_qk_norm_rope(const RopeArgs& a, bool interleaved, bool norm, cudaStream_t stream) {
  const int tpc = kRopeWarps / a.warps_per_token;
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.tokens) + tpc - 1) / tpc)), block(kRopeWarps * 32);
  if (interleaved)
    return norm ? launch_pdl(qk_norm_rope_kernel<T, D, true, true>, grid, block, 0, stream, a)
                : launch_pdl(qk_norm_rope_kernel<T, D, true, false>, grid, block, 0, stream, a);
  return norm ? launch_pdl(qk_norm_rope_kernel<T, D, false, true>, grid, block, 0, stream, a)
              : launch_pdl(qk_norm_rope_kernel<T, D, false, false>, grid, block, 0, stream, a);
}

template <typename T>
cudaError_t launch_qk_norm_rope(const RopeArgs& a, int d, bool interleaved, bool norm, cudaStream_t stream) {
  switch (d) {
    case 32: return launch_qk_norm_rope<T, 32>(a, interleaved, norm, stream);
    case 64: return launch_qk_norm_rope<T, 64>(a, interleaved, norm, stream);
    case 128: return launch_qk_norm_rope<T, 128>(a, interleaved, norm, stream);
    default: return launch_qk_norm_rope<T, 256>(a, interleaved, norm, stream);
  }
}

}  // namespace oasis

extern "C" int oasis_qk_norm_rope(const oasis_qk_norm_rope_t* p, cudaStream_t stream) {
  using namespace oasis;
  const char* who = "oasis_qk_norm_rope";
  if (!p) return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null arguments");
  if (p->tokens < 0 || p->heads <= 0 || p->kv_heads <= 0)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": bad token or head count");
  if (p->dtype < OASIS_DT_BF16 || p->dtype > OASIS_DT_FP32)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": bf16, fp16 or fp32");
  const int d = p->head_dim;
  if (d != 32 && d != 64 && d != 128 && d != 256)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": head_dim must be 32, 64, 128 or 256");
  if (p->axes < 1 || p->axes > OASIS_MAX_AXES)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": 1 to 4 position axes");
  RopeArgs a = {};
  int rot = 0;
  for (int i = 0; i < p->axes; ++i) {
    if (p->axis_dims[i] <= 0 || p->axis_dims[i] % 2 || p->axis_dims[i] > d)
      return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": axis dims must be even, 2..head_dim");
    rot += p->axis_dims[i];
    a.pair_end[i] = rot / 2;
  }
  if (rot > d) return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": the axes' dims exceed head_dim");
  if (!p->interleaved && rot % 16)
    return fail(OASIS_ERR_UNSUPPORTED, std::string(who) + ": the half-split form needs rotated dims % 16 == 0");
  if (!p->norm && (p->q_weight || p->k_weight))
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": weights without the norm");
  if (p->tokens == 0) return OASIS_OK;
  if (!p->q || !p->k || !p->q_out || !p->positions || !p->freqs)
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null pointer");
  const bool append = p->pages != nullptr;
  if (append) {
    if (int st = pages_check(p->pages, who)) return st;
    if (!p->v || !p->slots) return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": an append needs v and slots");
    if (p->pages->layers != 1 || p->pages->kv_heads != p->kv_heads || p->pages->head_dim != d ||
        p->pages->dtype != p->dtype)
      return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": the pages do not fit the keys (one layer, heads, head_dim, type)");
  } else if (!p->k_out) {
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null pointer");
  }
  const int esize = p->dtype == OASIS_DT_FP32 ? 4 : 2;
  const long long strides[] = {p->q_token_stride, p->q_head_stride, p->k_token_stride, p->k_head_stride,
                               p->q_out_token_stride, p->q_out_head_stride,
                               append ? p->v_token_stride : p->k_out_token_stride,
                               append ? p->v_head_stride : p->k_out_head_stride};
  for (long long s : strides)
    if ((s * esize) % 16) return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": strides must be multiples of 16 bytes");
  if (!aligned16(p->q) || !aligned16(p->k) || !aligned16(p->q_out) || !aligned16(append ? p->v : p->k_out))
    return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": bases must be 16-byte aligned");
  a.q = p->q, a.k = p->k, a.v = p->v, a.q_out = p->q_out;
  a.k_out = append ? p->pages->k : p->k_out;
  a.v_out = append ? p->pages->v : nullptr;
  a.q_ts = p->q_token_stride, a.q_hs = p->q_head_stride;
  a.k_ts = p->k_token_stride, a.k_hs = p->k_head_stride;
  a.v_ts = p->v_token_stride, a.v_hs = p->v_head_stride;
  a.qo_ts = p->q_out_token_stride, a.qo_hs = p->q_out_head_stride;
  a.ko_ts = p->k_out_token_stride, a.ko_hs = p->k_out_head_stride;
  a.tokens = p->tokens, a.heads = p->heads, a.kv_heads = p->kv_heads;
  a.eps = p->eps;
  a.qw = p->q_weight, a.kw = p->k_weight;
  a.positions = p->positions, a.positions_64 = p->positions_64;
  a.freqs = p->freqs, a.axes = p->axes;
  a.slots = append ? p->slots : nullptr;
  a.page_tokens = append ? p->pages->page_tokens : 1;
  a.n_slots = append ? static_cast<long long>(p->pages->pages) * p->pages->page_tokens : 0;
  // few tokens: several warps share one, so that the heads of a token run side by side
  a.warps_per_token = 1;
  while (a.warps_per_token < kRopeWarps &&
         static_cast<long long>(p->tokens) * a.warps_per_token < 16LL * num_sms())
    a.warps_per_token *= 2;
  cudaError_t e;
  if (p->dtype == OASIS_DT_BF16)
    e = launch_qk_norm_rope<__nv_bfloat16>(a, d, p->interleaved, p->norm, stream);
  else if (p->dtype == OASIS_DT_FP16)
    e = launch_qk_norm_rope<__half>(a, d, p->interleaved, p->norm, stream);
  else
    e = launch_qk_norm_rope<float>(a, d, p->interleaved, p->norm, stream);
  if (e != cudaSuccess) return cuda_status(e, "qk_norm_rope_kernel");
  return OASIS_OK;
}
