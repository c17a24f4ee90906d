// RMS norm of query and key heads with the rotation over several position axes, in one pass;
// optionally the append of keys and values into cache pages.
#include <algorithm>

#include "launch.cuh"

namespace oasis {

// 8 elements of a row in registers, two runs of 4: as four pairs of fp32, and back with one rounding to
// nearest even.  TWO: the runs are apart (two accesses), otherwise they follow each other.
template <typename T>
struct Vec8 {
  uint32_t w[4];
  template <bool TWO>
  __device__ __forceinline__ void load(const T* p, int second) {
    if (TWO) {
      const uint2 x = *reinterpret_cast<const uint2*>(p), y = *reinterpret_cast<const uint2*>(p + second);
      w[0] = x.x, w[1] = x.y, w[2] = y.x, w[3] = y.y;
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
  template <bool TWO>
  __device__ __forceinline__ void store(T* p, int second) const {
    if (TWO) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(p + second) = make_uint2(w[2], w[3]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ uint64_t pair(int i) const;
  __device__ __forceinline__ void set(int i, uint64_t p);
};
template <>
__device__ __forceinline__ uint64_t Vec8<__nv_bfloat16>::pair(int i) const {
  return pair_f32(w[i] << 16, w[i] & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void Vec8<__nv_bfloat16>::set(int i, uint64_t p) {
  const float2 f = unpair_f32(p);
  w[i] = pack_bf16x2(f.x, f.y);
}
template <>
__device__ __forceinline__ uint64_t Vec8<__half>::pair(int i) const {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
  return pair_f32(f.x, f.y);
}
template <>
__device__ __forceinline__ void Vec8<__half>::set(int i, uint64_t p) {
  const float2 f = unpair_f32(p);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  w[i] = *reinterpret_cast<const uint32_t*>(&h);
}
template <>
struct Vec8<float> {
  float4 a, b;
  template <bool TWO>
  __device__ __forceinline__ void load(const float* p, int second) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + (TWO ? second : 4));
  }
  template <bool TWO>
  __device__ __forceinline__ void store(float* p, int second) const {
    *reinterpret_cast<float4*>(p) = a;
    *reinterpret_cast<float4*>(p + (TWO ? second : 4)) = b;
  }
  __device__ __forceinline__ uint64_t pair(int i) const {
    return i == 0 ? pair_f32(a.x, a.y) : i == 1 ? pair_f32(a.z, a.w) : i == 2 ? pair_f32(b.x, b.y) : pair_f32(b.z, b.w);
  }
  __device__ __forceinline__ void set(int i, uint64_t p) {
    const float2 f = unpair_f32(p);
    if (i == 0) a.x = f.x, a.y = f.y;
    if (i == 1) a.z = f.x, a.w = f.y;
    if (i == 2) b.x = f.x, b.y = f.y;
    if (i == 3) b.z = f.x, b.w = f.y;
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

// A head of D elements is spread over L = D / 8 lanes, 8 elements each, so a warp takes 32 / L heads
// at a time and a mean of squares is log2(L) shuffles.  A lane holds whole pairs: neighbours are 8
// consecutive elements; with the half-split pairing a lane has 4 elements of the first half of the
// rotated dims and their 4 partners of the second (or 8 dims that are not rotated).  One or, where
// tokens are few, several warps take a token.  A warp asks for the first rows, then computes the
// cos and sin of the token's rotated pairs under those loads, one or more pairs per lane, and hands
// them round through shared memory: the angle is position * frequency in turns, reduced to
// [-1/2, 1/2] in fp64 (an fp32 angle of position 10^6 is off by 0.06 rad), then sincospi in fp32.
// Weight and rotation of a lane's elements become two factors each, kept for all heads of the
// token:  y = rsqrt(mean) * (A x + B x'),  x' the other element of the pair.
// Bound by HBM and by instructions at once: 36,864 tokens of 32 heads x 64 (302 MB) take
// 57 us, 5.3 TB/s with 70 % of the issue slots busy (63 us when the partners of the half-split pairs came by
// shuffle; more warps per SM with fewer rows in flight 72, fewer with more rows 71).
template <typename T, int D, bool INTERLEAVED, bool NORM>
__global__ void __launch_bounds__(kRopeWarps * 32, 4) qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = D / 8;
  constexpr int HPI = 32 / L;                // heads per warp and row group
  constexpr int U = sizeof(T) == 4 ? 2 : 4;  // row groups in flight
  constexpr bool TWO = !INTERLEAVED;
  __shared__ __align__(16) float s_cos[kRopeWarps][D / 2], s_sin[kRopeWarps][D / 2];
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wpt = a.warps_per_token;
  const long long t = static_cast<long long>(blockIdx.x) * (kRopeWarps / wpt) + warp / wpt;
  const int part = warp % wpt;
  if (t >= a.tokens) return;
  const int j = lane % L, sub = lane / L;
  const int pairs = a.pair_end[a.axes - 1];
  // this lane's elements: two runs of 4 at `first` and `first + second`, rotated by pairs pair0 ..
  const int turning = pairs / 4;  // half-split: lanes with rotated dims (pairs % 8 == 0)
  const int first = INTERLEAVED ? 8 * j : j < turning ? 4 * j : 2 * pairs + 8 * (j - turning);
  const int second = INTERLEAVED || j >= turning ? 4 : pairs;
  pdl_wait();
  Vec8<T> in[U];
  // row groups part, part + wpt, ... of a token's heads
  auto ask = [&](const T* p, long long hs, int heads, int g0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = (g0 + u * wpt) * HPI + sub;
      if (r < heads) in[u].template load<TWO>(p + r * hs, second);
    }
  };
  const T* qp = static_cast<const T*>(a.q) + t * a.q_ts + first;
  const T* kp = static_cast<const T*>(a.k) + t * a.k_ts + first;
  ask(qp, a.q_hs, a.heads, part);

  for (int p = lane; p < D / 2; p += 32) {
    float cs = 1.0f, sn = 0.0f;
    if (p < pairs) {
      int ax = 0;
#pragma unroll
      for (int i = 0; i + 1 < OASIS_MAX_AXES; ++i) ax += i + 1 < a.axes && p >= a.pair_end[i];
      const long long at = t * a.axes + ax;
      const double pos = a.positions_64 ? static_cast<double>(static_cast<const int64_t*>(a.positions)[at])
                                        : static_cast<double>(static_cast<const int32_t*>(a.positions)[at]);
      const double turns = pos * a.freqs[p] * 0.15915494309189533577;  // 1 / (2 pi)
      const float frac = static_cast<float>(turns - rint(turns));
      sincospif(2.0f * frac, &sn, &cs);
    }
    s_cos[warp][p] = cs;
    s_sin[warp][p] = sn;
  }
  long long slot_off = 0, slot_hs = 0;  // element offset of head 0 of the token's slot in the pages
  bool stored = true;
  if (a.slots) {
    const int s = a.slots[t];
    stored = s >= 0 && s < a.n_slots;
    const int page = s / a.page_tokens;
    slot_off = (static_cast<long long>(page) * a.kv_heads * a.page_tokens + (s - page * a.page_tokens)) * D;
    slot_hs = static_cast<long long>(a.page_tokens) * D;
  }
  __syncwarp();
  const bool turns_here = INTERLEAVED || j < turning;

  auto pass = [&](const T* src, long long hs, T* dst, long long dst_hs, int heads, const float* weight, bool keep,
                  bool asked) {
    uint64_t fa[4], fb[4];
    {
      float4 w0 = make_float4(1.0f, 1.0f, 1.0f, 1.0f), w1 = w0, c = w0, s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (NORM && weight) {
        w0 = *reinterpret_cast<const float4*>(weight + first);
        w1 = *reinterpret_cast<const float4*>(weight + first + second);
      }
      if (turns_here) {
        c = *reinterpret_cast<const float4*>(&s_cos[warp][4 * j]);
        s = *reinterpret_cast<const float4*>(&s_sin[warp][4 * j]);
      }
      if (INTERLEAVED) {  // pairs (0, 1) (2, 3) ..: a cos - b sin, b cos + a sin
        fa[0] = pair_f32(w0.x * c.x, w0.y * c.x), fb[0] = pair_f32(-w0.y * s.x, w0.x * s.x);
        fa[1] = pair_f32(w0.z * c.y, w0.w * c.y), fb[1] = pair_f32(-w0.w * s.y, w0.z * s.y);
        fa[2] = pair_f32(w1.x * c.z, w1.y * c.z), fb[2] = pair_f32(-w1.y * s.z, w1.x * s.z);
        fa[3] = pair_f32(w1.z * c.w, w1.w * c.w), fb[3] = pair_f32(-w1.w * s.w, w1.z * s.w);
      } else {  // pairs (0, 4) (1, 5) ..
        fa[0] = pair_f32(w0.x * c.x, w0.y * c.y), fa[1] = pair_f32(w0.z * c.z, w0.w * c.w);
        fa[2] = pair_f32(w1.x * c.x, w1.y * c.y), fa[3] = pair_f32(w1.z * c.z, w1.w * c.w);
        fb[0] = pair_f32(-w1.x * s.x, -w1.y * s.y), fb[1] = pair_f32(-w1.z * s.z, -w1.w * s.w);
        fb[2] = pair_f32(w0.x * s.x, w0.y * s.y), fb[3] = pair_f32(w0.z * s.z, w0.w * s.w);
      }
    }
    for (int g0 = part; g0 * HPI < heads; g0 += U * wpt) {
      if (g0 != part || !asked) ask(src, hs, heads, g0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r0 = (g0 + u * wpt) * HPI, r = r0 + sub;
        if (r0 >= heads) break;  // warp-uniform
        uint64_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = in[u].pair(i);
        uint64_t scale = 0;
        if (NORM) {
          uint64_t sq = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) sq = fma_f32x2(x[i], x[i], sq);
          const float2 s2 = unpair_f32(sq);
          float ss = s2.x + s2.y;
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float rs = rsqrtf(ss * (1.0f / D) + a.eps);
          scale = pair_f32(rs, rs);
        }
        Vec8<T> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint64_t y = mul_f32x2(x[i], fa[i]);
          if (INTERLEAVED) {
            const float2 f = unpair_f32(x[i]);
            if (4 * j + i < pairs) y = fma_f32x2(pair_f32(f.y, f.x), fb[i], y);
          } else if (turns_here) {
            y = fma_f32x2(x[i ^ 2], fb[i], y);
          }
          out.set(i, NORM ? mul_f32x2(y, scale) : y);
        }
        if (r < heads && keep) out.template store<TWO>(dst + r * dst_hs, second);
      }
    }
  };
  pass(qp, a.q_hs, static_cast<T*>(a.q_out) + t * a.qo_ts + first, a.qo_hs, a.heads, a.qw, true, true);
  pass(kp, a.k_hs, static_cast<T*>(a.k_out) + (a.slots ? slot_off : t * a.ko_ts) + first, a.slots ? slot_hs : a.ko_hs,
       a.kv_heads, a.kw, stored, false);
  if (a.slots && stored) {
    const T* vp = static_cast<const T*>(a.v) + t * a.v_ts + first;
    T* vo = static_cast<T*>(a.v_out) + slot_off + first;
    for (int g0 = part; g0 * HPI < a.kv_heads; g0 += U * wpt) {
      ask(vp, a.v_hs, a.kv_heads, g0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = (g0 + u * wpt) * HPI + sub;
        if (r < a.kv_heads) in[u].template store<TWO>(vo + r * slot_hs, second);
      }
    }
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
    const uintptr_t kb = reinterpret_cast<uintptr_t>(p->pages->k), vb = reinterpret_cast<uintptr_t>(p->pages->v);
    const uintptr_t pool = static_cast<uintptr_t>(p->pages->pages) * p->pages->kv_heads * p->pages->page_tokens * d * 2;
    if (kb < vb + pool && vb < kb + pool)
      return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": key and value pages overlap");
  } else if (!p->k_out) {
    return fail(OASIS_ERR_INVALID_ARG, std::string(who) + ": null pointer");
  }
  if ((p->q_weight && !aligned16(p->q_weight)) || (p->k_weight && !aligned16(p->k_weight)))
    return fail(OASIS_ERR_ALIGNMENT, std::string(who) + ": weights must be 16-byte aligned");
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
  // few tokens: several warps share one, so that its heads run side by side; a warp has a group of
  // heads at least (4,609 tokens of 32 fp32 heads x 128: two warps took 29.5 us where one took 35)
  const int groups = (std::max(p->heads, p->kv_heads) * d + 255) / 256;
  a.warps_per_token = 1;
  while (2 * a.warps_per_token <= std::min(kRopeWarps, groups) &&
         static_cast<long long>(p->tokens) * a.warps_per_token < 48LL * num_sms())
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
