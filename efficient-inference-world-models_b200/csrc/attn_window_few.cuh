// Window attention for few query rows (single tokens): at most NR = 8 or 16 rows of one (sequence,
// key head) at a time, split over the keys.  Included by attn_window.cu.
//
// Bound by HBM: every visible key and value is read once, straight into the registers of the
// mma.sync fragments that use it (no shared memory, no barriers in the loop), so the loads in
// flight are limited by registers only (12 warps of 8 KB per SM at D = 128, NR = 8).
// A warp takes 16 keys at a time (they lie in one page) from a run of its own:
//   S = Q K^T    Q the A operand (rows g, g + 8), key 8t + g the B columns; thread (g, c) of the warp
//                supplies 16-byte chunks c, c + 4, ... of its key, and Q takes the same order of dims;
//   O^T = V^T P^T  P's accumulators are the B operand as they stand; thread (g, c) supplies keys
//                2c, 2c+1, 2c+8, 2c+9 and dims 8g .. 8g+7 (+64), paired by byte permutes.
// The warps of a CTA (NW), then the CTAs of a cluster (up to 16, over distributed shared memory), join
// their maxima, sums and O in a fixed order: no workspace and no second launch.
#pragma once

namespace oasis {

constexpr int kFewSplits = 16;  // CTAs of a cluster, at most (above 8: where the device takes such clusters)

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a page, read once: not kept in L1.  (A plain load, not one through the read-only path: with
// dependent launches the kernel that appends to the pages may still run when this one starts.)
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <int D, int NR, int NW>
struct alignas(16) FewShared {
  float o[NW][NR][D];
  float m[NW][NR], l[NW][NR];
  // from the CTAs of the cluster: maxima and sums of all rows, and of this CTA's share of O, 4 dims
  // of a row at a time, unit e of the whole in place e / CTAs of CTA e % CTAs
  float cm[kFewSplits][NR], cl[kFewSplits][NR];
  float4 co[NR * D / 4 + kFewSplits];
  uint32_t marks[kFewSplits];
  uint32_t dirty;
};

template <typename T, int D, int NR, int NW>
__global__ void __launch_bounds__(NW * 32, NW == 8 ? 1 : D == 64 ? (NR == 8 ? 4 : 3) : (NR == 8 ? 3 : 2))
    attn_window_few_kernel(const __grid_constant__ WinArgs a, int splits) {
  constexpr int KC = D / 32;  // 16-byte chunks of a key per thread
  constexpr int VC = D / 64;  // of a value
  constexpr int RT = NR / 8;
  __shared__ FewShared<D, NR, NW> sh;
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int split = static_cast<int>(blockIdx.x) % splits;  // rank in the cluster
  const int kvh = static_cast<int>(blockIdx.x) / splits;
  const int b = blockIdx.z;
  if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA is here
  pdl_wait();
  const WinSeq seq = win_seq(a, b);
  const int rows = seq.n_q * a.group;
  const int32_t* table = a.table + static_cast<long long>(b) * a.width;
  const float sl2 = a.scale_log2;

  for (int row0 = 0; row0 < rows; row0 += NR) {  // one turn, unless the launch was told of fewer rows
    const int row1 = min(rows, row0 + NR);
    const WtSpan span = wt_span(a, seq, row0, row1);
    const WtTiles steps = wt_tiles(span, 16);
    if (threadIdx.x == 0) sh.dirty = 0;
    __syncthreads();
    // the rows of this thread's accumulators and what they see
    WinRange range[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = row0 + g + 8 * t;
      range[t] = r < row1 ? win_range(a, seq.kv - seq.n_q + a.by_group.div(r), seq.kv) : WinRange{0, 0, 0};
    }
    uint4 q[RT][KC];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = row0 + g + 8 * t;
#pragma unroll
      for (int i = 0; i < KC; ++i) {
        q[t][i] = make_uint4(0, 0, 0, 0);
        if (r < row1)
          q[t][i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                    static_cast<long long>(seq.q0 + a.by_group.div(r)) * a.q_ts +
                                                    (kvh * a.group + a.by_group.mod(r)) * a.q_hs + (4 * i + c) * 8);
      }
    }
    float o[VC][4][RT][4];
#pragma unroll
    for (int i = 0; i < VC; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][u][t][x] = 0.0f;
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = -INFINITY;
      l[t] = 0.0f;
    }
    uint32_t dirty = 0;

    // this warp's run of steps
    const int part = split * NW + warp, parts = splits * NW;
    const int j0 = static_cast<int>(static_cast<long long>(steps.n) * part / parts);
    const int j1 = static_cast<int>(static_cast<long long>(steps.n) * (part + 1) / parts);
    uint4 kb[2][KC], vb[4][VC];
    auto look_up = [&](int j) {  // page of a step, -1: none
      const int idx = j < j1 ? a.by_page.div(steps.tile(j) * 16) : a.width;
      return idx < a.width ? table[idx] : -1;
    };
    auto base_of = [&](int j, int page) {  // first element of the step's first key
      const int at = a.by_page.mod(steps.tile(j) * 16);
      return ((static_cast<long long>(page) * a.kv_heads + kvh) * a.page_tokens + at) * D;
    };
    auto there = [&](int page) { return page >= 0 && page < a.pages; };
    auto load_k = [&](long long base) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < KC; ++i)
          kb[t][i] = ld_stream(static_cast<const T*>(a.k) + base + (8 * t + g) * D + (4 * i + c) * 8);
    };
    auto load_v = [&](long long base) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int i = 0; i < VC; ++i)
          vb[x][i] = ld_stream(static_cast<const T*>(a.v) + base + (2 * c + (x & 1) + 8 * (x >> 1)) * D + (8 * i + g) * 8);
    };
    int page = look_up(j0), next_page = look_up(j0 + 1);
    long long base = 0;
    if (j0 < j1 && there(page)) {
      base = base_of(j0, page);
      load_k(base);
      load_v(base);
    }
    for (int j = j0; j < j1; ++j) {
      const int key0 = steps.tile(j) * 16;
      const bool have = there(page);
      const bool have_next = j + 1 < j1 && there(next_page);
      const long long next_base = have_next ? base_of(j + 1, next_page) : 0;
      const int after = look_up(j + 2);
      float s[2][RT][4];
      if (have) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            const uint4 z = make_uint4(0, 0, 0, 0);
            const uint4 qa = q[0][i], qb = RT == 2 ? q[RT - 1][i] : z;
            mma_16816<T>(acc, qa.x, qb.x, qa.y, qb.y, kb[t][i].x, kb[t][i].y);
            mma_16816<T>(acc, qa.z, qb.z, qa.w, qb.w, kb[t][i].z, kb[t][i].w);
          }
          s[t][0][0] = acc[0];
          s[t][0][1] = acc[1];
          if (RT == 2) {
            s[t][RT - 1][0] = acc[2];
            s[t][RT - 1][1] = acc[3];
          }
        }
      }
      if (have_next) load_k(next_base);
      if (have) {
        if (!span.all(key0, key0 + 16)) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if (!range[rt].sees(key0 + 8 * t + 2 * c + x)) s[t][rt][x] = -INFINITY;
          // 0 * NaN is not 0: values that no row sees are zeroed, and an infinity or NaN that
          // only some of the rows see has the rows computed one by one
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = key0 + 2 * c + (x & 1) + 8 * (x >> 1);
            if (span.all(key, key + 1)) continue;
            const bool seen = span.sees(key);
#pragma unroll
            for (int i = 0; i < VC; ++i) {
              if (!seen) vb[x][i] = make_uint4(0, 0, 0, 0);
              dirty |= nonfinite2<T>(vb[x][i].x) | nonfinite2<T>(vb[x][i].y) | nonfinite2<T>(vb[x][i].z) |
                       nonfinite2<T>(vb[x][i].w);
            }
          }
        }
        // running maximum, moved when it grows by more than 2^8 (as in the tile kernel)
        bool grow = false;
        float top[RT], alpha[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          float x = max3_nan(max3_nan(s[0][rt][0], s[0][rt][1], s[1][rt][0]), s[1][rt][1], s[1][rt][1]);
          float y = __shfl_xor_sync(0xffffffffu, x, 1);
          x = max3_nan(x, y, y);
          y = __shfl_xor_sync(0xffffffffu, x, 2);
          top[rt] = max3_nan(x, y, y);
          const bool up = !((top[rt] - m[rt]) * sl2 <= kWtLazy) && top[rt] != -INFINITY;
          alpha[rt] = 1.0f;
          if (up) {
            alpha[rt] = ex2((m[rt] - top[rt]) * sl2);
            m[rt] = top[rt];
            l[rt] *= alpha[rt];
          }
          grow = grow || up;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {  // the columns of O^T are rows 2c and 2c + 1
            const float a0 = __shfl_sync(0xffffffffu, alpha[rt], 8 * c), a1 = __shfl_sync(0xffffffffu, alpha[rt], 8 * c + 4);
#pragma unroll
            for (int i = 0; i < VC; ++i)
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                o[i][u][rt][0] *= a0;
                o[i][u][rt][1] *= a1;
                o[i][u][rt][2] *= a0;
                o[i][u][rt][3] *= a1;
              }
          }
        }
        uint32_t p[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float off = m[rt] == -INFINITY ? 0.0f : fmaf(m[rt], 0.0f, -m[rt] * sl2);  // NaN for +inf
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float e0 = ex2(fmaf(s[t][rt][0], sl2, off)), e1 = ex2(fmaf(s[t][rt][1], sl2, off));
            l[rt] += e0 + e1;
            p[rt][t] = pack2<T>(e0, e1);
          }
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          const uint32_t w[4][4] = {{vb[0][i].x, vb[0][i].y, vb[0][i].z, vb[0][i].w},
                                    {vb[1][i].x, vb[1][i].y, vb[1][i].z, vb[1][i].w},
                                    {vb[2][i].x, vb[2][i].y, vb[2][i].z, vb[2][i].w},
                                    {vb[3][i].x, vb[3][i].y, vb[3][i].z, vb[3][i].w}};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t a0 = __byte_perm(w[0][u], w[1][u], 0x5410), a1 = __byte_perm(w[0][u], w[1][u], 0x7632);
            const uint32_t a2 = __byte_perm(w[2][u], w[3][u], 0x5410), a3 = __byte_perm(w[2][u], w[3][u], 0x7632);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) mma_16816<T>(o[i][u][rt], a0, a1, a2, a3, p[rt][0], p[rt][1]);
          }
        }
      }
      if (have_next) load_v(next_base);
      page = next_page;
      next_page = after;
    }

    // ---- join: warps of the CTA
    if (dirty) sh.dirty = 1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 1);
      l[rt] += __shfl_xor_sync(0xffffffffu, l[rt], 2);
      if (c == 0) {
        sh.m[warp][8 * rt + g] = m[rt];
        sh.l[warp][8 * rt + g] = l[rt];
      }
#pragma unroll
      for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // row 8 rt + 2c + x, dims 64 i + 8 g ..
          float* dst = &sh.o[warp][8 * rt + 2 * c + x][64 * i + 8 * g];
          *reinterpret_cast<float4*>(dst) = make_float4(o[i][0][rt][x], o[i][0][rt][x + 2], o[i][1][rt][x], o[i][1][rt][x + 2]);
          *reinterpret_cast<float4*>(dst + 4) =
              make_float4(o[i][2][rt][x], o[i][2][rt][x + 2], o[i][3][rt][x], o[i][3][rt][x + 2]);
        }
    }
    __syncthreads();
    // weight of a partial result of maximum x under the joint maximum y
    auto weight = [&](float x, float y) { return x == -INFINITY ? 0.0f : ex2((x - y) * sl2); };
    auto join_max = [](float x, float y) { return max3_nan(x, y, y); };
    // what the others may write to: the CTAs are all here, and done with an earlier turn's parts
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int units = (row1 - row0) * (D / 4), share = (units + splits - 1) / splits;
    for (int e = threadIdx.x; e < units; e += NW * 32) {
      const int r = e / (D / 4), d = (e % (D / 4)) * 4;
      float top = sh.m[0][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) top = join_max(top, sh.m[w][r]);
      float sum = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = weight(sh.m[w][r], top);
        const float4 x = *reinterpret_cast<const float4*>(&sh.o[w][r][d]);
        sum += f * sh.l[w][r];
        acc.x = fmaf(f, x.x, acc.x), acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z), acc.w = fmaf(f, x.w, acc.w);
      }
      // sent to its owner (stores need no answer, loads from the others would wait for theirs)
      const int owner = e % splits;
      st_cluster4(mapa_shared(smem_u32(&sh.co[split * share + e / splits]), owner), __float_as_uint(acc.x),
                  __float_as_uint(acc.y), __float_as_uint(acc.z), __float_as_uint(acc.w));
      if (d == 0)
        for (int x = 0; x < splits; ++x) {
          st_cluster(mapa_shared(smem_u32(&sh.cm[split][r]), x), top);
          st_cluster(mapa_shared(smem_u32(&sh.cl[split][r]), x), sum);
        }
    }
    if (threadIdx.x < splits)
      st_cluster(mapa_shared(smem_u32(&sh.marks[split]), threadIdx.x),
                 __uint_as_float(*reinterpret_cast<volatile uint32_t*>(&sh.dirty)));
    __syncwarp();
    if (splits > 1)
      cluster_sync_all();
    else
      __syncthreads();
    // ---- and CTAs of the cluster, in rank order
    uint32_t marked = 0;
    for (int x = 0; x < splits; ++x) marked |= sh.marks[x];
    if (marked) {
      for (int r = row0 + part; r < row1; r += parts)
        window_row<T, D>(a, b, seq, a.by_group.div(r), kvh * a.group + a.by_group.mod(r), lane);
    } else {
      for (int i = threadIdx.x; i * splits + split < units; i += NW * 32) {
        const int e = i * splits + split;
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        float top = -INFINITY;
        for (int x = 0; x < splits; ++x) top = join_max(top, sh.cm[x][r]);
        float sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int x = 0; x < splits; ++x) {
          const float f = weight(sh.cm[x][r], top);
          const float4 z = sh.co[x * share + i];
          sum += f * sh.cl[x][r];
          acc.x = fmaf(f, z.x, acc.x), acc.y = fmaf(f, z.y, acc.y);
          acc.z = fmaf(f, z.z, acc.z), acc.w = fmaf(f, z.w, acc.w);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int qr = row0 + r;
        const long long tok = seq.q0 + a.by_group.div(qr);
        const int head = kvh * a.group + a.by_group.mod(qr);
        const bool none = sum == 0.0f;
        uint2 w2 = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        if (none) w2 = make_uint2(0, 0);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + d) = w2;
        if (a.lse && d == 0) a.lse[tok * a.heads + head] = none ? -INFINITY : (top * sl2 + log2f(sum)) * 0.6931471805599453f;
      }
    }
    __syncwarp();
    if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // done with the parts
    __syncthreads();
  }
  if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the last arrival's
}

}  // namespace oasis
