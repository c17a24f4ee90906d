// Window attention for prompts and frames: 256 query rows of one (sequence, key head) per CTA
// on tcgen05, keys and values by TMA.  Included by attn_window.cu.
//
// Rows are the queries of the key head's group, token-major (row r: token r / group, head
// r % group), so grouped heads share every key tile.  A CTA holds two tiles of 128 rows.
// Roles: warps 0-3 and 4-7 are the softmax of tile 0 and 1 (one row per thread, S read from
// TMEM); warp 8 issues the MMAs; warps 9 and 10 load K and V tiles of 128 keys page by page;
// warp 11 looks over the V tiles that some row sees only in part.
//
// For tile i and key tile j:  S_i = Q_i K_j^T (TMEM, 128 columns), the softmax thread takes
// P = exp2(S * scale - m) and writes it in 16 bits over S, O_i += P_i V_j (P from TMEM).  The MMA warp
// alternates PV_0(j), QK_0(j+1), PV_1(j), QK_1(j+1): while one tile's softmax runs, the tensor
// cores work for the other.  At D = 64 there is room for P beside S, and S_i(j+1) is computed while
// softmax i works on tile j.  m is the running maximum (Milakov and Gimelshein, "Online normalizer
// calculation for softmax", 2018), moved (and O rescaled) only when it grows by more than 2^8, which keeps
// every p below 2^8 and the sum exact to fp32.
#pragma once

namespace oasis {

constexpr int kWtRows = 128;     // query rows of a tile
constexpr int kWtKeys = 128;     // keys of a K/V tile
constexpr int kWtThreads = 384;  // 8 softmax warps, MMA, K loads, V loads, V looked over
constexpr int kWtRegs = 168;     // per thread at launch (which checks it); the softmax warps take from the others
constexpr float kWtLazy = 8.0f;  // log2 of how far scores may pass the maximum in use
constexpr int kWtClean = 0x7fffffff;

template <int D>
struct WtShape {
  static constexpr int kHalf = kWtKeys * 128;              // 16 KB: 128 rows of 64 elements
  static constexpr int kTile = kHalf * (D / 64);           // one Q, K or V tile
  // a K tile is done with a step before the V tile of the same keys: fewer of them
  static constexpr int kStagesK = D == 128 ? 2 : 4, kStagesV = D == 128 ? 3 : 4;
  static constexpr int kStages = kStagesK + kStagesV;
  static constexpr int kBars = 3 * kStages + 12;
  // D = 64 leaves TMEM columns for P beside S: the next S is then computed under the softmax
  static constexpr bool kEarly = D == 64;
  // quarters of P that the MMAs get before the rest is there: with two or three, 384 or 399 us for a
  // prompt of 8,191 tokens at D = 128 (short bursts; sustained 439), 77 or 71 us for 8 sessions' frames at D = 64
  static constexpr int kHandover = kEarly ? 3 : 2;
  // registers of a softmax and of a helping thread: the prompt takes 390 us with 208 and 88, 8 sessions'
  // frames 80 (the compiler orders the softmax by what it has)
  static constexpr int kSoftRegs = D == 128 ? 200 : 216, kHelpRegs = D == 128 ? 104 : 72;
  static_assert(256 * kSoftRegs + 128 * kHelpRegs <= kWtThreads * kWtRegs, "registers of the block");
  static constexpr int kO = 256, kP = kEarly ? kO + 2 * D : 0, kPStep = kEarly ? 64 : 128;  // columns of tile 0, 1
  static constexpr int kSmem = (2 + kStages) * kTile + 1024 + 256 + 8 * kBars;
};

// V tile as an MN-major operand: blocks of 64 dims (one swizzle atom) kHalf bytes apart.
__device__ __forceinline__ uint64_t wt_v_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((kWtKeys * 128) >> 4) << 16;  // leading byte offset: next 64 dims
  d |= static_cast<uint64_t>(1024u >> 4) << 32;            // stride byte offset: next 8 keys
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;  // SWIZZLE_128B
  return d;
}

// Register shares within a block (WtShape).
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// D (+)= A B^T with A from shared memory, and with A (P, K-major) from TMEM.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// 32 columns of this warp's 32 lanes, not waited for.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The registers pass through the wait, so that nothing reads them before it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31])::"memory");
}
// Waits for the stores so far, after `r` has been computed.
__device__ __forceinline__ void tmem_wait_st(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::st.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The larger of three; NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Bits lo..hi-1 of a word, both clamped to it.
__device__ __forceinline__ uint32_t wt_bits(int lo, int hi) {
  lo = max(0, min(lo, 32));
  hi = max(0, min(hi, 32));
  const uint32_t below_hi = hi == 32 ? ~0u : (1u << hi) - 1u, below_lo = lo == 32 ? ~0u : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}
__device__ __forceinline__ void wt_hide(uint32_t (&v)[32], uint32_t seen) {
#pragma unroll
  for (int x = 0; x < 32; ++x)
    if (!((seen >> x) & 1u)) v[x] = 0xff800000u;  // -inf
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Non-zero if one of the two 16-bit values of a word is an infinity or NaN: its magnitude is at least
// that of infinity, and then what is missing to 2^15 carries into the sign bit.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  constexpr uint32_t gap = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return ((w & 0x7FFF7FFFu) + gap) & 0x80008000u;
}

// Instruction descriptor of kind::f16 for this type: fp32 D, A K-major, B K-major or (b_mn) MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t umma_idesc(int m, int n, bool b_mn) {
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? (1u << 16) : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// What a run of rows of one CTA sees, from the ranges of its first and last row (both ends of a
// row's range only grow from row to row).
struct WtSpan {
  WinRange lo, hi;
  bool any;
  __device__ __forceinline__ bool all(int k0, int k1) const {  // every row sees all of [k0, k1)
    return k1 <= lo.end && (k0 >= hi.start || k1 <= lo.sink_end);
  }
  __device__ __forceinline__ bool some(int k0, int k1) const {  // some row may see some of it
    return any && k0 < hi.end && (k1 > lo.start || k0 < hi.sink_end);
  }
  __device__ __forceinline__ bool sees(int key) const {
    return key < hi.end && (key >= lo.start || key < hi.sink_end);
  }
};
__device__ __forceinline__ WtSpan wt_span(const WinArgs& a, const WinSeq& s, int row0, int row1) {
  WtSpan w;
  const int base = s.kv - s.n_q;
  const int p1 = base + a.by_group.div(max(row1 - 1, 0));
  w.any = row0 < row1 && p1 >= 0;
  w.lo = win_range(a, base + a.by_group.div(row0), s.kv);  // all zero where the position is negative
  w.hi = win_range(a, p1, s.kv);
  return w;
}

// The key tiles of a span: [0, sink) and [first, last).
struct WtTiles {
  int sink, first, n, skip;
  __device__ __forceinline__ int tile(int j) const { return j < sink ? skip + j : first + j - sink; }
  // The part of them that CTA `rank` of `parts` takes, numbered from 0.
  __device__ __forceinline__ void keep(int rank, int parts) {
    const int j0 = n * rank / parts, j1 = n * (rank + 1) / parts;
    sink -= j0;  // negative: all of the part lies in the window
    skip = j0;
    n = j1 - j0;
  }
};
__device__ __forceinline__ WtTiles wt_tiles(const WtSpan& w, int keys) {
  WtTiles t = {0, 0, 0, 0};
  if (!w.any) return t;
  t.sink = (min(w.hi.sink_end, w.lo.start) + keys - 1) / keys;
  t.first = max(w.lo.start / keys, t.sink);
  t.n = t.sink + max(0, (w.hi.end + keys - 1) / keys - t.first);
  return t;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWtThreads, 1)
    attn_window_tile_kernel(const __grid_constant__ WinArgs a, const __grid_constant__ CUtensorMap tm_k,
                            const __grid_constant__ CUtensorMap tm_v, int box_rows, int row_tiles, int splits) {
  using S = WtShape<D>;
  constexpr int kStages = S::kStages, kSK = S::kStagesK, kSV = S::kStagesV;  // slots: K, then V
  extern __shared__ uint8_t wt_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(wt_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* ring = sQ + 2 * S::kTile;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kStages * S::kTile);
  uint64_t* clean = full + kStages;
  uint64_t* empty = clean + kStages;
  uint64_t* q_full = empty + kStages;
  uint64_t* s_full = q_full + 1;   // [2]
  uint64_t* p_full = s_full + 2;   // [2]
  uint64_t* p_half = p_full + 2;   // [2]
  uint64_t* pv_done = p_half + 2;  // [2]
  uint64_t* s_free = pv_done + 2;  // [2] (kEarly)
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(s_free + 2);
  int* dirty = reinterpret_cast<int*>(tmem_holder + 1);  // kWtClean, or the first key of the first marked V tile

  pdl_trigger();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&clean[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_half[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&s_free[i], 4);
    }
    *dirty = kWtClean;
    mbar_fence_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 8) tmem_alloc<512>(tmem_holder);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  pdl_wait();

  const int b = blockIdx.z;
  const WinSeq seq = win_seq(a, b);
  const int rows = seq.n_q * a.group;
  // later rows of a causal prompt see more: they start first
  const int rank = static_cast<int>(blockIdx.x) % splits;  // in the cluster, which shares the keys
  const int unit = static_cast<int>(blockIdx.x) / splits;
  const int tile_id = row_tiles - 1 - unit / a.kv_heads;
  const int kvh = unit % a.kv_heads;
  const int row0 = tile_id * (2 * kWtRows);
  const int32_t* table = a.table + static_cast<long long>(b) * a.width;
  const int row1 = min(rows, row0 + 2 * kWtRows);
  const WtSpan span = wt_span(a, seq, row0, row1);
  const WtSpan half[2] = {wt_span(a, seq, row0, min(row1, row0 + kWtRows)),
                          wt_span(a, seq, min(row1, row0 + kWtRows), row1)};
  WtTiles tiles = wt_tiles(span, kWtKeys);
  tiles.keep(rank, splits);
  const int n = tiles.n;
  // The parts that the CTAs of a cluster send each other, over the ring once all are done with it:
  // of every CTA, for this one's share of the rows, O [share][D] fp32 (16-byte chunks swizzled by
  // row), the rows' maxima and sums, and the mark of warp 11.
  const int share = (row1 - row0 + splits - 1) / splits;
  float* part_o = reinterpret_cast<float*>(ring);
  float* part_m = part_o + splits * share * D;
  float* part_l = part_m + splits * share;
  int* part_mark = reinterpret_cast<int*>(part_l + splits * share);
  static_assert((2 * kWtRows + kWinSplits) * (D + 2) * 4 + kWinSplits * 4 <= kStages * S::kTile,
                "the ring holds a CTA's share of all parts");
  float m = -INFINITY, l = 0.0f;  // of a softmax thread's row
  uint32_t np = 0;
  bool ok = true;

  if (warp >= 8) {
    reg_dec<S::kHelpRegs>();
    if (row0 >= rows) {
      // nothing to do
    } else if (warp == 9 || warp == 10) {
      // -------------------------------------------------------------- loads: warp 9 K, warp 10 V
      const bool is_k = warp == 9;
      const int ring0 = is_k ? 0 : kSK, slots = is_k ? kSK : kSV;
      const int boxes = kWtKeys / box_rows;
      const int none = a.pages * a.kv_heads * a.page_tokens;  // beyond the pages: zeros
      auto box_row = [&](int j) {  // lane x takes box x
        const int key = tiles.tile(j) * kWtKeys + lane * box_rows;
        const int idx = a.by_page.div(key);
        const int page = idx < a.width ? table[idx] : -1;
        return page >= 0 && page < a.pages ? (page * a.kv_heads + kvh) * a.page_tokens + (key - idx * a.page_tokens)
                                           : none;
      };
      auto load = [&](int j, int row) {
        const int slot = ring0 + j % slots;
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], S::kTile);
        __syncwarp();
        if (lane < boxes) {
          uint8_t* dst = ring + slot * S::kTile + lane * box_rows * 128;
          // (two calls: a selected pointer would make the compiler copy the maps to the stack)
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            if (is_k)
              tma_load_2d(dst + h * S::kHalf, &tm_k, &full[slot], h * 64, row);
            else
              tma_load_2d(dst + h * S::kHalf, &tm_v, &full[slot], h * 64, row);
          }
        }
        __syncwarp();
      };
      bool ok = true;
      int j = 0, row = n > 0 ? box_row(0) : none;
      for (; j < n; ++j) {
        const int next = j + 1 < n ? box_row(j + 1) : none;  // looked up under the wait
        if (j >= slots) ok = __all_sync(0xffffffffu, mbar_wait(&empty[ring0 + j % slots], (j / slots - 1) & 1));
        if (!ok) break;
        load(j, row);
        row = next;
      }
      if (!ok)  // gave up: let the copies in flight land before the memory is given back
        for (int i = max(0, j - slots); i < j; ++i) mbar_wait(&full[ring0 + i % slots], (i / slots) & 1);
    } else if (warp == 11) {
      // -------------------------------------------------------------- V tiles seen in part
      // A V tile that some query does not see whole is looked over before the MMAs may have it:
      // rows that no query of this CTA sees (ends of pages, tokens before the window) are zeroed, since
      // their weights are 0 but 0 * NaN is not; an infinity or NaN in a row that only some queries
      // see marks the CTA with the tile's first key (the first such tile's, as keys go up).  A query tile
      // that sees as far computes its rows one by one (window_row); one that ends before must not depend
      // on whether this warp is ahead of it.
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int st = kSK + j % kSV;
        const int k0 = tiles.tile(j) * kWtKeys;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (j / kSV) & 1));
        if (ok && !span.all(k0, k0 + kWtKeys)) {
          uint8_t* v = ring + st * S::kTile;
          uint32_t bad = 0;
#pragma unroll 1
          for (int r0 = 0; r0 < kWtKeys; r0 += 32) {
            if (span.all(k0 + r0, k0 + r0 + 32)) continue;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              uint4 x[8];  // 4 rows at a time, 8 loads in flight
#pragma unroll
              for (int u = 0; u < 8; ++u) {
                const int r = r0 + u * 4 + lane / 8;
                uint4* p = reinterpret_cast<uint4*>(v + h * S::kHalf + r * 128 + (lane % 8) * 16);
                x[u] = make_uint4(0, 0, 0, 0);
                if (!span.sees(k0 + r))
                  *p = x[u];
                else if (!span.all(k0 + r, k0 + r + 1))
                  x[u] = *p;
              }
#pragma unroll
              for (int u = 0; u < 8; ++u)
                bad |= nonfinite2<T>(x[u].x) | nonfinite2<T>(x[u].y) | nonfinite2<T>(x[u].z) | nonfinite2<T>(x[u].w);
            }
          }
          if (bad && *reinterpret_cast<volatile int*>(dirty) == kWtClean) *dirty = k0;
          fence_async_smem_cta();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&clean[st]);
      }
    } else {
      // -------------------------------------------------------------- MMA: one lane issues, the
      // warp stays converged, so that descriptors are warp-uniform values
      constexpr uint32_t idesc_s = umma_idesc<T>(kWtRows, kWtKeys, false);
      constexpr uint32_t idesc_o = umma_idesc<T>(kWtRows, D, true);
      const uint64_t q_desc = umma_desc_sw128(smem_u32(sQ)), k_desc = umma_desc_sw128(smem_u32(ring));
      const uint64_t v_desc = wt_v_desc(smem_u32(ring));
      constexpr uint64_t kTile16 = S::kTile >> 4, kHalf16 = S::kHalf >> 4;
      auto qk = [&](int i, int st) {
        const uint64_t qa = q_desc + i * kTile16, ka = k_desc + st * kTile16;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(tmem + i * 128, qa + (k >> 2) * kHalf16 + (k & 3) * 2, ka + (k >> 2) * kHalf16 + (k & 3) * 2, idesc_s,
                  k > 0);
      };
      auto pv = [&](int i, int st, auto first, auto last, uint32_t acc) {  // keys 16 first .. 16 last - 1
        const uint64_t va = v_desc + st * kTile16;
#pragma unroll
        for (int k = decltype(first)::value; k < decltype(last)::value; ++k)
          umma_ts(tmem + S::kO + i * D, tmem + S::kP + i * S::kPStep + k * 8, va + k * 128, idesc_o,
                  k == 0 ? acc : 1u);
      };
      using Zero = std::integral_constant<int, 0>;
      using Hand = std::integral_constant<int, S::kHandover * 2>;
      using All = std::integral_constant<int, kWtKeys / 16>;
      bool ok = mbar_wait(q_full, 0);
      uint32_t np0 = 0, np1 = 0;  // P tiles taken
      if (n > 0) {
        const int t0 = tiles.tile(0) * kWtKeys;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&full[0], 0));
        tc_fence_after();
        if (ok && elect_one()) {
          if (half[0].some(t0, t0 + kWtKeys)) {
            qk(0, 0);
            umma_commit(&s_full[0]);
          }
          if (half[1].some(t0, t0 + kWtKeys)) {
            qk(1, 0);
            umma_commit(&s_full[1]);
          }
          umma_commit(&empty[0]);
        }
        __syncwarp();
      }
      // PV_i in two pieces, the second when the rest of P is there
      auto multiply = [&](int i, uint32_t& np, int vs) {
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&p_half[i], np & 1));
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) pv(i, vs, Zero{}, Hand{}, np > 0);
        __syncwarp();
        ok = __all_sync(0xffffffffu, mbar_wait(&p_full[i], np & 1));
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          pv(i, vs, Hand{}, All{}, 1u);
          umma_commit(&pv_done[i]);
        }
        __syncwarp();
        ++np;
      };
      auto score = [&](int i, int ks) {
        if (elect_one()) {
          qk(i, ks);
          umma_commit(&s_full[i]);
        }
        __syncwarp();
      };
      auto release = [&](int slot) {
        if (elect_one()) umma_commit(&empty[slot]);
        __syncwarp();
      };
      auto seen = [&](int i, int j) {
        const int k0 = tiles.tile(j) * kWtKeys;
        return (i ? half[1] : half[0]).some(k0, k0 + kWtKeys);
      };
      if (S::kEarly) {
        // QK_0(j+1), PV_1(j-1), QK_1(j+1), PV_0(j): S of the next tile as soon as the softmax has
        // this one in registers
        uint32_t ns0 = n > 0 && seen(0, 0), ns1 = n > 0 && seen(1, 0);  // S tiles issued
        auto next_score = [&](int i, uint32_t& ns, int j) {
          if (!seen(i, j)) return;
          if (ns > 0) ok = __all_sync(0xffffffffu, ok && mbar_wait(&s_free[i], (ns - 1) & 1));
          if (!ok) return;
          tc_fence_after();
          score(i, j % kSK);
          ++ns;
        };
        for (int j = 0; j <= n && ok; ++j) {
          const bool more = j + 1 < n;
          if (more) {
            ok = __all_sync(0xffffffffu, mbar_wait(&full[(j + 1) % kSK], ((j + 1) / kSK) & 1));
            if (ok) next_score(0, ns0, j + 1);
          }
          if (ok && j > 0) {
            const int vs = kSK + (j - 1) % kSV;
            if (seen(1, j - 1)) multiply(1, np1, vs);
            if (ok) release(vs);
          }
          if (ok && more) {
            next_score(1, ns1, j + 1);
            if (ok) release((j + 1) % kSK);
          }
          if (ok && j < n) {
            const int vs = kSK + j % kSV;
            ok = mbar_wait(&full[vs], (j / kSV) & 1) && mbar_wait(&clean[vs], (j / kSV) & 1);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (ok && seen(0, j)) multiply(0, np0, vs);
          }
        }
      } else {
        // PV_0(j), QK_0(j+1), PV_1(j), QK_1(j+1)
        for (int j = 0; j < n && ok; ++j) {
          const bool more = j + 1 < n;
          const int vs = kSK + j % kSV, ks = (j + 1) % kSK;
          ok = mbar_wait(&full[vs], (j / kSV) & 1) && mbar_wait(&clean[vs], (j / kSV) & 1);
          if (ok && more) ok = mbar_wait(&full[ks], ((j + 1) / kSK) & 1);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (seen(0, j)) multiply(0, np0, vs);
          if (ok && more && seen(0, j + 1)) score(0, ks);
          if (ok && seen(1, j)) multiply(1, np1, vs);
          if (ok && more && seen(1, j + 1)) score(1, ks);
          if (!ok) break;
          release(vs);
          if (more) release(ks);
        }
      }
    }
  } else {
    reg_inc<S::kSoftRegs>();
    if (row0 < rows) {
      // -------------------------------------------------------------- softmax
      const int i = warp >> 2;                  // tile
      const WtSpan mine = i ? half[1] : half[0];
      const int quarter = warp & 3;             // TMEM lanes of this warp
      const int r = quarter * 32 + lane;        // row in the tile
      const int row = row0 + i * kWtRows + r;   // row of the (sequence, key head)
      // Q rows of this warp into the swizzled tile, zeros past the end
      uint8_t* q_tile = sQ + i * S::kTile;
      constexpr int kChunks = D / 8;
      uint4 qv[kChunks];  // all loads before the first store, which the compiler could not tell apart
#pragma unroll
      for (int x = 0; x < kChunks; ++x) {
        const int c = x * 32 + lane;
        const int qrow = row0 + i * kWtRows + quarter * 32 + c / kChunks;
        qv[x] = make_uint4(0, 0, 0, 0);
        if (qrow < row1)
          qv[x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                  static_cast<long long>(seq.q0 + a.by_group.div(qrow)) * a.q_ts +
                                                  (kvh * a.group + a.by_group.mod(qrow)) * a.q_hs + c % kChunks * 8);
      }
#pragma unroll
      for (int x = 0; x < kChunks; ++x) {
        const int c = x * 32 + lane;
        const int rr = quarter * 32 + c / kChunks, ch = c % kChunks;
        *reinterpret_cast<uint4*>(q_tile + (ch >> 3) * S::kHalf + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4)) = qv[x];
      }
      fence_async_smem_cta();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const WinRange range =
          row < row1 ? win_range(a, seq.kv - seq.n_q + a.by_group.div(row), seq.kv) : WinRange{0, 0, 0};
      const uint32_t s_addr = tmem + i * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t p_addr = tmem + S::kP + i * S::kPStep + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t o_addr = tmem + S::kO + i * D + (static_cast<uint32_t>(quarter * 32) << 16);
      const float sl2 = a.scale_log2;
      // whether some page in sight is not there: only then are the tiles' pages looked up
      bool hole = false;
      if (n > 0) {
        const int last_sink = min(n, max(tiles.sink, 0));  // sink tiles of this CTA, then window tiles
        for (int j = 0; j < 2; ++j) {
          const int t0 = j ? last_sink : 0, t1 = j ? n : last_sink;
          if (t0 == t1) continue;
          const int p0 = a.by_page.div(tiles.tile(t0) * kWtKeys);
          const int p1 = min(a.by_page.div(min((tiles.tile(t1 - 1) + 1) * kWtKeys, mine.hi.end) + a.page_tokens - 1), a.width);
#pragma unroll 4
          for (int x = p0 + lane; x < p1; x += 32) hole |= static_cast<uint32_t>(table[x]) >= static_cast<uint32_t>(a.pages);
        }
      }
      const bool holes = __any_sync(0xffffffffu, hole && mine.any);
      for (int j = 0; j < n; ++j) {
        const int tile = tiles.tile(j), k0 = tile * kWtKeys;
        if (!mine.some(k0, k0 + kWtKeys)) continue;
        const bool part = holes || !mine.all(k0, k0 + kWtKeys);
        ok = mbar_wait(&s_full[i], np & 1);
        if (!__all_sync(0xffffffffu, ok)) break;
        tc_fence_after();
        uint32_t v[4][32];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        auto maxima = [&](int c) {
          if (part) {
            const int k = k0 + c * 32;
            uint32_t seen = wt_bits(range.start - k, range.end - k) | wt_bits(-k, range.sink_end - k);
            if (holes) {
#pragma unroll
              for (int x = 0; x < 32; x += 16) {  // a page is a multiple of 16 tokens
                const int idx = a.by_page.div(k + x);
                const int page = idx < a.width ? table[idx] : -1;
                if (page < 0 || page >= a.pages) seen &= ~(0xffffu << x);
              }
            }
            wt_hide(v[c], seen);
          }
#pragma unroll
          for (int x = 0; x < 32; x += 2)
            mx[(x >> 1) & 3] = max3_nan(mx[(x >> 1) & 3], __uint_as_float(v[c][x]), __uint_as_float(v[c][x + 1]));
        };
        tmem_ld32_nowait(s_addr, v[0]);
        tmem_ld32_nowait(s_addr + 32, v[1]);
        tmem_wait_ld(v[0]);
        tmem_wait_ld(v[1]);
        tmem_ld32_nowait(s_addr + 64, v[2]);
        tmem_ld32_nowait(s_addr + 96, v[3]);
        maxima(0);
        maxima(1);
        tmem_wait_ld(v[2]);
        tmem_wait_ld(v[3]);
        if (S::kEarly) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[i]);
        }
        maxima(2);
        maxima(3);
        const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
        // a NaN score makes the maximum and with it the whole row NaN; a tile without a visible
        // key (top -inf) changes nothing
        const bool grow = !((top - m) * sl2 <= kWtLazy) && top != -INFINITY;
        float alpha = 1.0f;
        if (grow) {
          alpha = ex2((m - top) * sl2);  // 0 at the first tile
          m = top;
          l *= alpha;
        }
        if (np > 0 && __any_sync(0xffffffffu, grow)) {
          ok = mbar_wait(&pv_done[i], (np - 1) & 1);
          if (!__all_sync(0xffffffffu, ok)) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {  // few columns at a time: the row of S stays in registers
            float o[16];
            tmem_ld16(o_addr + c * 16, o);
            uint32_t w[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) w[x] = __float_as_uint(o[x] * alpha);
            tmem_st16(o_addr + c * 16, w);
          }
        }
        // P of the previous tile has been read: with P in place of S that is so since S came after it
        if (S::kEarly && np > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[i], (np - 1) & 1));
          if (!ok) break;
          tc_fence_after();
        }
        const float base = m == -INFINITY ? 0.0f : fmaf(m, 0.0f, -m * sl2);  // NaN for a maximum of +inf
        uint64_t sum[2] = {0, 0};
        // (D = 128: the columns of P lie over those of S, which are all in registers.)  The MMAs take
        // the first kHandover quarters of the keys while the rest is computed.
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 32; x += 2) {
            float2 e =
                unpair_f32(fma_f32x2(pair_f32(v[c][x], v[c][x + 1]), pair_f32(sl2, sl2), pair_f32(base, base)));
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[(x >> 1) & 1] = add_f32x2(sum[(x >> 1) & 1], pair_f32(e.x, e.y));
            pk[x / 2] = pack2<T>(e.x, e.y);
          }
          if (c == S::kHandover) {
            tmem_wait_st(pk);  // of the earlier quarters, under the arithmetic of this one
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[i]);
          }
          tmem_st16(p_addr + c * 16, pk);
        }
        const float2 s2 = unpair_f32(add_f32x2(sum[0], sum[1]));
        l += s2.x + s2.y;
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[i]);
        ++np;
      }
      if (ok && np > 0) ok = mbar_wait(&pv_done[i], (np - 1) & 1);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      // warp 11's mark: its tiles up to this query tile's last were looked at before pv_done
      if (splits > 1) {
        // joined below
      } else if (ok && *reinterpret_cast<volatile int*>(dirty) < mine.hi.end) {
        for (int x = 0; x < 32; ++x) {
          const int rr = row0 + i * kWtRows + quarter * 32 + x;
          if (rr < row1) window_row<T, D>(a, b, seq, a.by_group.div(rr), kvh * a.group + a.by_group.mod(rr), lane);
        }
      } else if (ok) {
        // O / l through the warp's own rows of the Q tile (its last reader is done), then out in
        // whole rows
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const bool some = np > 0 && inv != 0.0f;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32] = {};
          if (np > 0) {
            tmem_ld32_nowait(o_addr + c * 32, o);
            tmem_wait_ld(o);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t w4[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w4[y] = some ? pack2<T>(__uint_as_float(o[8 * x + 2 * y]) * inv, __uint_as_float(o[8 * x + 2 * y + 1]) * inv)
                           : 0u;
            const int ch = c * 4 + x;
            *reinterpret_cast<uint4*>(q_tile + (ch >> 3) * S::kHalf + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) =
                make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
          const int c = x * 32 + lane;
          const int rr = quarter * 32 + c / kChunks, ch = c % kChunks;
          const int orow = row0 + i * kWtRows + rr;
          if (orow < row1) {
            T* dst = static_cast<T*>(a.out) + static_cast<long long>(seq.q0 + a.by_group.div(orow)) * a.o_ts +
                     (kvh * a.group + a.by_group.mod(orow)) * a.o_hs + ch * 8;
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(
                q_tile + (ch >> 3) * S::kHalf + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4));
          }
        }
        if (a.lse && row < row1)
          a.lse[static_cast<long long>(seq.q0 + a.by_group.div(row)) * a.heads + kvh * a.group + a.by_group.mod(row)] =
              l == 0.0f ? -INFINITY : (m * sl2 + log2f(l)) * 0.6931471805599453f;
      }
    }
    // more rows than the launch was told of: one by one
    if (tile_id == row_tiles - 1 && rank == 0)
      for (int r = row_tiles * (2 * kWtRows) + warp; r < rows; r += 8)
        window_row<T, D>(a, b, seq, a.by_group.div(r), kvh * a.group + a.by_group.mod(r), lane);
  }
  if (splits > 1) {
    // Join the cluster's parts, each CTA a share of the rows: stores into the owner's shared memory
    // need no answer, where loads from the others waited 4 us for theirs.
    __syncwarp();
    cluster_sync_all();  // every CTA's MMAs have read its ring
    if (warp < 8 && row0 < rows) {
      const int quarter = warp & 3, rr = (warp >> 2) * kWtRows + quarter * 32 + lane;
      const uint32_t o_addr = tmem + S::kO + (warp >> 2) * D + (static_cast<uint32_t>(quarter * 32) << 16);
      const int owner = min(rr / share, splits - 1), slot = rank * share + rr - owner * share;
      const bool mine = rr < row1 - row0;
      if (mine) {
        st_cluster(mapa_shared(smem_u32(part_m + slot), owner), ok ? m : __uint_as_float(0x7fffffffu));
        st_cluster(mapa_shared(smem_u32(part_l + slot), owner), l);
      }
      if (threadIdx.x < splits)
        st_cluster(mapa_shared(smem_u32(part_mark + rank), threadIdx.x), __int_as_float(*reinterpret_cast<volatile int*>(dirty)));
      const uint32_t dst = mapa_shared(smem_u32(part_o + slot * D), owner);
#pragma unroll 1
      for (int c = 0; np > 0 && c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32_nowait(o_addr + c * 32, o);
        tmem_wait_ld(o);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (mine) st_cluster4(dst + (((c * 8 + x) ^ (slot & 7)) << 4), o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
      }
    }
    __syncwarp();
    cluster_sync_all();
    const int own0 = rank * share, own = min(share, row1 - row0 - own0);  // this CTA's rows
    if (warp < 8 && own > 0) {
      bool marked = false;
      for (int x = 0; x < splits; ++x) marked |= part_mark[x] != kWtClean;
      if (marked) {
        for (int r = row0 + own0 + warp; r < row0 + own0 + own; r += 8)
          window_row<T, D>(a, b, seq, a.by_group.div(r), kvh * a.group + a.by_group.mod(r), lane);
      } else {
        const float sl2 = a.scale_log2;
        for (int e = threadIdx.x; e < own * (D / 8); e += 256) {
          const int r = e / (D / 8), ch = e % (D / 8) * 2;
          float top = -INFINITY;
          for (int x = 0; x < splits; ++x) top = max3_nan(top, part_m[x * share + r], part_m[x * share + r]);
          float sum = 0.0f;
          float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
          for (int x = 0; x < splits; ++x) {  // in rank order
            const int at = x * share + r;
            if (part_m[at] == -INFINITY) continue;  // (its O was not sent)
            const float f = ex2((part_m[at] - top) * sl2);
            const float4 p = *reinterpret_cast<const float4*>(part_o + at * D + ((ch ^ (at & 7)) << 2));
            const float4 q = *reinterpret_cast<const float4*>(part_o + at * D + (((ch + 1) ^ (at & 7)) << 2));
            sum += f * part_l[at];
            u.x = fmaf(f, p.x, u.x), u.y = fmaf(f, p.y, u.y), u.z = fmaf(f, p.z, u.z), u.w = fmaf(f, p.w, u.w);
            v.x = fmaf(f, q.x, v.x), v.y = fmaf(f, q.y, v.y), v.z = fmaf(f, q.z, v.z), v.w = fmaf(f, q.w, v.w);
          }
          const bool none = sum == 0.0f;
          const float inv = none ? 0.0f : 1.0f / sum;
          uint4 w4 = make_uint4(pack2<T>(u.x * inv, u.y * inv), pack2<T>(u.z * inv, u.w * inv),
                                pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
          if (none) w4 = make_uint4(0, 0, 0, 0);
          const int qr = row0 + own0 + r, head = kvh * a.group + a.by_group.mod(qr);
          const long long tok = seq.q0 + a.by_group.div(qr);
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + tok * a.o_ts + head * a.o_hs + ch * 4) = w4;
          if (a.lse && ch == 0)
            a.lse[tok * a.heads + head] = none ? -INFINITY : (top * sl2 + log2f(sum)) * 0.6931471805599453f;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc<512>(tmem);
}

}  // namespace oasis
