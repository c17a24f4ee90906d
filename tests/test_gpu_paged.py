"""The paged-cache operators on the GPU against their formulas in 64 bits.

Tolerances, element by element, with u = eps / 2 of the result's type (half a step, relative):
* the rotation: u |y| for the one rounding, and 2^-19 (|a| + |b|) for the fp32 arithmetic on the
  pair (a, b): mean of squares of up to 256 values summed in a tree (13 roundings, halved by the
  root), rsqrt, cos and sin (2 ulp each and the angle's last rounding to fp32 in turns, 2 pi 2^-25),
  five products and sums; each 2^-24 to 2^-22, together below 2^-19.
* attention: u |out| for the one rounding; the weights p are rounded to the type before the second
  product, u each, so u A with A = sum p |v| / sum p; fp32 scores are off by at most
  (D + 2) 2^-24 S with S the largest sum |q||k| scale, which moves p and the sum of p by that relative amount
  each; sums over n keys by n 2^-24 each and exp2 by 2^-21: A (2 (D + 2) 2^-24 S + 2 n 2^-24 + 2^-20).
  fp16 weights below 2^-14 (the largest is at least 1/256 of the scale's) are off by 2^-25 at most, which adds
  n 2^-25 max|v|.
"""

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, tol, what=""):
    if not want.numel():
        return
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    over = ((got - want).abs() - tol).nan_to_num(0.0)
    i = over.argmax()
    assert over.max() <= 0, f"{what}: {got.flatten()[i]} for {want.flatten()[i]}, tolerance {tol.flatten()[i]}"


# ------------------------------------------------------------------ norm + rotation


def rope_ref(x, w, positions, freqs, axes, interleaved, norm, eps):
    """fp64 result and the size of each element's pair."""
    x = x.double()
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * w.double()
    y, size = x.clone(), x.abs().clone()
    pairs, p = sum(axes) // 2, 0
    for a, dims in enumerate(axes):
        for _ in range(dims // 2):
            i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
            angle = positions[:, a].double()[:, None] * freqs[p]
            c, s = torch.cos(angle), torch.sin(angle)
            y[..., i] = x[..., i] * c - x[..., j] * s
            y[..., j] = x[..., j] * c + x[..., i] * s
            size[..., i] = size[..., j] = x[..., i].abs() + x[..., j].abs()
            p += 1
    return y, size


def rope_tol(y, size, dtype):
    return half_step(dtype) * y.abs() + 2.0 ** -19 * size + 1e-30 + (2.0 ** -25 if dtype == HF else 0)


def rope_inputs(pkg, cuda, tokens, h, hk, d, dtype, axes, seed=0, far=50000, i64=False):
    g = torch.Generator(device=cuda).manual_seed(seed)
    qkv = torch.randn(tokens, (h + 2 * hk) * d, device=cuda, generator=g).to(dtype)
    q, k, v = (z.unflatten(1, (-1, d)) for z in qkv.split([h * d, hk * d, hk * d], 1))
    pos = torch.randint(-far, far, (tokens, len(axes)), device=cuda, generator=g,
                        dtype=torch.int64 if i64 else torch.int32)
    wq, wk = (torch.rand(d, device=cuda, generator=g) + 0.5 for _ in range(2))
    return q, k, v, pos, wq, wk, pkg.rope_axis_freqs(axes, device=cuda)


@pytest.mark.parametrize("tokens,h,hk,d,dtype,axes,inter,norm", [
    (1, 1, 1, 32, BF, (32,), True, True),
    (1, 16, 16, 64, BF, (16, 24, 24), True, True),
    (5, 7, 1, 64, HF, (6, 10), True, True),          # odd heads, a part of the pairs
    (147, 16, 16, 64, BF, (16, 24, 24), False, True),
    (33, 24, 8, 128, F32, (32, 32, 32), False, True),
    (1000, 3, 3, 128, HF, (44, 42, 42), True, False),
    (2500, 5, 1, 256, BF, (64, 64, 64, 64), False, True),
    (19, 2, 2, 256, F32, (2, 2), True, True),
    (64, 4, 2, 32, F32, (8, 8), False, False),
    (3001, 4, 4, 64, F32, (64,), True, True),
])
def test_qk_norm_rope(pkg, cuda, tokens, h, hk, d, dtype, axes, inter, norm):
    q, k, _, pos, wq, wk, f = rope_inputs(pkg, cuda, tokens, h, hk, d, dtype, axes, i64=tokens % 2 == 0)
    kw = dict(axes=axes, interleaved=inter, norm=norm, eps=1e-5)
    if norm:
        kw.update(q_weight=wq, k_weight=wk)
    qo, ko = pkg.qk_norm_rope(q, k, pos, f, **kw)
    for x, o, w in ((q, qo, wq), (k, ko, wk)):
        y, size = rope_ref(x, w, pos, f, axes, inter, norm, 1e-5)
        check(o, y, rope_tol(y, size, dtype))


def test_qk_norm_rope_strides_and_in_place(pkg, cuda):
    """Head-major inputs, no weights, outputs over the inputs."""
    q, k, _, pos, _, _, f = rope_inputs(pkg, cuda, 77, 6, 2, 64, BF, (24, 24, 16))
    q = q.transpose(0, 1).contiguous().transpose(0, 1)
    k = k.transpose(0, 1).contiguous().transpose(0, 1)
    yq, sq = rope_ref(q, None, pos, f, (24, 24, 16), True, True, 1e-6)
    yk, sk = rope_ref(k, None, pos, f, (24, 24, 16), True, True, 1e-6)
    a, b = pkg.qk_norm_rope(q, k, pos, f, axes=(24, 24, 16), q_out=q, k_out=k)
    assert a is q and b is k
    check(q, yq, rope_tol(yq, sq, BF))
    check(k, yk, rope_tol(yk, sk, BF))


def test_qk_norm_rope_keeps_norms_and_far_angles(pkg, cuda):
    """A rotation changes no pair's length, and positions near 2^31 rotate like their formula."""
    q, k, _, pos, _, _, f = rope_inputs(pkg, cuda, 257, 4, 4, 64, F32, (64,), far=2 ** 31 - 1)
    qo, _ = pkg.qk_norm_rope(q, k, pos, f, axes=(64,), norm=False)
    y, size = rope_ref(q, None, pos, f, (64,), True, False, 0)
    # the reference's own angle, position * frequency in fp64, is off by 2^31 2^-53 2: far below
    check(qo, y, rope_tol(y, size, F32))
    length = qo.unflatten(-1, (32, 2)).norm(dim=-1)
    torch.testing.assert_close(length, q.unflatten(-1, (32, 2)).norm(dim=-1), rtol=2.0 ** -19, atol=0)


def test_qk_norm_rope_special_values(pkg, cuda):
    """Zero heads, NaN and infinities stay in their heads; dims behind the rotated ones stay apart."""
    q, k, _, pos, _, _, f = rope_inputs(pkg, cuda, 6, 4, 4, 64, BF, (16, 10))
    q[0, 1] = 0
    q[1, 2, 5] = float("nan")
    k[2, 0, 40] = float("inf")  # not rotated: only itself without the norm
    for norm in (True, False):
        for axes, ff, inter in (((16, 10), f, True), ((16,), f[:8].contiguous(), False)):
            p = pos[:, : len(axes)].contiguous()
            qo, ko = pkg.qk_norm_rope(q, k, p, ff, axes=axes, norm=norm, interleaved=inter)
            yq, sq = rope_ref(q, None, p, ff, axes, inter, norm, 1e-6)
            yk, sk = rope_ref(k, None, p, ff, axes, inter, norm, 1e-6)
            check(qo, yq, rope_tol(yq, sq, BF))
            keep = ~yk.isinf()
            assert torch.equal(ko.double().isinf(), ~keep)
            check(ko[keep], yk[keep], rope_tol(yk, sk, BF)[keep])


@pytest.mark.parametrize("tokens,h,hk,d,dtype,pt", [(1, 16, 16, 64, BF, 16), (145, 10, 2, 128, HF, 48),
                                                    (1152, 4, 4, 64, BF, 144)])
def test_qk_norm_rope_append(pkg, cuda, tokens, h, hk, d, dtype, pt):
    axes = (d // 4, d // 4, d // 2)
    q, k, v, pos, wq, wk, f = rope_inputs(pkg, cuda, tokens, h, hk, d, dtype, axes)
    n = -(-tokens // pt) + 2
    kp, vp = (torch.randn(n, hk, pt, d, device=cuda).to(dtype) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    slots = torch.randperm(n * pt, device=cuda)[:tokens].int()
    if tokens > 2:  # tokens that are not stored
        slots[1], slots[2] = -1, n * pt
    qo = pkg.qk_norm_rope_append(q, k, v, pos, f, kp, vp, slots, axes=axes, interleaved=False, q_weight=wq,
                                 k_weight=wk)
    q2, k2 = pkg.qk_norm_rope(q, k, pos, f, axes=axes, interleaved=False, q_weight=wq, k_weight=wk)
    assert torch.equal(qo, q2)
    ok = (slots >= 0) & (slots < n * pt)
    at = slots[ok].long()
    k0[at // pt, :, at % pt] = k2[ok]
    v0[at // pt, :, at % pt] = v[ok]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


# ------------------------------------------------------------------ attention


def attn_ref(q, kp, vp, table, kv_len, cu, window, sinks, frame, scale):
    """fp64 out, lse and the tolerance's A, S, n, max|v| of every row; rows of no sequence stay NaN."""
    n, h, d = q.shape
    hk, pt = kp.shape[1:3]
    out = torch.full((n, h, d), math.nan, dtype=torch.float64, device=q.device)
    amp, lse = out.clone(), out[..., 0].clone()
    top = torch.zeros(n, h, dtype=torch.float64, device=q.device)
    cnt, maxv = top.clone(), top.clone()
    for b in range(table.shape[0]):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        m, kv = r1 - r0, max(0, min(int(kv_len[b]), table.shape[1] * pt))
        key = torch.arange(kv, device=q.device)
        page = table[b].long()[key // pt]
        there = (page >= 0) & (page < kp.shape[0])
        page = page.clamp(0, kp.shape[0] - 1)
        pos = kv - m + torch.arange(m, device=q.device)[:, None]
        see = (key // frame <= torch.div(pos, frame, rounding_mode="floor")) & there & (pos >= 0)
        if window:
            see &= (torch.div(pos, frame, rounding_mode="floor") - key // frame < window) | (key // frame < sinks)
        for i in range(h):
            k, v = (p[page, i // (h // hk), key % pt].double() for p in (kp, vp))
            qi = q[r0:r1, i].double()
            s = (qi @ torch.where(see.any(0)[:, None], k, 0).T) * scale
            for j in see.any(0).logical_and(k.isnan().any(1)).nonzero():
                s[:, j] = math.nan
            s = s.masked_fill(~see, -math.inf)
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(l.isinf(), 0, l)[:, None])
            fine = v.isfinite().all(1)
            o = p[:, fine] @ v[fine]
            for j in (~fine).nonzero().flatten():
                o = o + torch.where(see[:, j, None], p[:, j, None] * v[j], 0)
            out[r0:r1, i], lse[r0:r1, i] = o, l
            vf = v.abs().nan_to_num(0, 0, 0)
            amp[r0:r1, i] = p.nan_to_num(0) @ vf
            size = (qi.abs() @ k.abs().nan_to_num(0, 0, 0).T) * scale
            top[r0:r1, i] = (size * see).amax(-1) if kv else 0
            cnt[r0:r1, i] = see.sum(-1)
            maxv[r0:r1, i] = (see[..., None] * vf).amax((1, 2)) if kv and kv * m * d < 1 << 28 else 6
    return out, lse, amp, top, cnt, maxv


def attn_tol(ref, dtype, d):
    out, _, amp, top, cnt, maxv = ref
    u = half_step(dtype)
    rel = u + 2 * (d + 2) * 2.0 ** -24 * top + 2 * cnt * 2.0 ** -24 + 2.0 ** -20
    tol = u * out.abs() + rel[..., None] * amp
    if dtype == HF:
        tol = tol + 2.0 ** -25 * (1 + cnt * maxv)[..., None]
    return tol


def attn_inputs(cuda, q_len, kv_len, h, hk, d, dtype, pt, seed=0, holes=(), sharp=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    need = [-(-n // pt) for n in kv_len]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(q_len), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at: at + n]
        at += n
    for b, i, x in holes:
        table[b, i] = x
    q = (torch.randn(sum(q_len), h, d, device=cuda, generator=g) * sharp).to(dtype)
    kp, vp = (torch.randn(pages, hk, pt, d, device=cuda, generator=g).to(dtype) for _ in range(2))
    # what no session's token fills holds anything: unlisted pages and the ends of last pages
    kp[order[at:].to(cuda)] = math.nan
    vp[order[at:].to(cuda)] = math.inf
    for b, n in enumerate(kv_len):
        if n % pt and 0 <= int(table[b, n // pt]) < pages:
            kp[int(table[b, n // pt]), :, n % pt:] = math.nan
            vp[int(table[b, n // pt]), :, n % pt:] = math.nan
    cu = torch.tensor([0] + q_len).cumsum(0).int()
    return q, kp, vp, table.to(cuda), torch.tensor(kv_len, dtype=torch.int32, device=cuda), cu.to(cuda)


def run_case(pkg, cuda, q_len, kv_len, h, hk, d, dtype, pt, window, sinks, frame, **kw):
    call = {k: kw.pop(k) for k in ("max_q", "max_kv", "scale") if k in kw}
    q, kp, vp, table, lens, cu = attn_inputs(cuda, q_len, kv_len, h, hk, d, dtype, pt, **kw)
    out, lse = pkg.attn_window(q, kp, vp, table, lens, cu, window=window, sinks=sinks, frame_tokens=frame,
                               return_lse=True, **call)
    ref = attn_ref(q, kp, vp, table, lens, cu, window, sinks, frame, call.get("scale", d ** -0.5))
    check(out, ref[0], attn_tol(ref, dtype, d), "out")
    # lse: the scores' error, the sum's, and log2 / exp2 of fp32
    tol = 2 * (d + 2) * 2.0 ** -24 * ref[3] + ref[4] * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * ref[1].abs()
    empty = ref[1].isinf()
    assert torch.equal(lse[empty], torch.full_like(lse[empty], -math.inf))
    check(lse[~empty], ref[1][~empty], tol[~empty], "lse")
    return q, kp, vp, table, lens, cu, out


TOKEN = [  # single tokens and few rows
    ([1], [1], 1, 1, 64, BF, 16, None, 0, 1),
    ([1], [577], 16, 16, 64, BF, 16, None, 0, 1),
    ([1, 1, 1], [15, 16, 17], 8, 2, 128, HF, 16, None, 0, 1),
    ([1] * 5, [1, 300, 31, 33, 1025], 6, 2, 64, HF, 48, 100, 7, 1),
    ([1] * 4, [4000, 64, 2500, 129], 32, 8, 128, BF, 16, 512, 16, 1),
    ([1, 1], [777, 2000], 16, 1, 128, BF, 144, 1000, 4, 1),   # all heads share one key head
    ([1, 1], [100, 290], 5, 5, 64, BF, 16, 2, 1, 60),         # frames, the first stays
    ([3, 0, 2], [300, 40, 2], 4, 2, 128, HF, 32, 50, 3, 1),   # several tokens, none, all of the cache
    ([1], [9000], 2, 2, 64, HF, 64, None, 0, 1),
    ([4], [70], 12, 4, 64, BF, 16, 1, 0, 1),                  # sees only itself
    ([7], [3], 2, 1, 64, BF, 16, None, 0, 1),                 # more queries than tokens: rows that see nothing
    ([2, 1], [0, 0], 4, 4, 64, HF, 16, 5, 1, 1),              # empty caches
    ([1, 1], [600, 500], 20, 1, 128, BF, 16, 99, 99, 3),      # 20 rows on one key head
    ([1], [6001], 8, 1, 128, BF, 16, None, 0, 1),             # one key head: the widest splits
    ([1], [5003], 16, 1, 128, HF, 32, 4000, 30, 1),
    ([2], [4100], 16, 2, 64, BF, 16, 1000, 10, 1),
    ([1, 1], [3000, 100], 24, 12, 128, BF, 48, None, 0, 1),
]

TILE = [  # prompts and frames
    ([17], [17], 1, 1, 64, BF, 16, None, 0, 1),
    ([128], [128], 2, 2, 64, BF, 16, None, 0, 1),
    ([129], [257], 2, 2, 128, HF, 16, None, 0, 1),
    ([255, 1, 300], [255, 1000, 301], 3, 3, 64, BF, 16, None, 0, 1),
    ([500], [500], 4, 1, 128, BF, 64, 130, 5, 1),
    ([144], [7056], 4, 4, 64, BF, 16, 32, 1, 144),
    ([144, 144], [1440, 144], 4, 4, 64, HF, 144, 4, 1, 144),
    ([100, 70], [333, 900], 6, 2, 128, HF, 32, 3, 2, 60),     # frames that end inside tiles and steps
    ([64], [1000], 10, 2, 64, BF, 48, 128, 0, 1),             # 5 heads to a key head
    ([33, 40], [2000, 41], 7, 1, 128, BF, 16, 256, 128, 1),   # 7 heads to a key head
    ([1000], [1000], 1, 1, 64, HF, 16, 1, 0, 1),
    ([200], [150], 2, 2, 64, BF, 16, None, 0, 1),             # rows that see nothing
    ([300], [300], 2, 2, 128, BF, 16, None, 0, 1000),         # one frame: everything sees everything
    ([257], [1500], 2, 1, 64, BF, 128, 300, 200, 1),          # sinks meet the window
    ([150, 0, 20], [0, 5, 20], 2, 2, 128, BF, 16, 4, 1, 7),
]


@pytest.mark.parametrize("case", TOKEN + TILE, ids=str)
def test_attn_window(pkg, cuda, case):
    run_case(pkg, cuda, *case)


@pytest.mark.parametrize("case", [TOKEN[4], TOKEN[7], TILE[4], TILE[7]], ids=str)
def test_attn_window_sharp_scores_and_scale(pkg, cuda, case):
    """Scores of up to some hundreds: most weights vanish, the maximum moves from tile to tile."""
    run_case(pkg, cuda, *case, sharp=20.0, scale=0.3)


@pytest.mark.parametrize("q_len", [[1, 1], [2, 3], [90, 140]])
def test_attn_window_page_holes(pkg, cuda, q_len):
    """Entries outside the pages hide their tokens."""
    holes = [(0, 0, -1), (0, 5, 1 << 30), (0, 6, -(1 << 31)), (1, 3, -7), (1, 1, 99999)]
    run_case(pkg, cuda, q_len, [300, 170], 4, 2, 64, BF, 16, None, 0, 1, holes=holes)
    run_case(pkg, cuda, q_len, [300, 170], 4, 2, 128, HF, 16, 64, 20, 1, holes=holes)
    run_case(pkg, cuda, q_len, [3000, 1700], 4, 2, 128, BF, 16, None, 0, 1, holes=holes)


@pytest.mark.parametrize("q_len", [[1, 1], [3, 2], [150, 130]])
def test_attn_window_what_is_not_seen_does_not_matter(pkg, cuda, q_len):
    """NaN and infinities in keys and values reach exactly the rows that see them."""
    case = (q_len, [400, 390], 4, 2, 64, BF, 16)
    for window, sinks, frame in ((40, 3, 1), (None, 0, 1), (3, 1, 20)):
        q, kp, vp, table, lens, cu = attn_inputs(cuda, *case, seed=3)
        for b, token, x in ((0, 2, math.nan), (0, 200, math.inf), (0, 361, -math.inf), (1, 10, math.nan),
                            (1, 380, math.nan), (1, 389, math.inf)):
            vp[int(table[b, token // 16]), 0, token % 16, 1] = x
            kp[int(table[b, token // 16]), 1, token % 16, 5] = math.nan
        out = pkg.attn_window(q, kp, vp, table, lens, cu, window=window, sinks=sinks, frame_tokens=frame)
        ref = attn_ref(q, kp, vp, table, lens, cu, window, sinks, frame, 0.125)
        assert torch.equal(out.isnan(), ref[0].isnan())
        assert torch.equal(out.double().isinf(), ref[0].isinf())
        fine = ref[0].isfinite()
        check(out[fine], ref[0][fine], attn_tol(ref, BF, 64)[fine])


@pytest.mark.parametrize("case", [TOKEN[4], TOKEN[7], TILE[3], TILE[7]], ids=str)
def test_attn_window_is_reproducible_and_hints_do_not_matter(pkg, cuda, case):
    """The same bits again, whatever the launch; bounds that are too small change nothing either."""
    q_len, kv_len, h, hk, d, dtype, pt, window, sinks, frame = case
    q, kp, vp, table, lens, cu = attn_inputs(cuda, q_len, kv_len, h, hk, d, dtype, pt)
    kw = dict(window=window, sinks=sinks, frame_tokens=frame)
    first = pkg.attn_window(q, kp, vp, table, lens, cu, **kw)
    assert torch.equal(first, pkg.attn_window(q, kp, vp, table, lens, cu, **kw))
    ref = attn_ref(q, kp, vp, table, lens, cu, window, sinks, frame, d ** -0.5)
    for max_q, max_kv in ((max(q_len), max(kv_len)), (1, 1), (1, None), (None, 1)):
        check(pkg.attn_window(q, kp, vp, table, lens, cu, max_q=max_q, max_kv=max_kv, **kw), ref[0],
              attn_tol(ref, dtype, d))


@pytest.mark.parametrize("q_len", [[1, 1], [60, 100]])
def test_attn_window_leaves_other_rows_and_takes_strides(pkg, cuda, q_len):
    q, kp, vp, table, lens, cu = attn_inputs(cuda, q_len, [100, 130], 4, 2, 64, BF, 16)
    n = sum(q_len)
    wide = torch.randn(n + 9, 3, 4, 64, device=cuda).bfloat16()  # queries as columns of a projection
    wide[:n, 1] = q
    out = torch.full((4, n + 9, 64), 7.0, device=cuda).bfloat16().transpose(0, 1)  # head-major
    got, lse = pkg.attn_window(wide[:, 1], kp, vp, table, lens, cu, out=out, return_lse=True)
    assert got is out and (out[n:] == 7).all()
    want, want_lse = pkg.attn_window(q, kp, vp, table, lens, cu, return_lse=True)
    ref = attn_ref(q, kp, vp, table, lens, cu, None, 0, 1, 0.125)
    check(out[:n], ref[0], attn_tol(ref, BF, 64))
    check(want, ref[0], attn_tol(ref, BF, 64))
    over = wide[:, 1]
    pkg.attn_window(over, kp, vp, table, lens, cu, out=over)  # the queries' own place
    check(over[:n], ref[0], attn_tol(ref, BF, 64))
    if q_len == [1, 1]:
        check(pkg.attn_window(q, kp, vp, table, lens), ref[0], attn_tol(ref, BF, 64))  # no cu_q


def test_attn_window_offsets_past_32_bits(pkg, cuda):
    """Pages beyond 2^32 bytes and 2^31 elements of the pools."""
    hk, pt, d = 16, 64, 128
    pages = (5 << 30) // (hk * pt * d * 2)  # 5 GiB of keys, 2.7e9 elements
    kp = torch.zeros(pages, hk, pt, d, dtype=BF, device=cuda)
    vp = torch.zeros_like(kp)
    last = [pages - 1, pages - 3, 1, pages - 7]
    kp[last] = torch.randn(4, hk, pt, d, device=cuda).bfloat16()
    vp[last] = torch.randn(4, hk, pt, d, device=cuda).bfloat16()
    table = torch.tensor([last], dtype=torch.int32, device=cuda)
    lens = torch.tensor([250], dtype=torch.int32, device=cuda)
    for n in (1, 130):
        q = torch.randn(n, 16, d, device=cuda).bfloat16()
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        out = pkg.attn_window(q, kp, vp, table, lens, cu)
        ref = attn_ref(q, kp, vp, table, lens, cu, None, 0, 1, d ** -0.5)
        check(out, ref[0], attn_tol(ref, BF, d))


# ------------------------------------------------------------------ page copies


@pytest.mark.parametrize("layers,pages,hk,pt,d,dtype,n", [
    (1, 4, 1, 16, 64, BF, 1), (3, 40, 2, 16, 64, HF, 17), (16, 30, 16, 16, 64, BF, 9),
    (2, 400, 5, 48, 128, BF, 150), (1, 7000, 1, 16, 64, HF, 3000),
])
def test_copy_pages(pkg, cuda, layers, pages, hk, pt, d, dtype, n):
    k, v = (torch.randn(layers, pages, hk, pt, d, device=cuda).to(dtype) for _ in range(2))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n))
    dst, src = order[:n], order[n:][torch.arange(n) % min(n, pages - n) // 2]  # sources repeat
    wk, wv = k.clone(), v.clone()
    wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    pkg.copy_pages(k, v, src.tolist(), dst.int())
    assert torch.equal(k, wk) and torch.equal(v, wv)
    k2, v2 = (torch.zeros(layers, n + 1, hk, pt, d, device=cuda, dtype=dtype) for _ in range(2))
    pkg.copy_pages(k, v, dst, list(range(n, 0, -1)), to=(k2, v2))
    assert torch.equal(k2[:, 1:].flip(1), k[:, dst]) and torch.equal(v2[:, 1:].flip(1), v[:, dst])
    assert not k2[:, 0].any() and torch.equal(k, wk)


def test_copy_pages_refusals(pkg, cuda):
    k, v = (torch.zeros(2, 8, 2, 16, 64, device=cuda, dtype=BF) for _ in range(2))
    for src, dst in (([1], [1]), ([0, 1], [2, 2]), ([0], [8]), ([-1], [2]), ([0, 1], [2])):
        with pytest.raises((ValueError, pkg.OasisError)):
            pkg.copy_pages(k, v, src, dst)
    with pytest.raises(ValueError, match="host"):
        pkg.copy_pages(k, v, torch.tensor([0], device=cuda), [1])
    with pytest.raises((ValueError, pkg.OasisError)):
        pkg.copy_pages(k, v, [0], [1], to=(k[:1], v[:1]))
    with pytest.raises(ValueError, match="contiguous"):
        pkg.copy_pages(k.transpose(0, 1), v.transpose(0, 1), [0], [1])
    pkg.copy_pages(k, v, [], [])


# ------------------------------------------------------------------ refusals, streams, graphs


def test_operator_refusals(pkg, cuda):
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [4], [40], 4, 2, 64, BF, 16)
    bad = [dict(q=q.half()), dict(q=q[0]), dict(q=q[..., ::2]), dict(kp=kp.float()), dict(kp=kp[:, :, ::2]),
           dict(table=table.long()), dict(lens=lens.repeat(2)), dict(cu=cu[:-1]), dict(cu=None),
           dict(table=table.cpu()), dict(window=0), dict(sinks=-1), dict(frame_tokens=0),
           dict(out=torch.empty(4, 4, 64, device=cuda)), dict(q=q[:, :3]), dict(q=q.float().requires_grad_().bfloat16()),
           dict(scale=-1.0), dict(q=q.cpu())]
    for change in bad:
        a = dict(q=q, kp=kp, vp=vp, table=table, lens=lens, cu=cu)
        kw = {}
        for name, x in change.items():
            (a if name in a else kw)[name] = x
        with pytest.raises((ValueError, pkg.OasisError)):
            pkg.attn_window(a["q"], a["kp"], a["vp"], a["table"], a["lens"], a["cu"], **kw)
    q, k, v, pos, wq, wk, f = rope_inputs(pkg, cuda, 4, 4, 2, 64, BF, (16, 24, 24))
    axes = (16, 24, 24)
    for change in (dict(axes=(16, 24)), dict(axes=(16, 24, 26)), dict(axes=()), dict(q_weight=wq.half()),
                   dict(q_weight=wq, norm=False), dict(q_out=torch.empty(4, 4, 64, device=cuda)),
                   dict(k_weight=wk[:32])):
        kw = dict(axes=axes)
        kw.update(change)
        with pytest.raises((ValueError, pkg.OasisError)):
            pkg.qk_norm_rope(q, k, pos, f, **kw)
    for args in ((q, k, pos.float(), f), (q, k, pos[:3], f), (q, k, pos, f.float()), (q, k[:3], pos, f),
                 (q, k.half(), pos, f), (q[..., 1:], k, pos, f), (q, k.cpu(), pos, f)):
        with pytest.raises((ValueError, pkg.OasisError)):
            pkg.qk_norm_rope(*args, axes=axes)
    slots = torch.arange(4, device=cuda, dtype=torch.int32)
    for kp_, s in ((kp.half(), slots), (kp, slots.long()), (kp, slots[:3]), (kp[:, :1].contiguous(), slots)):
        with pytest.raises((ValueError, pkg.OasisError)):
            pkg.qk_norm_rope_append(q, k, v, pos, f, kp_, kp_.clone(), s, axes=axes)


def test_other_stream(pkg, cuda):
    """A stream given: the work and the new tensors belong to it."""
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [1, 150], [300, 200], 4, 2, 64, BF, 16)
    want = pkg.attn_window(q, kp, vp, table, lens, cu)
    side = torch.cuda.Stream(device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        q2 = q.clone()
    got = pkg.attn_window(q2, kp, vp, table, lens, cu, stream=side)  # after the clone, on its stream
    pkg.copy_pages(kp, vp, [int(table[0, 0])], [int(table[0, 1])], stream=side)
    again = pkg.attn_window(q2, kp, vp, table, lens, cu, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and not torch.equal(again, want)


def test_one_element_dimensions_and_expanded_tensors(pkg, cuda):
    """Strides of dimensions of one element say nothing; expanded inputs are read, expanded outputs refused."""
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [1], [40], 1, 1, 64, BF, 16)
    odd = torch.as_strided(q, (1, 1, 64), (3, 5, 1))
    assert torch.equal(pkg.attn_window(odd, kp, vp, table, lens, cu), pkg.attn_window(q, kp, vp, table, lens, cu))
    f = pkg.rope_axis_freqs((64,), device=cuda)
    pos = torch.tensor([7], dtype=torch.int32, device=cuda)
    a, b = pkg.qk_norm_rope(odd, q, pos, f, axes=(64,))
    assert torch.equal(a, b)
    wide = q.expand(3, 4, 64)
    pos3 = torch.arange(3, device=cuda)[:, None]
    a, b = pkg.qk_norm_rope(wide, q.expand(3, 1, 64), pos3, f, axes=(64,))
    assert torch.equal(a, b.expand(3, 4, 64).contiguous())
    with pytest.raises(ValueError, match="expanded"):
        pkg.qk_norm_rope(wide, q.expand(3, 1, 64), pos3, f, axes=(64,), q_out=wide)
    with pytest.raises(ValueError, match="gradient"):
        pkg.attn_window(q, kp.requires_grad_(), vp, table, lens, cu)
    with torch.no_grad():
        pkg.attn_window(q, kp, vp, table, lens, cu)
    with pytest.raises(ValueError, match="gradient"):
        pkg.copy_pages(kp, vp, [0], [1])


def test_calls_side_by_side(pkg, cuda):
    """Two captured graphs and eager calls on three streams at once share nothing."""
    cases = [attn_inputs(cuda, [1, 1], [3000, 900], 8, 2, 128, BF, 16, seed=1),
             attn_inputs(cuda, [144], [2000], 4, 4, 64, BF, 16, seed=2),
             attn_inputs(cuda, [300], [700], 4, 2, 128, HF, 32, seed=3)]
    want = [pkg.attn_window(*c) for c in cases]
    outs = [torch.empty_like(w) for w in want]
    graphs = []
    for c, o in zip(cases[:2], outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(5):
                o.fill_(0)
                o.copy_(pkg.attn_window(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream(device=cuda) for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            outs[2].copy_(pkg.attn_window(*cases[2]))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    pkg._native.check(pkg.lib().oasis_check_device_error())


FIRST_CALL = """
import importlib, sys, torch
sys.path[:0] = [{root!r}, {tests!r}]
import test_gpu_paged as t
pkg = importlib.import_module({name!r})
dev = torch.device("cuda:0")
pkg.lib()
case = t.attn_inputs(dev, [144], [2000], 4, 4, 64, torch.bfloat16, 16)
few = t.attn_inputs(dev, [1], [500], 4, 4, 64, torch.bfloat16, 16)
k, v = (torch.nan_to_num(p) for p in case[1:3])
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = pkg.attn_window(*case)
    one = pkg.attn_window(*few)
    pkg.copy_pages(k, v, [0, 1], [126, 127])
graph.replay()
assert torch.equal(out, pkg.attn_window(*case)) and torch.equal(one, pkg.attn_window(*few))
assert torch.equal(k[126:], k[:2]) and torch.equal(v[126:], v[:2])
print("fine")
"""


def test_first_call_under_capture(pkg, cuda):
    """A process whose first use of the operators is a capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = FIRST_CALL.format(root=os.path.dirname(here), tests=here, name=pkg.__name__)
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


def test_session_end_to_end(pkg, cuda):
    """Sessions that grow by frames, fork, evict, compact and move, layer by layer, through the cache's
    methods and one captured graph, against attention over the whole history in 64 bits."""
    layers, h, hk, d, frame, window, sinks = 2, 4, 2, 64, 20, 3, 1
    axes = (16, 24, 24)
    f = pkg.rope_axis_freqs(axes, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    wq, wk = (torch.rand(d, device=cuda, generator=g) + 0.5 for _ in range(2))
    cache = pkg.PagedKVCacheB200(layers, 64, kv_heads=hk, head_dim=d, device=cuda)
    hist = {}  # session -> per layer [(k, v)] of every token, as stored
    kw = dict(axes=axes, q_weight=wq, k_weight=wk)
    look = dict(window=window, sinks=sinks, frame_tokens=frame)

    def frames(seqs, first):
        n = frame * len(seqs)
        x = torch.randn(n, (h + 2 * hk) * d, device=cuda, generator=g).bfloat16()
        t = torch.tensor([cache.length(s) // frame + first for s in seqs], device=cuda).repeat_interleave(frame)
        i = torch.arange(frame, device=cuda).repeat(len(seqs))
        pos = torch.stack([t, i // 5, i % 5], 1).int()
        return [z.unflatten(1, (-1, d)) for z in x.split([h * d, hk * d, hk * d], 1)] + [pos]

    def record(seqs, k, v, pos):
        kk = pkg.qk_norm_rope(k, k, pos, f, axes=axes, q_weight=wk, k_weight=wk)[1]
        for i, s in enumerate(seqs):
            rows = slice(i * frame, (i + 1) * frame)
            hist[s].append((kk[rows], v[rows]))

    def expect(seqs, q, pos, out):
        qq = pkg.qk_norm_rope(q, q, pos, f, axes=axes, q_weight=wq, k_weight=wq)[0]
        for i, s in enumerate(seqs):
            k, v = (torch.cat([p[j] for p in hist[s]]) for j in (0, 1))
            n = k.shape[0]
            pt = 16
            pad = -n % pt
            kp, vp = (torch.nn.functional.pad(z, (0, 0, 0, 0, 0, pad)).unflatten(0, (-1, pt)).transpose(1, 2)
                      for z in (k, v))
            rows = slice(i * frame, (i + 1) * frame)
            ref = attn_ref(qq[rows], kp, vp, torch.arange(kp.shape[0], device=cuda)[None].int(), [n], [0, frame], window, sinks,
                           frame, d ** -0.5)
            check(out[rows], ref[0], attn_tol(ref, BF, d))

    def advance(seqs):
        q, k, v, pos = frames(seqs, 0)
        b = cache.step(seqs, frame)
        record(seqs, k, v, pos)
        for layer in range(layers):
            qo = cache.append(layer, b, q, k, v, pos, f, **kw)
            out = cache.attend(layer, b, qo, **look)
        expect(seqs, q, pos, out)
        return b

    a, b = cache.new(), cache.new()
    hist[a], hist[b] = [], []
    for _ in range(5):
        advance([a, b])
    c, e = cache.fork(a, 2)
    hist[c], hist[e] = list(hist[a]), list(hist[a])
    advance([c, a])
    advance([b])
    for s in (a, b, c):
        assert cache.evict(s, window, sinks, frame) > 0
    advance([a, c, e, b])
    cache.free(c)
    used = cache.compact()
    assert used == 64 - cache.free_pages
    advance([e, a])
    # another solver step of the newest frame: its keys and values anew
    q, k, v, pos = frames([e], -1)
    step = cache.step([e], frame, extend=False)
    hist[e].pop()
    record([e], k, v, pos)
    qo = cache.append(1, step, q, k, v, pos, f, **kw)
    expect([e], q, pos, cache.attend(1, step, qo, **look))
    # a captured step, replayed on later frames
    q, k, v, pos = frames([a, b], 0)
    plan = cache.step([a, b], frame, table_width=30)
    static = [z.clone() for z in (q, k, v, pos)]

    def body():
        for layer in range(layers):
            qo = cache.append(layer, plan, *static, f, **kw)
            o = cache.attend(layer, plan, qo, **look)
        return o

    record([a, b], k, v, pos)
    body()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = body()
    graph.replay()
    expect([a, b], q, pos, out)
    for _ in range(3):
        q, k, v, pos = frames([a, b], 0)
        for z, x in zip(static, (q, k, v, pos)):
            z.copy_(x)
        cache.step([a, b], frame, into=plan)
        record([a, b], k, v, pos)
        graph.replay()
        expect([a, b], q, pos, out)
    # a session moves to another cache
    other = pkg.PagedKVCacheB200(layers, 40, kv_heads=hk, head_dim=d, device=cuda)
    moved = other.adopt(cache, a)
    hist[moved] = hist[a]
    cache.free(a)
    cache, kept = other, cache
    advance([moved])
    assert kept.free_pages > 0


def test_attention_after_evictions_sees_the_whole_window(pkg, cuda):
    """Evict before each frame, write the frame several times (solver steps): attention agrees with the whole
    history; rewrites that reach behind the eviction are refused."""
    h, d, frame, window, sinks = 2, 64, 20, 3, 1
    f = pkg.rope_axis_freqs((64,), device=cuda)
    g = torch.Generator(device=cuda).manual_seed(5)
    cache = pkg.PagedKVCacheB200(1, 40, kv_heads=h, head_dim=d, device=cuda)
    a = cache.new()
    keys, values = [], []
    for i in range(9):
        cache.evict(a, window, sinks, frame)
        pos = torch.arange(i * frame, (i + 1) * frame, device=cuda, dtype=torch.int32)[:, None]
        for rewrite in (False, True, True):
            q, k, v = torch.randn(3, frame, h, d, device=cuda, generator=g).bfloat16()
            plan = cache.step([a], frame, extend=not rewrite)
            qo = cache.append(0, plan, q, k, v, pos, f, axes=(64,), norm=False)
            out = cache.attend(0, plan, qo, window=window, sinks=sinks, frame_tokens=frame)
            q2, k2 = pkg.qk_norm_rope(q, k, pos, f, axes=(64,), norm=False)
            keys[i:], values[i:] = [k2], [v]
            n = (i + 1) * frame
            kp, vp = (torch.nn.functional.pad(torch.cat(z), (0, 0, 0, 0, 0, -n % 16)).unflatten(0, (-1, 16)).transpose(1, 2)
                      for z in (keys, values))
            ref = attn_ref(q2, kp, vp, torch.arange(kp.shape[0], device=cuda)[None].int(), [n], [0, frame], window,
                           sinks, frame, d ** -0.5)
            check(out, ref[0], attn_tol(ref, BF, d))
    assert cache.pages_of(a).count(-1) > 3
    with pytest.raises(ValueError, match="evicted page"):
        cache.step([a], 2 * frame, extend=False)
    cache.truncate(a, 8 * frame - 5)
    with pytest.raises(ValueError, match="evicted page"):
        cache.step([a], 5)


def test_step_on_another_stream(pkg, cuda):
    """step(stream=) makes the plan on that stream: work queued on the current stream keeps its memory."""
    cache = pkg.PagedKVCacheB200(1, 512, kv_heads=1, head_dim=64, device=cuda)
    side = torch.cuda.Stream(device=cuda)
    seqs = [cache.new() for _ in range(64)]
    n = 2 * 64 + 1 + 64 * 40 + 64  # the size of the plan's buffer
    kept = torch.empty(n, dtype=torch.int32, device=cuda)
    for _ in range(4):
        block = torch.arange(n, dtype=torch.int32, device=cuda)
        torch.cuda._sleep(50_000_000)
        kept.copy_(block)  # queued: reads the block after it was given back
        at = block.data_ptr()
        del block
        plan = cache.step(seqs, 1, table_width=40, stream=side)
        assert plan._buffer.data_ptr() != at
        torch.cuda.synchronize()
        assert torch.equal(kept, torch.arange(n, dtype=torch.int32, device=cuda))
        assert plan.kv_len.tolist() == [cache.length(s) for s in seqs]
        assert plan.page_table[:, 0].tolist() == [cache.pages_of(s)[0] for s in seqs]
    # append and attend follow on the same stream
    f = pkg.rope_axis_freqs((64,), device=cuda)
    q, k, v = torch.randn(3, 64, 1, 64, device=cuda).bfloat16()
    pos = torch.zeros(64, 1, dtype=torch.int32, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    qo = cache.append(0, plan, q, k, v, pos, f, axes=(64,), norm=False, stream=side)
    out = cache.attend(0, plan, qo, window=1, stream=side)
    side.synchronize()
    assert torch.equal(out, v)  # a token that sees itself alone


def test_copies_follow_appends_back_to_back(pkg, cuda):
    """A page copy, an append into the copy, a copy of that: each sees what the launch before it stored."""
    hk, d, pt, n = 8, 128, 16, 64
    f = pkg.rope_axis_freqs((d,), device=cuda)
    pos = torch.zeros(n * pt, 1, dtype=torch.int32, device=cuda)
    kp, vp = (torch.zeros(4 * n, hk, pt, d, dtype=BF, device=cuda) for _ in range(2))
    first, second, third = (list(range(i * n, (i + 1) * n)) for i in range(3))
    at = torch.arange(n * pt, dtype=torch.int32, device=cuda)
    slots = [at + i * n * pt for i in range(3)]
    x = [torch.randn(3, n * pt, hk, d, device=cuda).bfloat16() for _ in range(6)]
    got = []
    for i in range(0, 6, 2):
        for (q, k, v), to in ((x[i], 0), (x[i + 1], 1)):
            pkg.qk_norm_rope_append(q, k, v, pos, f, kp, vp, slots[to], axes=(d,), norm=False)
            pkg.copy_pages(kp, vp, first if to == 0 else second, second if to == 0 else third)
        got.append((kp.clone(), vp.clone()))

    def as_pages(z):  # position 0 turns nothing
        return z.unflatten(0, (n, pt)).transpose(1, 2)

    for i, (k, v) in zip(range(0, 6, 2), got):
        for pages, which in ((k, 1), (v, 2)):
            assert torch.equal(pages[:n], as_pages(x[i][which]))
            assert torch.equal(pages[n: 2 * n], as_pages(x[i + 1][which]))
            assert torch.equal(pages[2 * n: 3 * n], as_pages(x[i + 1][which]))
            assert not pages[3 * n:].any()


def test_gradients_are_refused_in_every_argument(pkg, cuda):
    """Backward and forward gradients of any input, and outputs that require them."""
    ad = torch.autograd.forward_ad
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [4], [40], 4, 2, 64, BF, 16)
    x, k, v, pos, wq, wk, f = rope_inputs(pkg, cuda, 4, 4, 2, 64, BF, (16, 24, 24))
    slots = torch.arange(4, device=cuda, dtype=torch.int32)
    kw = dict(axes=(16, 24, 24))

    def attn(q=q, kp=kp, vp=vp, **kw):
        return pkg.attn_window(q, kp, vp, table, lens, cu, **kw)

    def rope(q=x, k=k, f=f, wq=wq, wk=wk, **more):
        return pkg.qk_norm_rope(q, k, pos, f, q_weight=wq, k_weight=wk, **kw, **more)

    def append(q=x, k=k, v=v, f=f, wq=wq, wk=wk, kp=kp, vp=vp, **more):
        return pkg.qk_norm_rope_append(q, k, v, pos, f, kp, vp, slots, q_weight=wq, k_weight=wk, **kw, **more)

    calls = [(attn, dict(q=q, kp=kp, vp=vp, out=torch.empty_like(q))),
             (rope, dict(q=x, k=k, f=f, wq=wq, wk=wk, q_out=torch.empty_like(x), k_out=torch.empty_like(k))),
             (append, dict(q=x, k=k, v=v, f=f, wq=wq, wk=wk, kp=kp, vp=vp, q_out=torch.empty_like(x)))]
    for call, args in calls:
        call()
        for name, t in args.items():
            leaf = t.detach().clone().requires_grad_()
            with pytest.raises(ValueError, match="gradient"):
                call(**{name: leaf})
            with torch.no_grad():
                call(**{name: leaf})
            with ad.dual_level(), torch.no_grad():
                call(**{name: t})
                with pytest.raises(ValueError, match="gradient"):
                    call(**{name: ad.make_dual(t.detach().clone(), torch.ones_like(t))})
    with ad.dual_level(), pytest.raises(ValueError, match="gradient"):
        pkg.copy_pages(ad.make_dual(kp, torch.ones_like(kp)), vp, [0], [1])


def test_outputs_that_overlap_other_tensors_are_refused(pkg, cuda):
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [4], [40], 4, 4, 64, BF, 16)
    x, k, v, pos, wq, wk, f = rope_inputs(pkg, cuda, 4, 4, 4, 64, BF, (64,))
    slots = torch.arange(4, device=cuda, dtype=torch.int32)
    shifted = torch.zeros(7, 4, 64, dtype=BF, device=cuda)
    one = kp.view(-1, 4, 64)
    for call in (lambda: pkg.attn_window(shifted[:4], kp, vp, table, lens, cu, out=shifted[1:5]),
                 lambda: pkg.attn_window(q, kp, vp, table, lens, cu, out=one[:4]),
                 lambda: pkg.qk_norm_rope(x, k, pos, f, axes=(64,), q_out=k),
                 lambda: pkg.qk_norm_rope(x, k, pos, f, axes=(64,), k_out=x),
                 lambda: pkg.qk_norm_rope(x, x, pos, f, axes=(64,), q_out=x, k_out=x),
                 lambda: pkg.qk_norm_rope(x, k, pos, f, axes=(64,), q_out=shifted[:4], k_out=shifted[1:5]),
                 lambda: pkg.qk_norm_rope_append(x, k, v, pos, f, kp, vp, slots, axes=(64,), q_out=v),
                 lambda: pkg.qk_norm_rope_append(x, k, v, pos, f, kp, vp, slots, axes=(64,), q_out=one[:4]),
                 lambda: pkg.qk_norm_rope_append(x, k, v, pos, f, kp, kp, slots, axes=(64,))):
        with pytest.raises((ValueError, pkg.OasisError), match="overlap"):
            call()
    want = pkg.qk_norm_rope(x, k, pos, f, axes=(64,))  # in place among the columns of one projection
    got = pkg.qk_norm_rope(x, k, pos, f, axes=(64,), q_out=x, k_out=k)
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and got[0] is x and got[1] is k


@pytest.mark.parametrize("d,dtype", [(64, BF), (64, HF), (128, BF)])
def test_attn_window_with_non_finite_values_is_reproducible(pkg, cuda, d, dtype):
    """Prompts whose second 128 rows see an infinity in part, which the first 128 do not see: the same bits every
    time, and right ones."""
    n = 80  # enough sequences that no cluster shares the keys of one
    q, kp, vp, table, lens, cu = attn_inputs(cuda, [256] * n, [256] * n, 2, 2, d, dtype, 16)
    for b in range(n):  # token 250 in one head, an early one (seen by all rows after it) in the other
        vp[int(table[b, 15]), 0, 10, 3] = math.inf
        vp[int(table[b, 0]), 1, 5 + b % 8, 7] = -math.inf
    want = pkg.attn_window(q, kp, vp, table, lens, cu, max_q=256)
    for _ in range(20):
        assert torch.equal(pkg.attn_window(q, kp, vp, table, lens, cu, max_q=256).view(torch.int16),
                           want.view(torch.int16))
    for b in (0, n - 1):
        rows = slice(256 * b, 256 * (b + 1))
        ref = attn_ref(q[rows], kp, vp, table[b: b + 1], lens[b: b + 1], [0, 256], None, 0, 1, d ** -0.5)
        fine = ref[0].isfinite()
        check(want[rows][fine], ref[0][fine], attn_tol(ref, dtype, d)[fine])
        assert (want[rows][250:, 0, 3] == math.inf).all() and want[rows][:250, 0, 3].isfinite().all()
