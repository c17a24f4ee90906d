"""Cases of the paged-cache operators: query / key head norms with the rotation over several
position axes (and the append into cache pages), attention over cache pages with a sliding
window and sink frames, and page copies (forks, compaction).

``run`` computes each in its plain form (torch operations in 32 bits, angles in 64), or, where
``own`` is set, calls the package's operators on the same tensors.

Cache pages are ``[layers][pages][kv heads][page tokens][head dim]`` (one layer of them for the
attention and the append), the page table of a sequence lists its pages in order, and the new
tokens of a step are packed ``[tokens][heads][head dim]`` with ``cu_q`` giving where each
sequence's begin.  Frames of 144 tokens, 16 heads of 64, 16 layers and 32-frame windows are this
repository's model; the wider grouped-head sizes are generic.
"""

import importlib
import math

import numpy as np
import torch

own = False

PACKAGE = "efficient-inference-world-models_b200"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one new token of one session enters its cache: a launch's latency
        dict(name="rope append 1 token", op="rope", append=True, tokens=1, heads=16, kv_heads=16,
             head_dim=64, dtype="bf16", axes="16,24,24", interleaved=True, norm=True, page_tokens=16),
        # one new frame of eight sessions: the per-layer step of a rollout
        dict(name="rope append 8 frames", op="rope", append=True, tokens=1152, heads=16, kv_heads=16,
             head_dim=64, dtype="bf16", axes="16,24,24", interleaved=True, norm=True, page_tokens=16),
        # a ragged prompt in 32 bits with grouped heads; a quarter of each head is not rotated
        dict(name="rope fp32 4609 tokens", op="rope", append=False, tokens=4609, heads=24, kv_heads=8,
             head_dim=128, dtype="fp32", axes="32,32,32", interleaved=False, norm=True, page_tokens=16),
        # the full windows of eight sessions at once (a prefill)
        dict(name="rope 36864 tokens", op="rope", append=False, tokens=36864, heads=16, kv_heads=16,
             head_dim=64, dtype="fp16", axes="16,24,24", interleaved=False, norm=True, page_tokens=16),
        # one token of one session over a short cache: latency
        dict(name="attn 1 token, 1 session", op="attn", batch=1, q_min=1, q_max=1, kv_min=577, kv_max=577,
             heads=16, kv_heads=16, head_dim=64, dtype="bf16", page_tokens=16, frame_tokens=1,
             window=0, sinks=0),
        # single tokens of 32 sequences of ragged lengths, grouped heads, window and sinks
        dict(name="attn 1 token, 32 sequences", op="attn", batch=32, q_min=1, q_max=1, kv_min=2001,
             kv_max=16384, heads=32, kv_heads=8, head_dim=128, dtype="bf16", page_tokens=16,
             frame_tokens=1, window=8192, sinks=16),
        # one new frame of one session against 32 frames and the first: the rollout's step
        dict(name="attn 1 frame, 1 session", op="attn", batch=1, q_min=144, q_max=144, kv_min=7056,
             kv_max=7056, heads=16, kv_heads=16, head_dim=64, dtype="bf16", page_tokens=16,
             frame_tokens=144, window=32, sinks=1),
        # the same step of eight sessions of different ages
        dict(name="attn 1 frame, 8 sessions", op="attn", batch=8, q_min=144, q_max=144, kv_min=1440,
             kv_max=9216, heads=16, kv_heads=16, head_dim=64, dtype="fp16", page_tokens=16,
             frame_tokens=144, window=32, sinks=1),
        # a long odd-sized prompt with grouped heads, token-wise window and sinks: the largest
        dict(name="attn prompt of 8191", op="attn", batch=1, q_min=8191, q_max=8191, kv_min=8191,
             kv_max=8191, heads=32, kv_heads=8, head_dim=128, dtype="bf16", page_tokens=64,
             frame_tokens=1, window=4096, sinks=64),
        # the shared last page of one forked session is copied before it is written to
        dict(name="pages 1", op="pages", pages=1, layers=16, kv_heads=16, head_dim=64, dtype="bf16",
             page_tokens=16, fan=1),
        # eight sessions forked into four branches each (every last frame copied)
        dict(name="pages 288", op="pages", pages=288, layers=16, kv_heads=16, head_dim=64, dtype="bf16",
             page_tokens=16, fan=4),
        # a pool half emptied by evictions is compacted
        dict(name="pages 1500", op="pages", pages=1500, layers=16, kv_heads=16, head_dim=64, dtype="fp16",
             page_tokens=16, fan=1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "attn", "attn", "pages"))
    head_dim = rng.choice((64, 128))
    if op == "pages":
        fan, page_tokens = rng.choice((1, 1, 3, 4)), rng.choice((16, 32, 64))
        layers, kv_heads = rng.randint(1, 16), rng.choice((1, 2, 5, 8, 16))
        most = 1500 * 16 * 16 * 16 * 64 // (page_tokens * layers * kv_heads * head_dim)
        return dict(op=op, pages=fan * max(1, _log(rng, 1, min(4000, most)) // fan), layers=layers,
                    kv_heads=kv_heads, head_dim=head_dim, dtype=rng.choice(("bf16", "fp16")),
                    page_tokens=page_tokens, fan=fan)
    kv_heads, group = rng.choice((1, 2, 4, 6, 8, 16)), rng.choice((1, 2, 3, 4, 5, 8))
    if op == "rope":
        append = rng.random() < 0.5
        axes = {64: ("16,24,24", "64", "32,32", "8,12,12", "24,20,20"),
                128: ("44,42,42", "128", "64,64", "32,32,32", "16,16")}[head_dim]
        most = 36864 * 32 * 64 // ((group + 1) * kv_heads * head_dim)
        return dict(op=op, append=append, tokens=_log(rng, 1, min(36864, most // 2)), heads=kv_heads * group,
                    kv_heads=kv_heads, head_dim=head_dim,
                    dtype=rng.choice(("bf16", "fp16") if append else ("bf16", "fp16", "fp32")),
                    axes=rng.choice(axes), interleaved=rng.random() < 0.5, norm=rng.random() < 0.8,
                    page_tokens=rng.choice((16, 32, 64)))
    kind = rng.choice(("token", "tokens", "frame", "prompt"))
    frame_tokens = rng.choice((1, 144, 60)) if kind != "frame" else rng.choice((144, 60, 256))
    case = dict(op=op, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                dtype=rng.choice(("bf16", "fp16")), page_tokens=rng.choice((16, 32, 64)), frame_tokens=frame_tokens)
    if kind == "prompt":
        batch = rng.randint(1, 3)
        q = _log(rng, 200, 4500 // batch)
        case.update(batch=batch, q_min=max(1, q // 2), q_max=q, kv_min=q, kv_max=q + _log(rng, 1, 1000))
    else:
        batch = _log(rng, 1, 32)
        kv = _log(rng, 300, 16384)
        q = {"token": 1, "tokens": rng.randint(2, 9), "frame": frame_tokens}[kind]
        batch = max(1, min(batch, int(6e8 / (kv * q * kv_heads * group)), int(6e8 / (kv * kv_heads * head_dim))))
        case.update(batch=batch, q_min=q, q_max=q, kv_min=max(q, kv // 3), kv_max=max(q, kv))
    span = max(1, case["kv_max"] // frame_tokens)
    case.update(window=rng.choice((0, _log(rng, 1, span), _log(rng, max(1, span // 4), span))))
    case.update(sinks=0 if not case["window"] else rng.choice((0, 1, 4, 33)))
    return case


# ------------------------------------------------------------------ inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _frequencies(axes):
    """Angular frequency of every rotated pair: axis a of d dimensions has d/2 of 10000^(-2i/d)."""
    parts = [10000.0 ** (-2.0 * np.arange(d // 2) / d) for d in axes]
    return torch.from_numpy(np.concatenate(parts)).to("cuda")


def prepare(case, seed):
    return {"rope": _prepare_rope, "attn": _prepare_attn, "pages": _prepare_pages}[case["op"]](case, seed)


def _prepare_rope(case, seed):
    g, r = _generator(seed), np.random.RandomState(seed % (1 << 32))
    n, h, hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim"))
    dtype, axes = DTYPES[case["dtype"]], tuple(int(a) for a in case["axes"].split(","))
    # queries, keys and values as one projection leaves them: columns of one row per token
    qkv = _randn(g, n, (h + 2 * hk) * d, dtype=dtype)
    s = dict(op="rope", axes=axes, interleaved=case["interleaved"], norm=case["norm"], append=case["append"],
             q=qkv[:, : h * d].view(n, h, d), k=qkv[:, h * d: (h + hk) * d].view(n, hk, d),
             v=qkv[:, (h + hk) * d:].view(n, hk, d), freqs=_frequencies(axes))
    # tokens of 9 x 16 grids, frames that are far from the first
    t = np.arange(n)
    grid = np.stack([t // 144 + r.randint(0, 100000), t % 144 // 16, t % 16], 1)
    s["positions"] = torch.from_numpy(grid[:, : len(axes)].copy()).to("cuda", torch.int32)
    s["q_weight"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    s["k_weight"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
    if case["append"]:
        pt = case["page_tokens"]
        pages = -(-n // pt) + 3
        s["k_pages"] = _randn(g, pages, hk, pt, d, dtype=dtype)
        s["v_pages"] = _randn(g, pages, hk, pt, d, dtype=dtype)
        order = r.permutation(pages)
        at = t + r.randint(0, pt)  # the first page already holds some tokens
        s["slots"] = torch.from_numpy(order[at // pt] * pt + at % pt).to("cuda", torch.int32)
    return s


def _lengths(case):
    """Queries and cached tokens (the queries' own among them) of every sequence: the same for every seed."""
    r = np.random.RandomState(7)
    b = case["batch"]
    q = r.randint(case["q_min"], case["q_max"] + 1, b)
    kv = np.maximum(q, r.randint(case["kv_min"], case["kv_max"] + 1, b))
    if case["frame_tokens"] > 1 and case["q_min"] == case["frame_tokens"]:  # whole frames
        kv = np.maximum(q, kv // case["frame_tokens"] * case["frame_tokens"])
    return q, kv


def _prepare_attn(case, seed):
    g, r = _generator(seed), np.random.RandomState(seed % (1 << 32))
    q_len, kv_len = _lengths(case)
    h, hk, d, pt = (case[k] for k in ("heads", "kv_heads", "head_dim", "page_tokens"))
    dtype = DTYPES[case["dtype"]]
    need = -(-kv_len // pt)
    pages = int(need.sum()) + 2
    order = r.permutation(pages)
    table = np.full((case["batch"], int(need.max())), -1, np.int32)
    filled = np.arange(table.shape[1])[None] < need[:, None]
    table[filled] = order[: int(need.sum())]
    cu = np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)
    # queries of some heads look far more sharply than others'
    sharp = torch.linspace(0.5, 2.5, h, device="cuda")[:, None]
    q = (torch.randn(int(cu[-1]), h, d, generator=g, device="cuda") * sharp).to(dtype)
    return dict(op="attn", q=q, k_pages=_randn(g, pages, hk, pt, d, dtype=dtype),
                v_pages=_randn(g, pages, hk, pt, d, dtype=dtype), table=torch.from_numpy(table).to("cuda"),
                kv_len=torch.from_numpy(kv_len.astype(np.int32)).to("cuda"), cu_q=torch.from_numpy(cu).to("cuda"),
                max_q=int(q_len.max()), max_kv=int(kv_len.max()), window=case["window"] or None,
                sinks=case["sinks"], frame_tokens=case["frame_tokens"])


def _prepare_pages(case, seed):
    g, r = _generator(seed), np.random.RandomState(seed % (1 << 32))
    n, fan = case["pages"], case["fan"]
    pages = n + n // fan + 2
    shape = (case["layers"], pages, case["kv_heads"], case["page_tokens"], case["head_dim"])
    dtype = DTYPES[case["dtype"]]
    order = r.permutation(pages).astype(np.int32)
    return dict(op="pages", k=_randn(g, *shape, dtype=dtype), v=_randn(g, *shape, dtype=dtype),
                src=torch.from_numpy(np.repeat(order[n: n + n // fan], fan)[:n].copy()),
                dst=torch.from_numpy(order[:n].copy()))


# ------------------------------------------------------------------ one pass


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _plain_rope, "attn": _plain_attn, "pages": _plain_pages}[s["op"]](s)


def _run_own(s):
    b200 = importlib.import_module(PACKAGE)
    if s["op"] == "pages":
        b200.copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return s["k"], s["v"]
    if s["op"] == "attn":
        return b200.attn_window(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_len"], s["cu_q"],
                                window=s["window"], sinks=s["sinks"], frame_tokens=s["frame_tokens"],
                                max_q=s["max_q"], max_kv=s["max_kv"])
    kw = dict(axes=s["axes"], interleaved=s["interleaved"], norm=s["norm"])
    if s["norm"]:
        kw.update(q_weight=s["q_weight"], k_weight=s["k_weight"])
    if s["append"]:
        q = b200.qk_norm_rope_append(s["q"], s["k"], s["v"], s["positions"], s["freqs"], s["k_pages"],
                                     s["v_pages"], s["slots"], **kw)
        return q, s["k_pages"], s["v_pages"]
    return b200.qk_norm_rope(s["q"], s["k"], s["positions"], s["freqs"], **kw)


def _plain_norm_rope(x, weight, cos, sin, s):
    y = x.float()
    if s["norm"]:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight
    rot = 2 * cos.shape[-1]
    r, rest = y[..., :rot], y[..., rot:]
    if s["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([r, rest], -1).to(x.dtype)


def _plain_rope(s):
    owner = torch.repeat_interleave(torch.arange(len(s["axes"])), torch.tensor([a // 2 for a in s["axes"]]))
    angle = s["positions"].double()[:, owner.to("cuda")] * s["freqs"]  # 64 bits: positions may be far
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q = _plain_norm_rope(s["q"], s["q_weight"], cos, sin, s)
    k = _plain_norm_rope(s["k"], s["k_weight"], cos, sin, s)
    if not s["append"]:
        return q, k
    pt = s["k_pages"].shape[2]
    page, at = s["slots"].long() // pt, s["slots"].long() % pt
    s["k_pages"][page, :, at] = k
    s["v_pages"][page, :, at] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _plain_attn(s):
    q, table, cu, kv_len = s["q"], s["table"].long().clamp_min(0), s["cu_q"].long(), s["kv_len"].long()
    n, h, d = q.shape
    hk, pt = s["k_pages"].shape[1:3]
    b, w = table.shape
    k, v = (p[table].permute(0, 2, 1, 3, 4).reshape(b, hk, w * pt, d).float() for p in (s["k_pages"], s["v_pages"]))
    row = torch.arange(s["max_q"], device=q.device)
    q_len = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + row).clamp_max(n - 1)
    qs = q[at].float().reshape(b, s["max_q"], hk, h // hk, d)
    score = torch.matmul(qs.permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d) * d ** -0.5, k.transpose(2, 3))
    score = score.view(b, hk, h // hk, s["max_q"], w * pt)
    f = s["frame_tokens"]
    key = torch.arange(w * pt, device=q.device)
    q_frame = ((kv_len - q_len)[:, None] + row).div(f, rounding_mode="floor")[:, :, None]
    see = (key // f <= q_frame) & (key < kv_len[:, None, None])
    if s["window"]:
        see &= (q_frame - key // f < s["window"]) | (key // f < s["sinks"])
    score = score.masked_fill_(~see[:, None, None], -torch.inf)
    p = score.sub_(score.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, hk, -1, w * pt), v).view(b, hk, h // hk, s["max_q"], d) / total.clamp_min(1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], h, d).to(q.dtype)
    return out[row < q_len[:, None]]


def _plain_pages(s):
    src, dst = s["src"].to("cuda").long(), s["dst"].to("cuda").long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


# ------------------------------------------------------------------ what a pass cannot do without


def _visible(q_len, kv_len, case):
    """(keys that some query sees, pairs of a query and a key that it sees) of one sequence."""
    f, w, sinks = case["frame_tokens"], case["window"], case["sinks"]
    p = np.arange(kv_len - q_len, kv_len, dtype=np.int64)
    end = np.minimum((p // f + 1) * f, kv_len)
    start = np.maximum(0, (p // f - w + 1) * f) if w else np.zeros_like(p)
    sink = np.minimum(np.minimum(sinks * f, start), end) if w else np.zeros_like(p)
    keys = end.max() - start.min() + min(sinks * f, start.min()) if w else end.max()
    return int(keys), int((end - start + sink).sum())


def work(case):
    d = case["head_dim"]
    if case["op"] == "pages":
        page = case["layers"] * case["kv_heads"] * case["page_tokens"] * d * 2 * 2
        return {"bytes": page * (case["pages"] + case["pages"] // case["fan"]), "flops": 0}
    h, hk = case["heads"], case["kv_heads"]
    if case["op"] == "rope":
        size = DTYPES[case["dtype"]].itemsize
        values = (h + hk) * d + (hk * d if case["append"] else 0)
        return {"bytes": case["tokens"] * (2 * values * size + 4 * len(case["axes"].split(","))),
                "flops": 8 * case["tokens"] * (h + hk) * d}
    q_len, kv_len = _lengths(case)
    seen = [_visible(int(q), int(k), case) for q, k in zip(q_len, kv_len)]
    return {"bytes": sum(k for k, _ in seen) * hk * d * 2 * 2 + 2 * int(q_len.sum()) * h * d * 2,
            "flops": 4 * d * h * sum(p for _, p in seen)}


# ------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pages":
        if s["k"].numel() > 1 << 28:
            return None
        k, v = s["k"].double(), s["v"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
        return k, v
    if case["op"] == "rope":
        return _exact_rope(s)
    return _exact_attn(s, case)


def _exact_rope(s):
    angle = torch.cat([s["positions"][:, i, None].double() * f for i, f in
                       enumerate(s["freqs"].split([a // 2 for a in s["axes"]]))], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    half = turn.shape[-1]

    def one(x, weight):
        x = x.double()
        if s["norm"]:
            x = x * weight.double() / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        z = x[..., : 2 * half]
        z = z.unflatten(-1, (half, 2)) if s["interleaved"] else z.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
        z = z if s["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), x[..., 2 * half:]], -1)

    q, k = one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])
    if not s["append"]:
        return q, k
    pages = [s["k_pages"].double(), s["v_pages"].double()]
    for p, x in zip(pages, (k, s["v"].double())):
        flat = p.transpose(1, 2).reshape(-1, *p.shape[1:2], p.shape[3])  # [slot][head][dim]
        flat[s["slots"].long()] = x
        p.copy_(flat.view(p.shape[0], p.shape[2], p.shape[1], p.shape[3]).transpose(1, 2))
    return (q, *pages)


def _exact_attn(s, case):
    h, hk, d, pt, f = (case[k] for k in ("heads", "kv_heads", "head_dim", "page_tokens", "frame_tokens"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, lens = s["cu_q"].tolist(), s["kv_len"].tolist()
    for b, n in enumerate(lens):
        pages = s["table"][b, : -(-n // pt)].long()
        m = cu[b + 1] - cu[b]
        query, key = torch.arange(n - m, n, device="cuda")[:, None] // f, torch.arange(n, device="cuda") // f
        hidden = key > query
        if case["window"]:
            hidden |= (key <= query - case["window"]) & (key >= case["sinks"])
        for j in range(hk):
            k, v = (p[pages, j].reshape(-1, d)[:n].double() for p in (s["k_pages"], s["v_pages"]))
            for i in range(j * (h // hk), (j + 1) * (h // hk)):
                score = s["q"][cu[b]: cu[b + 1], i].double() @ k.T / math.sqrt(d)
                score[hidden] = -math.inf
                out[cu[b]: cu[b + 1], i] = torch.softmax(score, -1) @ v
    return out
