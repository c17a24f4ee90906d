"""Host side of the paged cache: the book of pages (on CPU tensors, where no kernel runs) and the
C entry points' refusals (checked before any launch)."""

import ctypes

import numpy as np
import pytest
import torch

P = ctypes.c_void_p


def make(pkg, pages=12, layers=2, **kw):
    c = pkg.PagedKVCacheB200(layers, pages, page_tokens=16, kv_heads=2, head_dim=64, device="cpu", **kw)

    def copy(src, dst, stream=None):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        c.k[:, dst], c.v[:, dst] = c.k[:, src], c.v[:, src]

    c.copy_pages = copy  # the device copy, restated for CPU tensors
    return c


def fill(c, seq, first, values):
    """Token first + i of the session holds the number values[i]."""
    for i, x in enumerate(values):
        page = c.pages_of(seq)[(first + i) // 16]
        c.k[:, page, :, (first + i) % 16] = x
        c.v[:, page, :, (first + i) % 16] = -x


def read(c, seq, first=0):
    out = []
    for i in range(first, c.length(seq)):
        page = c.pages_of(seq)[i // 16]
        out.append(float(c.k[0, page, 0, i % 16, 0]))
        assert float(c.v[1, page, 1, i % 16, 63]) == -out[-1]
    return out


def owned(c):
    """Every page is free or referenced as often as the sessions list it."""
    held = [p for s in c.sessions for p in c.pages_of(s) if p >= 0]
    for p in range(c.pages):
        assert c._refs[p] == held.count(p)
    assert sorted(c._free) == [p for p in range(c.pages) if p not in held]


def test_step_plan_arrays(pkg):
    c = make(pkg)
    a, b = c.new(), c.new()
    s = c.step([a, b], [20, 3])
    assert s.cu_q.tolist() == [0, 20, 23] and s.kv_len.tolist() == [20, 3]
    assert s.page_table.tolist() == [c.pages_of(a), c.pages_of(b) + [-1]]
    pa, pb = c.pages_of(a), c.pages_of(b)
    assert s.slots.tolist() == ([pa[0] * 16 + i for i in range(16)] + [pa[1] * 16 + i for i in range(4)]
                                + [pb[0] * 16 + i for i in range(3)])
    assert (s.max_q, s.max_kv) == (20, 32)
    again = c.step([b, a], [1, 0], extend=False)  # the last token of b anew, a only looked at
    assert again.slots.tolist() == [pb[0] * 16 + 2] and again.kv_len.tolist() == [3, 20]
    assert not s.stale and c.length(b) == 3
    owned(c)


def test_fork_shares_until_written(pkg):
    c = make(pkg)
    a = c.new()
    c.step([a], 20)
    fill(c, a, 0, range(20))
    b, d = c.fork(a, 2)
    assert c.free_pages == 10 and c.pages_of(b) == c.pages_of(a)
    c.step([a, b, d], [1, 2, 0])  # a and b write into the shared second page, d keeps it
    owned(c)
    assert len({c.pages_of(x)[1] for x in (a, b, d)}) == 3
    assert len({c.pages_of(x)[0] for x in (a, b, d)}) == 1
    fill(c, a, 20, [100])
    fill(c, b, 20, [200, 201])
    base = [float(i) for i in range(20)]
    assert read(c, a) == base + [100] and read(c, b) == base + [200, 201] and read(c, d) == base
    c.step([d], 1)  # the last sharer writes in place
    assert c.free_pages == 12 - 4
    c.step([b], 20, extend=False)  # rewriting back into the shared first page copies it
    assert c.pages_of(b)[0] != c.pages_of(a)[0] and read(c, b)[:2] == [0.0, 1.0]
    owned(c)
    for s in (a, b, d):
        c.free(s)
    assert c.free_pages == 12


def test_full_cache_refuses_and_changes_nothing(pkg):
    c = make(pkg, pages=3)
    a = c.new()
    c.step([a], 40)
    b = c.fork(a)[0]
    before = (c.pages_of(a), c.pages_of(b), list(c._refs), list(c._free))
    with pytest.raises(RuntimeError, match="1 pages needed, 0 free"):
        c.step([a, b], 1)
    assert before == (c.pages_of(a), c.pages_of(b), list(c._refs), list(c._free)) and c.length(a) == 40


def test_evict_truncate_compact(pkg):
    c = make(pkg, pages=20)
    a, b = c.new(), c.new()
    c.step([a, b], [100, 40])
    fill(c, a, 0, range(100))
    fill(c, b, 0, range(200, 240))
    # the next token (100) sees 70..100 and 0..3: pages of 16..63 go
    assert c.evict(a, window=31, sinks=4) == 3
    assert [p < 0 for p in c.pages_of(a)] == [False, True, True, True, False, False, False]
    assert c.evict(a, window=31, sinks=4) == 0
    owned(c)
    c.truncate(b, 17)
    assert c.free_pages == 20 - 4 - 2
    old = c.step([b], 0)
    assert c.compact() == 6 and old.stale
    assert sorted(p for s in (a, b) for p in c.pages_of(s) if p >= 0) == list(range(6))
    owned(c)
    assert read(c, b) == [float(x) for x in range(200, 217)]
    assert read(c, a, 64) == [float(x) for x in range(64, 100)]
    with pytest.raises(ValueError, match="evicted page"):
        c.step([a], 60, extend=False)
    # frames of 10 tokens, window of 2 frames: token 100 (frame 10) sees from token 90 on
    assert c.evict(a, window=2, frame_tokens=10) == 2 and c.pages_of(a)[:5] == [-1] * 5


def test_plans_go_stale_and_are_rebuilt(pkg):
    c = make(pkg)
    a, b = c.new(), c.new()
    s = c.step([a, b], 1, table_width=4)
    assert s.max_kv == 64
    buf = s.kv_len.data_ptr()
    c.step([a, b], 1, into=s)
    assert s.kv_len.tolist() == [2, 2] and s.kv_len.data_ptr() == buf and not s.stale
    c.step([a], 1)
    with pytest.raises(ValueError, match="out of date"):
        c.attend(0, s, torch.zeros(2, 2, 64))
    with pytest.raises(ValueError, match="room for 4"):
        c.step([a, b], [80, 1], into=s)
    with pytest.raises(ValueError, match="2 sessions and 2 tokens"):
        c.step([a, b], [2, 1], into=s)
    other = c.new()
    c.step([a, other], 1, into=s)
    c.free(b)  # no longer one of the plan's
    assert not s.stale
    c.free(other)
    assert s.stale


def test_plans_of_forked_sessions_and_of_other_caches(pkg):
    """A plan must not write into pages that a fork shares, nor be used on another cache."""
    c, other = make(pkg), make(pkg)
    a = c.new()
    s = c.step([a], 3)
    b = c.fork(a)[0]
    z = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="out of date"):
        c.append(0, s, z, z, z, None, None, axes=(64,))
    again = c.step([a], 3, extend=False)  # the same tokens, in a page of its own
    assert c.pages_of(a) != c.pages_of(b) and not again.stale
    owned(c)
    n = other.new()
    for call in (lambda: other.attend(0, again, z), lambda: other.step([n], 3, into=again)):
        with pytest.raises(ValueError, match="another cache"):
            call()


def seen_pages(plan, row, first, window, sinks, frame):
    """The plan's page entries that hold tokens visible to the query at position `first`."""
    n = int(plan.kv_len[row])
    end = min((first // frame + 1) * frame, n)
    start = max(0, (first // frame - window + 1) * frame)
    tokens = [j for j in range(end) if j >= start or j < sinks * frame]
    return [int(plan.page_table[row, i]) for i in sorted({j // 16 for j in tokens})]


@pytest.mark.parametrize("window,sinks,frame,length", [(2, 1, 20, 120), (3, 0, 16, 96), (2, 0, 10, 95), (40, 5, 1, 100)])
def test_evicted_pages_are_not_in_sight_of_any_step(pkg, window, sinks, frame, length):
    """After an eviction every step that is taken sees all it should; one that would not is refused."""
    c = make(pkg, pages=20)
    a = c.new()
    c.step([a], length)
    assert c.evict(a, window, sinks, frame) > 0
    b = c.fork(a)[0]
    before = (c.pages_of(a), list(c._refs), list(c._free), c.length(a))
    refused = 0
    for n in range(1, 2 * frame + 18):  # the last n tokens again
        try:
            plan = c.step([a], n, extend=False)
        except ValueError as e:
            assert "evicted page" in str(e)
            refused += 1
            continue
        for first in range(length - n, length):
            assert min(seen_pages(plan, 0, first, window, sinks, frame)) >= 0
    assert refused
    # what the eviction was for goes on: later tokens, and those again; the fork remembers as well
    for s in (a, b):
        done = c.step([s], 7)
        again = c.step([s], 7, extend=False)
        for plan in (done, again):
            for first in range(length, length + 7):
                assert min(seen_pages(plan, 0, first, window, sinks, frame)) >= 0
    with pytest.raises(ValueError, match="evicted page"):
        c.step([b], 2 * frame + 24, extend=False)
    assert before[3] == length and c.length(a) == c.length(b) == length + 7
    owned(c)


def test_refused_step_after_eviction_changes_nothing(pkg):
    c = make(pkg, pages=20)
    a, b = c.new(), c.new()
    c.step([a, b], [120, 10])
    assert c.evict(a, window=2, sinks=1, frame_tokens=20) == 4  # pages 2..5: frame 6 sees 100 and later
    plan = c.step([b], 1)
    before = (c.pages_of(a), c.pages_of(b), list(c._refs), list(c._free), c.length(a), c.length(b))
    for seqs, tokens in (([b, a], [5, 20]), ([a], [20])):  # frame 5 sees frame 4 (80 .. 99)
        with pytest.raises(ValueError, match="evicted page"):
            c.step(seqs, tokens, extend=False)
    assert before == (c.pages_of(a), c.pages_of(b), list(c._refs), list(c._free), c.length(a), c.length(b))
    assert not plan.stale
    owned(c)


def test_evict_truncate_step(pkg):
    """Rejected frames are generated anew: refused where they see what was evicted, and not otherwise."""
    c = make(pkg, pages=20)
    a = c.new()
    c.step([a], 120)
    c.evict(a, window=2, frame_tokens=20)  # the next frame is 6: pages 0..5 (tokens 0..95) go
    assert c.pages_of(a) == [-1] * 6 + c.pages_of(a)[6:]
    c.truncate(a, 100)
    with pytest.raises(ValueError, match="evicted page"):
        c.step([a], 20)  # frame 5 sees frame 4
    assert c.length(a) == 100
    c.truncate(a, 0)  # all of it goes, and with it what was evicted
    plan = c.step([a], 40)
    assert min(plan.page_table[0].tolist()) >= 0
    owned(c)


def test_evictions_under_different_windows(pkg):
    """A session is held to the windows under which its pages went, not to others."""
    c = make(pkg, pages=20)
    a = c.new()
    c.step([a], 100)
    assert c.evict(a, window=31, sinks=20) == 2      # pages 2, 3; the sinks' 0, 1 stay
    assert c.evict(a, window=31) == 2                # no sinks any more
    assert c.pages_of(a)[:5] == [-1] * 4 + c.pages_of(a)[4:5]
    c.step([a], 6, extend=False)                     # token 94 sees from 64 on
    with pytest.raises(ValueError, match="evicted page"):
        c.step([a], 7, extend=False)                 # token 93 sees token 63
    c.step([a], 1)
    assert c.evict(a, window=5) == 2                 # the next token (101) sees from 97 on
    c.step([a], 1, extend=False)
    with pytest.raises(ValueError, match="evicted page"):
        c.step([a], 6, extend=False)                 # token 95 sees from 91 on
    owned(c)


@pytest.mark.parametrize("where", ["copy", "plan", "upload", "rebuild"])
def test_step_that_raises_changes_nothing(pkg, monkeypatch, where):
    """A failing copy, plan allocation or upload leaves the book and the plans as they were."""
    c = make(pkg, pages=20)
    a = c.new()
    c.step([a], 40)
    fill(c, a, 0, range(40))
    b, d = c.fork(a, 2)
    live = c.step([d], 0)
    old = c.step([a, b], [0, 0], table_width=5)

    def book():
        return ([(c.pages_of(x), c.length(x)) for x in (a, b, d)], list(c._refs), list(c._free), live.stale,
                old.stale, old.seqs, old.kv_len.tolist(), old.page_table.tolist(), read(c, a), read(c, b), read(c, d))

    before = book()

    def fail(*args, **kw):
        raise RuntimeError("planted")

    copy = c.copy_pages
    with monkeypatch.context() as m:
        if where == "copy":
            m.setattr(c, "copy_pages", fail)
        elif where == "plan":
            m.setattr(pkg.paged, "PagedBatchB200", fail)
        else:
            m.setattr(torch, "from_numpy", fail)
        with pytest.raises(RuntimeError, match="planted"):
            if where == "rebuild":
                c.step([a, b], [0, 0], into=old, extend=True)
            else:
                c.step([a, b, d], [3, 20, 0])
    assert before == book()
    owned(c)
    assert c.copy_pages is copy
    c.step([a, b, d], [3, 20, 0])  # and it goes on from there
    assert read(c, a)[:40] == read(c, b)[:40] == read(c, d) == [float(i) for i in range(40)]
    owned(c)


def test_plan_is_allocated_under_the_given_stream(pkg, monkeypatch):
    """The plan's memory belongs to the stream that fills it."""
    c = make(pkg)
    a = c.new()
    inside, made = [], []

    class Context:
        def __enter__(self):
            inside.append(True)

        def __exit__(self, *exc):
            inside.pop()

    plan = pkg.paged.PagedBatchB200

    def make_plan(*args):
        made.append(bool(inside))
        return plan(*args)

    monkeypatch.setattr(pkg.paged, "_elsewhere", lambda device, stream: Context() if stream else None)
    monkeypatch.setattr(pkg.paged, "PagedBatchB200", make_plan)
    c.step([a], 3, stream="another")
    c.step([a], 3)
    assert made == [True, False]


def test_fork_takes_whole_numbers(pkg):
    c = make(pkg)
    a = c.new()
    c.step([a], 20)
    before = (c.sessions, list(c._refs), list(c._free))
    for copies in (1.5, "2", None, -1):
        with pytest.raises((TypeError, ValueError)):
            c.fork(a, copies)
    assert before == (c.sessions, list(c._refs), list(c._free))
    assert len(c.fork(a, np.int64(2))) == 2
    owned(c)


@pytest.mark.parametrize("bad", ["twice", "none", "unknown", "negative", "few", "rewrite"])
def test_step_refusals(pkg, bad):
    c = make(pkg)
    a, b = c.new(), c.new()
    args = {"twice": ([a, a], 1), "none": ([], 1), "unknown": ([a, 9], 1), "negative": ([a], -1),
            "few": ([a, b], [1]), "rewrite": ([a], 1)}[bad]
    with pytest.raises(ValueError):
        c.step(*args, extend=bad != "rewrite")
    assert c.free_pages == 12 and c.length(a) == 0


def test_cache_refusals(pkg):
    for kw in (dict(page_tokens=8), dict(head_dim=80), dict(dtype=torch.float32), dict(pages=0)):
        args = dict(layers=1, pages=2, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            pkg.PagedKVCacheB200(**args)
    c = make(pkg)
    a = c.new()
    others = [make(pkg, layers=3), make(pkg, dtype=torch.float16)]
    for o in others:
        o.new()
    for call in (lambda: c.adopt(others[0], 0), lambda: c.adopt(others[1], 0), lambda: c.fork(a, -1), lambda: c.truncate(a, 1), lambda: c.evict(a, 0), lambda: c.free(7),
                 lambda: c.adopt(c, a)):
        with pytest.raises(ValueError):
            call()


def test_axis_frequencies(pkg):
    f = pkg.rope_axis_freqs((4, 2, 6), theta=(100.0, 7.0, 10000.0), device="cpu")
    want = [1.0, 0.1, 1.0] + [10000.0 ** (-2 * i / 6) for i in range(3)]
    assert f.dtype == torch.float64
    np.testing.assert_allclose(f.numpy(), want, rtol=1e-15)
    for axes, theta in (((3,), 10.0), ((), 10.0), ((4,), -1.0), ((4, 4), (1.0,))):
        with pytest.raises(ValueError):
            pkg.rope_axis_freqs(axes, theta, device="cpu")


def test_no_gradient_is_dropped_silently(pkg):
    """Inputs that require gradients, backward or forward, are refused."""
    check = pkg.paged._no_grad
    x = torch.zeros(4, 2, 64)
    check(x, None)
    with pytest.raises(ValueError, match="gradient"):
        check(x, x.clone().requires_grad_())
    with torch.no_grad():
        check(x.clone().requires_grad_())
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        check(x, None)
        with pytest.raises(ValueError, match="gradient"):
            check(x, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="gradient"):
            check(dual)  # tangents pass through no_grad
        check(torch.autograd.forward_ad.unpack_dual(dual).primal)
    out = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        pkg.paged._out_check("out", out, x)
    with torch.no_grad():
        pkg.paged._out_check("out", out, x)


def test_overlap_of_views_matches_a_count_of_elements(pkg):
    """Random [tokens][heads][dims] views of one buffer: _overlap against the sets of their elements."""
    rng = np.random.RandomState(0)
    base = torch.zeros(4096, dtype=torch.bfloat16)
    where = torch.arange(4096)
    found = [0, 0]
    for i in range(600):
        views = []
        for _ in range(2):
            t, h, d = rng.randint(1, 6), rng.randint(1, 5), 8 * rng.randint(1, 4)
            strides = sorted(8 * rng.randint(0, 12, 2))
            if rng.rand() < 0.5:
                strides.reverse()
            if views and rng.rand() < 0.7:  # mostly of one token stride, as the columns of a projection
                strides = [views[0][1][0], strides[1]]
            views.append(((t, h, d), [int(x) for x in strides] + [1], int(8 * rng.randint(0, 120))))
        a, b = (torch.as_strided(base, *v) for v in views)
        x, y = (set(torch.as_strided(where, *v).flatten().tolist()) for v in views)
        found[bool(x & y)] += 1
        assert pkg.paged._overlap(a, b) == bool(x & y), views
        assert pkg.paged._overlap(b, a) == bool(x & y), views
        assert pkg.paged._folds(a) == (len(x) < a.numel()), views[0]
    assert min(found) > 100
    assert not pkg.paged._overlap(base[:0].view(0, 2, 8), base.view(-1, 2, 8))


def test_outputs_stay_off_other_tensors(pkg):
    qkv = torch.zeros(6, 12 * 64, dtype=torch.bfloat16)
    q, k, v = (z.unflatten(1, (4, 64)) for z in qkv.split(4 * 64, 1))
    check = pkg.paged._out_check
    check("q_out", q, q, k=k, v=v)  # its own input, between the others
    check("q_out", torch.empty_like(q), q, k=k, v=v)
    check("q_out", torch.zeros(4, 6, 64, dtype=torch.bfloat16).transpose(0, 1), q, k=k, v=v)
    check("k_out", k, k, q=q, q_out=q)
    rows = torch.zeros(9, 4, 64, dtype=torch.bfloat16)
    for out, like, others in ((k, q, dict(k=k)),                            # another input
                              (rows[1:7], rows[:6], {}),                    # its input, one row on
                              (rows[:6], rows[2:8], {}),
                              (k, k, dict(q_out=k)),                        # two outputs
                              (rows[:6], q, dict(k_pages=rows)),
                              (torch.as_strided(rows, (6, 4, 64), (128, 64, 1)), q, {})):  # its own rows
        with pytest.raises(ValueError, match="overlap|one memory"):
            check("out", out, like, **others)


# ---------------------------------------------------------------- refusals of the C entry points


def pages(pkg, **kw):
    f = dict(k=16, v=1 << 40, layers=1, pages=4, kv_heads=2, page_tokens=16, head_dim=64, dtype=0)
    f.update(kw)
    return pkg._native.Pages(**f)


def copy(pkg, src, dst, a, b):
    i32 = ctypes.c_int32 * max(1, len(a))
    return pkg.lib().oasis_pages_copy(src, dst, i32(*a), i32(*b), len(a), None)


@pytest.mark.parametrize("change,a,b,status", [
    ({}, [0, 1], [2, 2], 1),                # a destination twice
    ({}, [0, 1], [1, 2], 1),                # source and destination at once
    ({}, [0], [4], 1), ({}, [-1], [2], 1), ({}, [4], [2], 1),
    ({"pages": 5}, [0], [1], 1),            # the same pool, another size
    ({"k": 32}, [0], [1], 1),               # overlapping pools
    ({"kv_heads": 1}, [0], [1], 1), ({"dtype": 1}, [0], [1], 1), ({"dtype": 2}, [0], [1], 6),
    ({"v": (1 << 40) + 8}, [0], [1], 2), ({"k": None}, [0], [1], 1), ({"pages": 0}, [0], [1], 1),
    ({"pages": 1 << 28}, [0], [1], 6),
])
def test_pages_copy_refusals(pkg, change, a, b, status):
    assert copy(pkg, pages(pkg), pages(pkg, **change), a, b) == status
    assert b"oasis_pages_copy" in pkg.lib().oasis_last_error()


def test_pages_copy_of_nothing(pkg):
    assert copy(pkg, pages(pkg), pages(pkg), [], []) == 0


def rope_args(pkg, **kw):
    f = dict(q=16, k=16, v=None, q_out=16, k_out=16, q_token_stride=128, q_head_stride=64, k_token_stride=128,
             k_head_stride=64, v_token_stride=128, v_head_stride=64, q_out_token_stride=128,
             q_out_head_stride=64, k_out_token_stride=128, k_out_head_stride=64, tokens=4, heads=2,
             kv_heads=2, head_dim=64, dtype=0, norm=1, interleaved=1, eps=1e-6, q_weight=None, k_weight=None,
             positions=16, positions_64=0, freqs=16, axes=3, axis_dims=(16, 24, 24), slots=None)
    f.update(kw)
    return pkg._native.QkNormRope(**f)


@pytest.mark.parametrize("change,status", [
    ({"tokens": -1}, 1), ({"heads": 0}, 1), ({"dtype": 3}, 6), ({"head_dim": 80}, 6), ({"axes": 0}, 1),
    ({"axes": 5}, 1), ({"axis_dims": (16, 24, 25)}, 1), ({"axis_dims": (16, 24, 26)}, 1),
    ({"axis_dims": (16, 24, 0)}, 1), ({"interleaved": 0, "axis_dims": (16, 24, 16)}, 6),
    ({"norm": 0, "q_weight": 16}, 1), ({"q": None}, 1), ({"k_out": None}, 1), ({"positions": None}, 1),
    ({"freqs": None}, 1), ({"q": 24}, 2), ({"q_head_stride": 63}, 2), ({"k_out_token_stride": 4}, 2),
])
def test_qk_norm_rope_refusals(pkg, change, status):
    assert pkg.lib().oasis_qk_norm_rope(rope_args(pkg, **change), None) == status
    assert b"oasis_qk_norm_rope" in pkg.lib().oasis_last_error()


@pytest.mark.parametrize("page,change,status", [
    ({}, {"v": None}, 1), ({}, {"slots": None}, 1), ({"layers": 2}, {}, 1), ({"kv_heads": 1}, {}, 1),
    ({"head_dim": 128}, {}, 1), ({"dtype": 1}, {}, 1), ({"k": 8}, {}, 2), ({}, {"v": 24}, 2),
])
def test_qk_norm_rope_append_refusals(pkg, page, change, status):
    args = dict(v=16, k_out=None, slots=16)
    args.update(change)
    args["pages"] = ctypes.pointer(pages(pkg, **page))
    assert pkg.lib().oasis_qk_norm_rope(rope_args(pkg, **args), None) == status


def test_qk_norm_rope_append_refuses_one_pool_for_both(pkg):
    """Keys and values of a slot cannot lie in the same memory (4 pages of 2 heads x 16 x 64: 16384 bytes)."""
    for v, status in ((16, 1), (32, 1), (16 + 16384 - 16, 1)):
        args = dict(v=16, k_out=None, slots=16, pages=ctypes.pointer(pages(pkg, v=v)))
        assert pkg.lib().oasis_qk_norm_rope(rope_args(pkg, **args), None) == status
        assert b"overlap" in pkg.lib().oasis_last_error()


def test_no_tokens_launch_nothing(pkg):
    assert pkg.lib().oasis_qk_norm_rope(rope_args(pkg, tokens=0), None) == 0
    assert pkg.lib().oasis_attn_window(attn_args(pkg, tokens=0, batch=0), None) == 0


def attn_args(pkg, **kw):
    f = dict(q=16, out=16, lse=None, q_token_stride=128, q_head_stride=64, out_token_stride=128, out_head_stride=64,
             k=16, v=1 << 40, pages=4, kv_heads=2, page_tokens=16, head_dim=64, dtype=0, page_table=16,
             table_width=2, kv_len=16, cu_q=16, batch=1, tokens=4, heads=2, max_q=0, max_kv=0, window=0,
             sinks=0, frame_tokens=1, scale=0.125)
    f.update(kw)
    return pkg._native.AttnWindow(**f)


@pytest.mark.parametrize("change,status", [
    ({"heads": 3}, 1), ({"heads": 0}, 1), ({"batch": -1}, 1), ({"table_width": 0}, 1), ({"window": -1}, 1),
    ({"sinks": -1}, 1), ({"frame_tokens": 0}, 1), ({"head_dim": 96}, 6), ({"page_tokens": 24}, 6),
    ({"dtype": 2}, 6), ({"scale": 0.0}, 1), ({"scale": float("nan")}, 1), ({"scale": float("inf")}, 1),
    ({"batch": 65536}, 6), ({"table_width": 1 << 27}, 6), ({"cu_q": None}, 1), ({"q": None}, 1),
    ({"kv_len": None}, 1), ({"k": None}, 1), ({"v": 24}, 2), ({"out": 24}, 2), ({"q_head_stride": 68}, 2),
    ({"pages": 0}, 1), ({"pages": 1 << 28}, 6), ({"pages": 1 << 26, "kv_heads": 2}, 6),
    ({"tokens": 1 << 30, "heads": 4}, 6),
])
def test_attn_window_refusals(pkg, change, status):
    assert pkg.lib().oasis_attn_window(attn_args(pkg, **change), None) == status
    assert b"oasis_attn_window" in pkg.lib().oasis_last_error()


def test_paged_struct_layouts_match_header(pkg):
    """The ctypes mirrors have the C layouts."""
    n = pkg._native
    assert ctypes.sizeof(n.Pages) == 40
    assert (n.QkNormRope.tokens.offset, n.QkNormRope.q_weight.offset, n.QkNormRope.axis_dims.offset,
            n.QkNormRope.pages.offset, ctypes.sizeof(n.QkNormRope)) == (120, 152, 196, 216, 232)
    assert (n.AttnWindow.k.offset, n.AttnWindow.page_table.offset, n.AttnWindow.cu_q.offset,
            n.AttnWindow.scale.offset, ctypes.sizeof(n.AttnWindow)) == (56, 96, 120, 160, 168)
    # the packed forms that the functions send are the same layouts
    fields = list(range(1, len(n.AttnWindow._fields_)))
    raw = pkg.paged._ATTN.pack(*fields, 0.5)
    back = n.AttnWindow.from_buffer_copy(raw + bytes(4))
    assert [getattr(back, f[0]) for f in n.AttnWindow._fields_] == fields + [0.5]
    names = [f[0] for f in n.QkNormRope._fields_]
    want = {f: i + 1 for i, f in enumerate(names)}
    want.update(eps=0.25, axis_dims=[7, 8, 9, 10], pages=0)
    flat = [x for f in names for x in (want[f] if f == "axis_dims" else [want[f]])]
    back = n.QkNormRope.from_buffer_copy(pkg.paged._ROPE.pack(*flat))
    got = {f: getattr(back, f) for f in names}
    got.update(axis_dims=list(back.axis_dims), pages=0 if not back.pages else 1)
    assert got == want
