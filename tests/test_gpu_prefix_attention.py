"""Shared-prefix attention against 64-bit attention over each request's joined
context (bound: tests/_fp8_cases.py), bf16 and 8-bit pools."""
import numpy as np
import pytest
import torch

from tests import _fp8_cases as fc

pytestmark = pytest.mark.gpu
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def _pool(rng, fp8, pages, P, Hkv, D):
    """(device caches, kv_scale, k values, v values)."""
    if fp8:
        p = fc.pool(rng, pages, P, Hkv, D)
        kc, vc, sc = fc.on_gpu(*p[:3])
        return (kc, vc), sc, p[3], p[4]
    k, v = (fc.rows(rng, pages, P, Hkv, D) for _ in range(2))
    return tuple(torch.from_numpy(x).cuda().bfloat16() for x in (k, v)), None, k, v


def _tables(rng, c, P, pages):
    perm = rng.permutation(pages)
    at = 0
    out = []
    for lens in (c["prefix"], c["kv"]):
        tabs = []
        for n in lens:
            m = -(-n // P)
            tabs.append([int(x) for x in perm[at:at + m]])
            at += m
        out.append(tabs)
    return out


def _spans(c, ptabs, tabs, k, v):
    Hkv, D = k.shape[2:]

    def rows(x, t, n):
        return x[t].reshape(-1, Hkv, D)[:n] if n else np.zeros((0, Hkv, D))
    spans = []
    for b, (t, n) in enumerate(zip(tabs, c["kv"])):
        g = int(np.searchsorted(c["groups"], b, side="right") - 1)
        spans.append(tuple(np.concatenate([rows(x, ptabs[g], c["prefix"][g]), rows(x, t, n)])
                           for x in (k, v)))
    return spans


def _want(q, c, ptabs, tabs, k, v, causal=True, scale=None):
    # bottom-right causal over the joined context is the own part's rule
    return fc.attention(q, _spans(c, ptabs, tabs, k, v), c["q"], causal, scale)


def _plan(w, c, ptabs, tabs, heads, P, fp8, **kw):
    qo = np.concatenate([[0], np.cumsum(c["q"])]).astype(np.int32)
    w.plan(qo, c["groups"], *fc.csr(ptabs, c["prefix"], P), *fc.csr(tabs, c["kv"], P), *heads, P,
           kv_data_type=FP8 if fp8 else BF16, **kw)


def _wrapper(mb=192, **kw):
    from nanosglang_amd.kernels import SharedPrefixAttentionWrapper
    return SharedPrefixAttentionWrapper(torch.empty(mb << 20, dtype=torch.uint8, device="cuda"),
                                        **kw)


def _case(seed, c, heads, P, fp8, **kw):
    rng = np.random.default_rng(seed)
    Hq, Hkv, D = heads
    pages = sum(-(-n // P) for n in c["prefix"] + c["kv"]) + 3
    caches, sc, k, v = _pool(rng, fp8, pages, P, Hkv, D)
    ptabs, tabs = _tables(rng, c, P, pages)
    q = fc.bf16(rng.standard_normal((sum(c["q"]), Hq, D)))
    w = _wrapper()
    _plan(w, c, ptabs, tabs, heads, P, fp8, **kw)
    got = w.run(torch.from_numpy(q).cuda().bfloat16(), caches, kv_scale=sc)
    assert w.check_flags() == 0
    fc.check(got, *_want(q, c, ptabs, tabs, k, v, kw.get("causal", True), kw.get("sm_scale")))
    return w


HEADS = [(14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (48, 1, 64)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("P", [1, 16, 64])
def test_groups_of_all_kinds(heads, P, fp8):
    """Prefixes of none, one and many tokens, groups of one and several
    requests, requests without queries, own parts from one token on."""
    c = dict(q=[1, 5, 0, 2, 1, 9, 3, 1], kv=[1, 5, 4, 70, 300, 9, 65, 16],
             groups=[0, 2, 3, 6, 7, 8], prefix=[333, 20, 0, 1, 64])
    _case(heads[0] + P, c, heads, P, fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,n,q,prefix,P,rows", [
    ((32, 8, 128), 3, 1, 2500, 16, 16),      # one launch with the own parts: 12 rows
    ((32, 8, 128), 13, 1, 1999, 16, 64),     # ... 52
    ((14, 2, 64), 3, 5, 1111, 16, 64),       # ... 105: two tiles of 64
    ((48, 1, 64), 1, 1, 999, 16, 48),        # ... own tiles taller than 16 rows
    ((32, 8, 128), 3, 1, 2500, 8, 16),       # small pages: one KV group
    ((32, 8, 128), 13, 1, 1999, 8, 64),
    ((14, 2, 64), 3, 5, 1111, 8, 64),
    ((32, 8, 128), 25, 1, 1500, 8, 64),
    ((32, 8, 128), 30, 9, 1500, 16, 64),     # 1080 rows, tiles of one KV group
    ((14, 2, 64), 33, 5, 700, 8, 64),
    ((14, 2, 64), 33, 5, 9000, 8, 128),      # launches of their own: 1155 rows, 128-row tiles
    ((32, 8, 128), 28, 1, 9000, 1, 128),     # ... 112 rows
    ((32, 8, 128), 30, 9, 5000, 16, 256),    # 1080 rows: 256-row tiles, the last partly filled
])
def test_tile_shapes(heads, n, q, prefix, P, rows, fp8):
    rng = np.random.default_rng(n)
    c = dict(q=[q] * n, kv=[int(q + x) for x in rng.integers(0, 150, n)], groups=[0, n],
             prefix=[prefix])
    pl = _case(n, c, heads, P, fp8).plan_info
    assert pl.prefix_rows == rows
    assert pl.one_launch == (rows <= 64)


@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_long_own_parts_and_a_long_prefix(fp8):
    _case(1, dict(q=[700, 800, 900], kv=[700, 1000, 900], groups=[0, 3], prefix=[200]),
          (32, 8, 128), 16, fp8)
    _case(2, dict(q=[1, 2], kv=[3000, 4000], groups=[0, 1, 2], prefix=[9000, 17]), (14, 2, 64), 16,
          fp8)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads,n,q", [((14, 2, 64), 3, 1), ((14, 2, 64), 33, 5),
                                       ((32, 8, 128), 3, 1), ((32, 8, 128), 25, 1),
                                       ((32, 8, 128), 30, 9)])
def test_scores_that_leave_the_first_steps_maximum_far_behind(heads, n, q, fp8):
    """Scores that rise by several hundred along the prefix, past 2^127 times
    its first step's probabilities, and fall along the own parts."""
    from oracle import kv_fp8
    Hq, Hkv, D = heads
    rng = np.random.default_rng(9)
    P, pages = 16, 900
    c = dict(q=[q] * n, kv=[int(q + x) for x in rng.integers(0, 200, n)], groups=[0, n],
             prefix=[1500])
    ptabs, tabs = _tables(rng, c, P, pages)
    k, v = (fc.rows(rng, pages, P, Hkv, D) for _ in range(2))
    for tab, m, slope in [(ptabs[0], 1500, 14.0)] + [(t, m, -9.0) for t, m in zip(tabs, c["kv"])]:
        r = fc.ramp(rng, m, Hkv, D, slope)
        for j in range(m):
            k[tab[j // P], j % P] = r[j]
    if fp8:
        (kc, ke), (vc, ve) = kv_fp8.quantise(k, False), kv_fp8.quantise(v, True)
        scale = np.ascontiguousarray(np.stack([ke, ve], 2).transpose(0, 3, 2, 1))
        k, v = fc.values(kc, vc, scale)
        *caches, sc = fc.on_gpu(kc, vc, scale)
    else:
        caches, sc = [torch.from_numpy(x).cuda().bfloat16() for x in (k, v)], None
    x = fc.bf16(np.abs(rng.standard_normal((n * q, Hq, D))) + 3)
    w = _wrapper()
    _plan(w, c, ptabs, tabs, heads, P, fp8)
    got = w.run(torch.from_numpy(x).cuda().bfloat16(), caches, kv_scale=sc)
    fc.check(got, *_want(x, c, ptabs, tabs, k, v))


def test_not_causal_and_own_scale():
    _case(3, dict(q=[5, 3], kv=[2, 100], groups=[0, 2], prefix=[50]), (14, 2, 64), 16, False,
          causal=False, sm_scale=0.4)


@pytest.mark.parametrize("fp8", [False, True])
def test_agrees_with_the_per_request_wrapper(fp8):
    """The same contexts through BatchPrefillWithPagedKVCacheWrapper over joined
    page tables (whole prefix pages): both within their bounds of the same
    reference, so within their sum of each other."""
    from nanosglang_amd.kernels import BatchPrefillWithPagedKVCacheWrapper
    rng = np.random.default_rng(5)
    heads, P = (32, 8, 128), 16
    c = dict(q=[5] * 6, kv=[40 + 7 * i for i in range(6)], groups=[0, 4, 6], prefix=[640, 320])
    caches, sc, k, v = _pool(rng, fp8, 150, P, 8, 128)
    ptabs, tabs = _tables(rng, c, P, 150)
    q = fc.bf16(rng.standard_normal((30, 32, 128)))
    qd = torch.from_numpy(q).cuda().bfloat16()
    w = _wrapper()
    _plan(w, c, ptabs, tabs, heads, P, fp8)
    got = w.run(qd, caches, kv_scale=sc)
    joined = [ptabs[0 if b < 4 else 1] + t for b, t in enumerate(tabs)]
    lens = [n + (640 if b < 4 else 320) for b, n in enumerate(c["kv"])]
    w2 = BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8,
                                                         device="cuda"))
    w2.plan(np.arange(0, 31, 5, dtype=np.int32), *fc.csr(joined, lens, P), *heads, P,
            kv_data_type=FP8 if fp8 else BF16)
    per = w2.run(qd, caches, kv_scale=sc)
    want, bound = _want(q, c, ptabs, tabs, k, v)
    fc.check(got, want, bound)
    fc.check(per, want, bound)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("max_kv_len,Hq", [(0, 14), (800, 14), (800, 4), (0, 28), (800, 28)])
def test_graph_mode_replays_after_each_plan(fp8, max_kv_len, Hq):
    """One captured run; requests grow, leave and change groups between the
    replays; rows past the plan's stay as they were."""
    rng = np.random.default_rng(6)
    heads, P, B, mq = (Hq, 2, 64), 16, 8, 5
    pages = 500
    caches, sc, k, v = _pool(rng, fp8, pages, P, 2, 64)
    w = _wrapper(use_cuda_graph=True, max_batch=B, max_q_len=mq, max_groups=3,
                 max_prefix_pages=100, max_pages=420, max_kv_len=max_kv_len)
    qd = torch.zeros(B * mq, Hq, 64, device="cuda", dtype=BF16)
    out = torch.zeros_like(qd)
    graph = None
    for c in (dict(q=[5] * 8, kv=[5 + i for i in range(8)], groups=[0, 8], prefix=[1600]),
              dict(q=[5] * 8, kv=[300 + 60 * i for i in range(8)], groups=[0, 3, 8],
                   prefix=[777, 1000]),
              dict(q=[1, 5, 2], kv=[9, 790, 31], groups=[0, 1, 2, 3], prefix=[0, 64, 15])):
        ptabs, tabs = _tables(rng, c, P, pages)
        _plan(w, c, ptabs, tabs, heads, P, fp8)
        n = sum(c["q"])
        q = fc.bf16(rng.standard_normal((B * mq, Hq, 64)))
        qd.copy_(torch.from_numpy(q))
        if graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                w.run(qd, caches, out=out, kv_scale=sc)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                w.run(qd, caches, out=out, kv_scale=sc)
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert w.check_flags() == 0
        assert w.plan_info.one_launch == (Hq < 28)           # up to 512 rows
        assert (w.plan_info.own.kv_groups > 1) == (max_kv_len > 0)
        fc.check(out[:n], *_want(q[:n], c, ptabs, tabs, k, v))
        assert (out[n:] == 9.0).all()


def test_a_run_on_another_stream_outlives_the_next_plan():
    """The plan's arrays go back to the allocator when the wrapper plans again,
    but not while another stream's run may still read them."""
    rng = np.random.default_rng(8)
    heads, P = (14, 2, 64), 16
    caches, sc, k, v = _pool(rng, True, 300, P, 2, 64)
    w = _wrapper()
    c = dict(q=[2] * 8, kv=[20] * 8, groups=[0, 8], prefix=[2000])
    ptabs, tabs = _tables(rng, c, P, 300)
    q = fc.bf16(rng.standard_normal((16, 14, 64)))
    qd = torch.from_numpy(q).cuda().bfloat16()
    side = torch.cuda.Stream()
    want = _want(q, c, ptabs, tabs, k, v)
    for _ in range(3):
        _plan(w, c, ptabs, tabs, heads, P, True)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)                # about 10 ms before the run starts
            out = w.run(qd, caches, kv_scale=sc)
        c2 = dict(q=[1], kv=[7], groups=[0, 1], prefix=[100])
        _plan(w, c2, *_tables(rng, c2, P, 300), heads, P, True)
        junk = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (64, 200, 500, 1000) * 8]
        torch.cuda.synchronize()
        del junk
        fc.check(out, *want)


def test_a_captured_run_keeps_its_plan():
    """Without graph mode: a later plan leaves the captured graph's arrays
    alone, and a wrapper plans and runs on."""
    rng = np.random.default_rng(7)
    heads, P = (32, 8, 128), 16
    caches, sc, k, v = _pool(rng, False, 200, P, 8, 128)
    w = _wrapper()
    c = dict(q=[1] * 4, kv=[30, 40, 50, 60], groups=[0, 4], prefix=[1000])
    ptabs, tabs = _tables(rng, c, P, 200)
    _plan(w, c, ptabs, tabs, heads, P, False)
    q = fc.bf16(rng.standard_normal((4, 32, 128)))
    qd = torch.from_numpy(q).cuda().bfloat16()
    w.run(qd, caches)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = w.run(qd, caches)
    want = _want(q, c, ptabs, tabs, k, v)
    for _ in range(3):
        c2 = dict(q=[1] * 2, kv=[7, 8], groups=[0, 2], prefix=[100])
        p2, t2 = _tables(rng, c2, P, 200)
        _plan(w, c2, p2, t2, heads, P, False)
        q2 = fc.bf16(rng.standard_normal((2, 32, 128)))
        got = w.run(torch.from_numpy(q2).cuda().bfloat16(), caches)
        fc.check(got, *_want(q2, c2, p2, t2, k, v))
        junk = [torch.full((1000,), -1, dtype=torch.int32, device="cuda") for _ in range(20)]
        graph.replay()
        torch.cuda.synchronize()
        del junk
        fc.check(out, *want)


@pytest.mark.parametrize("fp8", [False, True])
def test_bad_page_ids_raise_the_flag(fp8):
    rng = np.random.default_rng(8)
    heads, P = (14, 2, 64), 16
    caches, sc, *_ = _pool(rng, fp8, 60, P, 2, 64)
    c = dict(q=[1, 1], kv=[30, 40], groups=[0, 2], prefix=[500])
    for bad in ("prefix", "own"):
        ptabs, tabs = _tables(rng, c, P, 60)
        (ptabs[0] if bad == "prefix" else tabs[1])[1] = 60
        w = _wrapper()
        _plan(w, c, ptabs, tabs, heads, P, fp8)
        w.run(torch.zeros(2, 14, 64, device="cuda", dtype=BF16), caches, kv_scale=sc)
        assert w.check_flags() == 1 and w.check_flags() == 0


def test_refusals():
    w = _wrapper(1)
    c = dict(q=[1], kv=[30], groups=[0, 1], prefix=[50])
    caches, _, *_ = _pool(np.random.default_rng(0), False, 60, 16, 2, 64)
    q = torch.zeros(1, 14, 64, device="cuda", dtype=BF16)
    with pytest.raises(RuntimeError, match="before plan"):
        w.run(q, caches)
    ptabs, tabs = [[1, 2, 3, 4]], [[5, 6]]
    _plan(w, c, ptabs, tabs, (14, 2, 64), 16, False)
    with pytest.raises(ValueError, match="kv_scale is for"):
        w.run(q, caches, kv_scale=q)
    with pytest.raises(ValueError, match="q shape"):
        w.run(q.expand(2, 14, 64).contiguous(), caches)
    with pytest.raises(ValueError, match="out must"):
        w.run(q, caches, out=torch.zeros(1, 14, 64, device="cuda"))
    with pytest.raises(ValueError, match="disagree"):
        w.plan([0, 1], [0, 1], [0, 4], [1, 2, 3, 4], [2, 3], [0, 2], [5, 6], [14], 14, 2, 64, 16)
    with pytest.raises(ValueError, match="page ids"):
        w.plan([0, 1], [0, 1], [0, 4], [1, 2, 3], [2], [0, 2], [5, 6], [14], 14, 2, 64, 16)
    with pytest.raises(RuntimeError, match="workspace too small"):
        c = dict(q=[9] * 40, kv=[30] * 40, groups=[0, 40], prefix=[500])
        rng = np.random.default_rng(1)
        _plan(w, c, *_tables(rng, c, 16, 200), (32, 8, 128), 16, False)
