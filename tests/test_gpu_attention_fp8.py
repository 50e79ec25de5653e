"""Paged attention over the 8-bit pool against 64-bit attention over the
values that the pool stands for (bound: tests/_fp8_cases.py)."""
import numpy as np
import pytest
import torch

from tests import _fp8_cases as fc

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _wrapper(**kw):
    from nanosglang_amd.kernels import BatchPrefillWithPagedKVCacheWrapper
    return BatchPrefillWithPagedKVCacheWrapper(
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda"), "NHD", **kw)


def _case(seed, q_lens, kv_lens, Hq, Hkv, D, P, causal=True, scale=None):
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // P) for n in kv_lens) + 5
    pool = fc.pool(rng, pages, P, Hkv, D)
    tabs = fc.tables(rng, kv_lens, P, pages)
    ptr, idx, last = fc.csr(tabs, kv_lens, P)
    qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    q = fc.bf16(rng.standard_normal((int(qo[-1]), Hq, D)))
    return dict(q=q, pool=pool, tabs=tabs, qo=qo, ptr=ptr, idx=idx, last=last, q_lens=q_lens,
                kv_lens=kv_lens, dims=(Hq, Hkv, D, P), causal=causal, scale=scale)


def _want(c, pool=None):
    k, v = (pool or c["pool"])[3:]
    Hkv, D = k.shape[2:]
    spans = [(k[t].reshape(-1, Hkv, D)[:n], v[t].reshape(-1, Hkv, D)[:n])
             for t, n in zip(c["tabs"], c["kv_lens"])]
    return fc.attention(c["q"], spans, c["q_lens"], c["causal"], c["scale"])


def _plan(w, c):
    w.plan(c["qo"], c["ptr"], c["idx"], c["last"], *c["dims"], causal=c["causal"],
           sm_scale=c["scale"], kv_data_type=FP8)


def _run(c, out=None):
    w = _wrapper()
    _plan(w, c)
    kc, vc, sc = fc.on_gpu(*c["pool"][:3])
    q = torch.from_numpy(c["q"]).cuda().bfloat16()
    got = w.run(q, (kc, vc), out=out, kv_scale=sc)
    assert w.check_flags() == 0
    return got, w


SHAPES = [(14, 2, 64), (32, 8, 128), (16, 16, 64), (8, 1, 128), (4, 4, 128), (3, 1, 64),
          (48, 1, 64)]


@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
@pytest.mark.parametrize("P", [1, 2, 16, 64])
def test_short_steps(Hq, Hkv, D, P):
    """Decode and verify rows over contexts from one token on, page and step
    edges among them."""
    q_lens = [1, 1, 2, 5, 5, 9, 3, 1, 1]
    kv_lens = [1, 2, 2, 16, 63, 64, 65, 128, 333]
    c = _case(Hq + P, q_lens, kv_lens, Hq, Hkv, D, P)
    got, _ = _run(c)
    fc.check(got, *_want(c))


@pytest.mark.parametrize("Hq,Hkv,D,q,L,B", [(14, 2, 64, 1, 5000, 3), (32, 8, 128, 9, 2500, 5),
                                            (8, 1, 128, 1, 9000, 1), (14, 2, 64, 5, 1300, 40),
                                            (16, 16, 64, 2, 1777, 20)])
@pytest.mark.parametrize("P", [1, 16])
def test_long_contexts_split_and_merged(Hq, Hkv, D, q, L, B, P):
    rng = np.random.default_rng(L)
    kv = [int(x) for x in rng.integers(L // 2, L + 1, B)]
    c = _case(L + P, [q] * B, kv, Hq, Hkv, D, P)
    got, _ = _run(c)
    fc.check(got, *_want(c))


@pytest.mark.parametrize("Hq,Hkv,D,rows", [(32, 8, 128, 256), (32, 8, 128, 128), (14, 2, 64, 128)])
def test_prefill_tiles(Hq, Hkv, D, rows):
    """Enough query tokens for the prefill kernel's tiles, of both sizes."""
    if rows == 256:
        q_lens, kv_lens = [1024, 1000, 900], [1024, 1500, 900]
    elif D == 128:
        q_lens, kv_lens = [128] * 66, [128] * 60 + [350] * 6
    else:
        q_lens, kv_lens = [500] * 20 + [313], [500] * 19 + [777, 313]
    c = _case(rows + D, q_lens, kv_lens, Hq, Hkv, D, 16)
    got, w = _run(c)
    assert w.plan_info.row_tiles * 16 == rows
    fc.check(got, *_want(c))


@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 64), (32, 8, 128)])
def test_not_causal_and_own_scale(Hq, Hkv, D):
    c = _case(4, [3, 1, 70], [10, 400, 65], Hq, Hkv, D, 16, causal=False, scale=0.3)
    got, _ = _run(c)
    fc.check(got, *_want(c))


@pytest.mark.parametrize("q_lens,kv_lens", [([4, 2], [70, 200]), ([4, 1], [5000, 1]),
                                            ([700, 700, 700], [700, 800, 700])])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_rows_reach_only_who_sees_them(q_lens, kv_lens, what):
    """A row that stands for NaN at a request's third-last position: its last
    three queries are NaN, those before are as if it were any other row."""
    c = _case(11, q_lens, kv_lens, 32, 8, 128, 16)
    kc, vc, sc = (x.copy() for x in c["pool"][:3])
    for tab, n in zip(c["tabs"], kv_lens):
        if n < 3:
            continue
        page, at = tab[(n - 3) // 16], (n - 3) % 16
        (kc if what == "k" else vc)[page, at] = 0x7F if what == "k" else 0
        sc[page, :, 0 if what == "k" else 1, at] = 255
    c["pool"] = (kc, vc, sc, *fc.values(kc, vc, sc))
    got, _ = _run(c)
    k, v = c["pool"][3:]
    spans = []
    for t, n in zip(c["tabs"], kv_lens):
        kk, vv = (np.array(x[t].reshape(-1, 8, 128)[:n]) for x in (k, v))
        if n >= 3 and what == "k":      # the reference: NaN V instead of NaN K
            kk[n - 3] = 0
            vv[n - 3] = np.nan
        spans.append((kk, vv))
    want, bound = fc.attention(c["q"], spans, q_lens)
    fc.check(got, want, bound)
    t0 = 0
    for n, L in zip(q_lens, kv_lens):
        if L >= 3 and n > 3:
            assert not np.isnan(want[t0:t0 + n - 3]).any() and np.isnan(want[t0 + n - 3:t0 + n]).all()
        t0 += n


@pytest.mark.parametrize("Hq,Hkv,D,q_lens,kv_lens", [
    (14, 2, 64, [1, 5, 3], [300, 640, 70]), (32, 8, 128, [9, 9], [4000, 5001]),
    (8, 1, 128, [1], [9000]), (32, 8, 128, [1000, 900, 800], [1000, 1500, 800]),
    (14, 2, 64, [500] * 20, [500] * 20), (48, 1, 64, [1, 2], [700, 800])])
@pytest.mark.parametrize("slope", [14.0, -14.0])
def test_scores_that_leave_the_first_steps_maximum_far_behind(Hq, Hkv, D, q_lens, kv_lens, slope):
    """Scores that rise (or fall) by several hundred along a context: far past
    2^127 times the first step's probabilities."""
    from oracle import kv_fp8
    c = _case(16, q_lens, kv_lens, Hq, Hkv, D, 16)
    kc, vc, sc = (x.copy() for x in c["pool"][:3])
    rng = np.random.default_rng(0)
    for tab, n in zip(c["tabs"], kv_lens):
        codes, e = kv_fp8.quantise(fc.ramp(rng, n, Hkv, D, slope), False)
        for j in range(n):
            kc[tab[j // 16], j % 16] = codes[j]
            sc[tab[j // 16], :, 0, j % 16] = e[j]
    c["pool"] = (kc, vc, sc, *fc.values(kc, vc, sc))
    c["q"] = fc.bf16(np.abs(c["q"]) + 3)
    got, _ = _run(c)
    fc.check(got, *_want(c))


def test_rows_behind_the_last_token_are_not_read():
    """Slots past a request's length, on its own last page and on others, may
    hold anything: NaN codes and NaN scales change nothing."""
    c = _case(12, [5, 1, 300], [70, 33, 1000], 14, 2, 64, 16)
    got, _ = _run(c)
    kc, vc, sc = (x.copy() for x in c["pool"][:3])
    used = np.zeros(kc.shape[:2], bool)
    for t, n in zip(c["tabs"], c["kv_lens"]):
        for j in range(n):
            used[t[j // 16], j % 16] = True
    kc[~used], vc[~used] = 0x7F, 0x7F
    sc.transpose(0, 3, 1, 2)[~used] = 255
    c["pool"] = (kc, vc, sc)
    again, _ = _run(c)
    assert torch.equal(got, again)


def test_bad_page_ids_raise_the_flag_and_spare_the_others():
    c = _case(13, [1, 1, 1], [40, 90, 1], 14, 2, 64, 16)
    want, bound = _want(c)
    idx = c["idx"].copy()
    idx[c["ptr"][1]] = c["pool"][0].shape[0] + 7
    w = _wrapper()
    w.plan(c["qo"], c["ptr"], idx, c["last"], *c["dims"], kv_data_type=FP8)
    kc, vc, sc = fc.on_gpu(*c["pool"][:3])
    got = w.run(torch.from_numpy(c["q"]).cuda().bfloat16(), (kc, vc), kv_scale=sc)
    assert w.check_flags() == 1 and w.check_flags() == 0
    ok = [0, 2]
    fc.check(got[ok], want[ok], bound[ok])


def test_out_argument_and_rows_of_nobody():
    """A given output; a request without query tokens between others."""
    c = _case(14, [2, 0, 3], [50, 20, 70], 32, 8, 128, 16)
    out = torch.full((5, 32, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    got, _ = _run(c, out=out)
    assert got is out
    fc.check(out, *_want(c))


@pytest.mark.parametrize("max_kv_len", [0, 1500])
def test_graph_plans_replay_over_growing_contexts(max_kv_len):
    """Graph mode: one captured run, re-planned for longer contexts, each
    replay against the 64-bit reference."""
    from nanosglang_amd.kernels import BatchPrefillWithPagedKVCacheWrapper
    Hq, Hkv, D, P, B, q = 14, 2, 64, 16, 6, 5
    rng = np.random.default_rng(3)
    pages = 700
    pool = fc.pool(rng, pages, P, Hkv, D)
    kc, vc, sc = fc.on_gpu(*pool[:3])
    i32 = dict(dtype=torch.int32, device="cuda")
    w = BatchPrefillWithPagedKVCacheWrapper(
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda"), "NHD", use_cuda_graph=True,
        qo_indptr_buf=torch.zeros(B + 1, **i32), paged_kv_indptr_buf=torch.zeros(B + 1, **i32),
        paged_kv_indices_buf=torch.zeros(600, **i32),
        paged_kv_last_page_len_buf=torch.zeros(B, **i32), max_q_len=q, max_kv_len=max_kv_len)
    qd = torch.zeros(B * q, Hq, D, device="cuda", dtype=torch.bfloat16)
    graph = out = None
    for step, base in enumerate([7, 300, 1400]):
        kv = [base + 13 * b for b in range(B)]
        tabs = fc.tables(rng, kv, P, pages)
        ptr, idx, last = fc.csr(tabs, kv, P)
        qo = np.arange(B + 1, dtype=np.int32) * q
        w.plan(qo, ptr, idx, last, Hq, Hkv, D, P, kv_data_type=FP8)
        x = fc.bf16(rng.standard_normal((B * q, Hq, D)))
        qd.copy_(torch.from_numpy(x))
        if graph is None:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                w.run(qd, (kc, vc), kv_scale=sc)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = w.run(qd, (kc, vc), kv_scale=sc)
        graph.replay()
        torch.cuda.synchronize()
        spans = [tuple(y[t].reshape(-1, Hkv, D)[:n] for y in pool[3:]) for t, n in zip(tabs, kv)]
        fc.check(out, *fc.attention(x, spans, [q] * B))


def test_agrees_with_the_bf16_pool_of_the_same_values():
    """The bf16 kernels over a bf16 pool of the same values: both within their
    bound of the same reference."""
    for q_lens, kv_lens in (([1024, 1000], [1024, 1800]), ([5, 9, 1], [300, 2000, 64])):
        c = _case(15, q_lens, kv_lens, 32, 8, 128, 16)
        want, bound = _want(c)
        fc.check(_run(c)[0], want, bound)
        k, v = (torch.from_numpy(x).cuda().bfloat16() for x in c["pool"][3:])
        w = _wrapper()
        w.plan(c["qo"], c["ptr"], c["idx"], c["last"], *c["dims"])
        fc.check(w.run(torch.from_numpy(c["q"]).cuda().bfloat16(), (k, v)), want, bound)
