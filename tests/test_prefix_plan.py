"""The shared-prefix planner without a GPU: every query row meets every token
of its prefix and of its own context exactly once, merge items point at the
items that hold a row's partials, fixed plans keep one grid, bad input is
refused."""
import ctypes as C

import numpy as np
import pytest

from nanosglang_amd._native import NSG_ATTN_WORK_INTS, PrefixAttnPlan


def _arrays(q_lens, kv_lens, groups, prefix_lens, P):
    def csr(lens):
        n = [-(-x // P) for x in lens]
        return (np.concatenate([[0], np.cumsum(n)]).astype(np.int32),
                np.asarray([(x - 1) % P + 1 if x else 0 for x in lens], np.int32))
    qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    return (qo, np.asarray(groups, np.int32), *csr(prefix_lens), *csr(kv_lens))


def _plan(lib, q_lens, kv_lens, groups, prefix_lens, Hq=32, Hkv=8, D=128, P=16, causal=1, cus=256,
          cap=20000, fixed=None):
    qo, g, pptr, plast, ptr, last = _arrays(q_lens, kv_lens, groups, prefix_lens, P)
    work = np.full(cap * NSG_ATTN_WORK_INTS, 77, np.int32)
    pl = PrefixAttnPlan()
    args = (qo.ctypes.data, g.ctypes.data, len(g) - 1, pptr.ctypes.data, plast.ctypes.data,
            ptr.ctypes.data, last.ctypes.data, len(q_lens), Hq, Hkv, D, P, causal, cus)
    if fixed is None:
        rc = lib.nsg_prefix_attn_plan(*args, work.ctypes.data, cap, C.byref(pl))
    else:
        rc = lib.nsg_prefix_attn_plan_fixed(*args, *fixed, work.ctypes.data, cap, C.byref(pl))
    w = work.reshape(-1, NSG_ATTN_WORK_INTS)
    a, b = pl.own.num_work, pl.own.num_work + pl.num_prefix_work
    n = pl.num_prefix_work
    own, pre = (w[n:b], w[:n]) if pl.one_launch else (w[:a], w[a:b])
    return rc, pl, (own, pre, w[b:b + pl.num_merge]), (qo, pptr, ptr)


def _check(pl, items, arrays, q_lens, kv_lens, groups, prefix_lens, G, P, causal=True):
    own, pre, merge = items
    qo, pptr, ptr = arrays
    T, TP = pl.own.q_tile_tokens, pl.prefix_tile_tokens
    seen = np.zeros(qo[-1], int)
    for qs, qn, wi0, ns, pw0, pns, g0, tiles in merge:
        if qn == 0:
            continue
        b = int(np.searchsorted(qo, qs, side="right") - 1)
        while qo[b + 1] == qs:
            b += 1
        g = int(np.searchsorted(groups, b, side="right") - 1)
        seen[qs:qs + qn] += 1
        if pl.one_launch:                             # partials: the prefix items' first
            wi0 -= pl.num_prefix_work
        assert qs + qn <= qo[b + 1] and qn <= T and g0 == qo[groups[g]]
        L = kv_lens[b]
        end = L - q_lens[b] + (qs - qo[b]) + qn if causal else L
        rng = []
        for w in own[wi0:wi0 + ns]:
            assert (w[0], w[1], w[3]) == (qs, qn, ptr[b] + pptr[-1]) and w[6] >= 2
            assert w[2] == (L - q_lens[b] + qs - qo[b] if causal else L - 1)
            rng.append((w[4], w[5]))
        assert rng[0][0] == 0 and rng[-1][1] == end
        assert all(x[1] == y[0] for x, y in zip(rng, rng[1:]))
        assert pns > 0 or prefix_lens[g] == 0
        for t in range(qs, qs + qn):                  # where the merge looks each token up
            tile, row = divmod(t - g0, TP)
            assert tile < tiles == -(-(qo[groups[g + 1]] - g0) // TP)
            its = [pre[pw0 + tile + s * tiles] for s in range(pns)]
            assert all(w[0] == g0 + tile * TP and row < w[1] and w[3] == pptr[g] for w in its)
            assert all(w[2] >= 1 << 29 and w[6] >= 2 for w in its)
            if pns:
                assert its[0][4] == 0 and its[-1][5] == prefix_lens[g]
                assert all(x[5] == y[4] for x, y in zip(its, its[1:]))
                assert all((w[5] - 1) // P - w[4] // P + 1 <= 1024 and w[4] < w[5] for w in its)
    assert (seen == 1).all()
    assert TP * G <= pl.prefix_rows or TP == 1


@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (48, 1, 64), (8, 1, 128)])
@pytest.mark.parametrize("P", [1, 16, 64])
@pytest.mark.parametrize("cus", [2, 256])
def test_every_row_meets_every_token_once(lib, Hq, Hkv, D, P, cus):
    rng = np.random.default_rng(Hq + P)
    q_lens = [5, 5, 0, 1, 9, 1, 1, 3, 40, 5]
    kv_lens = [int(q + rng.integers(1, 400)) for q in q_lens]
    for groups, pre in (([0, 10], [5000]), ([0, 2, 3, 8, 10], [300, 70, 0, 1]),
                        ([0, 0, 10, 10], [9, 2222, 0])):
        rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, groups, pre, Hq, Hkv, D, P, cus=cus)
        assert rc == 0, lib.nsg_last_error()
        _check(pl, items, arrays, q_lens, kv_lens, groups, pre, Hq // Hkv, P)
        rows = 4 * Hkv * (D + 4)
        assert pl.own_rows >= pl.own.row_tiles * 16
        assert not pl.one_launch or pl.own_rows == pl.prefix_rows
        assert pl.workspace_bytes >= 256 + rows * (pl.own.num_work * pl.own_rows
                                                   + pl.num_prefix_work * pl.prefix_rows)


def test_short_shares_for_the_cus_that_even_ones_leave_idle(lib):
    """64 x 9 rows of 4 queries a KV head are 9 tiles of 256: 8 heads x 9 x 3 long
    shares, and a short one of each tile for the 40 CUs left, two apiece."""
    q_lens, kv_lens, groups, prefix = [9] * 64, [200] * 64, [0, 64], [8192]
    rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, groups, prefix)
    assert rc == 0 and (pl.prefix_rows, pl.one_launch, pl.num_prefix_work) == (256, 0, 36)
    _check(pl, items, arrays, q_lens, kv_lens, groups, prefix, 4, 16)
    steps = (items[1][:, 5] - items[1][:, 4]) // 64
    assert (steps[27:] * 2 < steps[:27].min()).all() and steps[:27].max() < 43
    # 8 tiles a head: four even shares for every CU
    rc, pl, items, arrays = _plan(lib, [8] * 64, kv_lens, groups, prefix)
    assert rc == 0 and pl.num_prefix_work == 32
    assert (items[1][:, 5] - items[1][:, 4] == 2048).all()


@pytest.mark.parametrize("n,q,prefix,P,one_launch,kv_groups,rows", [
    (3, 1, 2500, 16, 1, 2, 16), (32, 1, 4001, 16, 1, 2, 64),   # few tiles: KV groups
    (128, 1, 400, 16, 1, 1, 64), (32, 5, 500, 16, 1, 1, 64),   # many, a short prefix
    (128, 1, 20000, 16, 0, 1, 256), (30, 9, 5000, 16, 0, 1, 256), (28, 1, 9000, 1, 0, 1, 128),
    (3, 1, 2500, 8, 1, 1, 16),                                 # pages of less than 16 tokens
    (64, 9, 0, 16, 0, 1, 256),                                 # no prefix
])
def test_which_launches(lib, n, q, prefix, P, one_launch, kv_groups, rows):
    q_lens, kv_lens = [q] * n, [q + 100] * n
    rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, [0, n], [prefix], P=P)
    assert rc == 0
    assert (pl.one_launch, pl.own.kv_groups, pl.prefix_rows) == (one_launch, kv_groups, rows)
    _check(pl, items, arrays, q_lens, kv_lens, [0, n], [prefix], 4, P)


def test_prompts_and_not_causal(lib):
    q_lens, kv_lens = [1000, 900, 1100], [1000, 1900, 1100]
    rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, [0, 3], [700])
    assert rc == 0 and pl.own.row_tiles >= 8        # the prefill kernel's tiles
    _check(pl, items, arrays, q_lens, kv_lens, [0, 3], [700], 4, 16)
    q_lens, kv_lens = [5, 9], [3, 70]               # more queries than own tokens: not causal
    rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, [0, 2], [100], causal=0)
    assert rc == 0
    _check(pl, items, arrays, q_lens, kv_lens, [0, 2], [100], 4, 16, causal=False)


@pytest.mark.parametrize("Hq,Hkv,D,P", [(32, 8, 128, 16), (14, 2, 64, 16), (14, 2, 64, 1)])
@pytest.mark.parametrize("max_kv", [0, 900])
@pytest.mark.parametrize("small", [False, True])
def test_fixed_plans_keep_one_grid(lib, Hq, Hkv, D, P, max_kv, small):
    B, mq, mg, pages = 12, 5, 3, -(-6000 // P)
    if small:
        B, mq = 12, 1
    c = [C.c_int32(0) for _ in range(3)]
    assert lib.nsg_prefix_attn_fixed_capacity(B, mq, mg, Hq, Hkv, D, 256, max_kv, pages, P,
                                              *map(C.byref, c)) == 0
    fixed = (B, mq, max_kv, *(x.value for x in c))
    rng = np.random.default_rng(1)
    shapes = set()
    for n, groups, pre in ((12, [0, 12], [6000]), (12, [0, 1, 7, 12], [6000, 6000, 5999]),
                           (1, [0, 1], [0]), (7, [0, 3, 7], [17, 3000])):
        q_lens = [int(x) for x in rng.integers(1, mq + 1, n)]
        kv_lens = [int(q + rng.integers(0, 890)) for q in q_lens]
        rc, pl, items, arrays = _plan(lib, q_lens, kv_lens, groups, pre, Hq, Hkv, D, P,
                                      fixed=fixed)
        assert rc == 0, lib.nsg_last_error()
        _check(pl, items, arrays, q_lens, kv_lens, groups, pre, Hq // Hkv, P)
        shapes.add((pl.own.num_work, pl.num_prefix_work, pl.num_merge, pl.own.row_tiles,
                    pl.own.kv_groups, pl.prefix_rows, pl.prefix_tile_tokens, pl.prefix_partials,
                    pl.workspace_bytes))
        for part in items:                             # the unused tail is empty
            used = np.flatnonzero(part[:, 1])
            assert not part[used[-1] + 1 if len(used) else 0:].any()
    assert len(shapes) == 1
    assert pl.one_launch == (B * mq * Hq // Hkv <= 512)
    rc, *_ = _plan(lib, [1] * 13, [5] * 13, [0, 13], [10], Hq, Hkv, D, P, fixed=fixed)
    assert rc == 1 and b"exceeds" in lib.nsg_last_error()


def test_refusals(lib):
    def err(*a, **kw):
        rc, pl, *_ = _plan(lib, *a, **kw)
        return rc, lib.nsg_last_error().decode(), pl
    ok = ([1, 1], [5, 6], [0, 2], [40])
    assert err(*ok)[0] == 0
    assert "group_indptr" in err([1, 1], [5, 6], [0, 1], [40])[1]
    assert "group_indptr" in err([1, 1], [5, 6], [1, 2], [40])[1]
    assert "decreasing" in err([1, 1], [5, 6], [0, 2, 1, 2], [40, 1, 1])[1]
    assert "decreasing" in err([1, 1], [5, 6], [0, 50, 2], [40, 1])[1]
    assert "empty KV" in err([1, 1], [5, 0], [0, 2], [40])[1]
    assert "query length" in err([1, 9], [5, 6], [0, 2], [40])[1]
    assert err(*ok, D=96)[0] == 2 and err(*ok, Hq=9)[0] == 1
    assert "power of two" in err(*ok, P=12)[1]
    rc, msg, pl = err(*ok, cap=2)
    assert rc == 3 and pl.own.num_work + pl.num_prefix_work + pl.num_merge > 2
    # bad last-page lengths, a null argument
    qo, g, pptr, plast, ptr, last = _arrays(*ok, 16)
    plast[0] = 17
    p = PrefixAttnPlan()
    w = np.zeros(800, np.int32)
    a = [qo.ctypes.data, g.ctypes.data, 1, pptr.ctypes.data, plast.ctypes.data, ptr.ctypes.data,
         last.ctypes.data, 2, 32, 8, 128, 16, 1, 256, w.ctypes.data, 100]
    assert lib.nsg_prefix_attn_plan(*a, C.byref(p)) == 1 and b"last_page" in lib.nsg_last_error()
    a[4] = None
    assert lib.nsg_prefix_attn_plan(*a, C.byref(p)) == 1


OK = 0x1000


@pytest.mark.parametrize("change,rc,match", [
    (dict(q=None), 1, "null"), (dict(idx=None), 1, "null"), (dict(page=5), 1, "page_size"),
    (dict(page=8), 1, "KV groups"), (dict(num_pages=0), 1, "num_pages"), (dict(sm=-1.0), 1, "sm"),
    (dict(out=OK + 8), 1, "aligned"), (dict(ws=100), 3, "workspace")])
def test_run_refuses(lib, change, rc, match):
    r, pl, *_ = _plan(lib, [1, 1], [5, 6], [0, 2], [40])
    assert r == 0 and pl.own.kv_groups > 1
    a = dict(q=OK, out=OK, idx=OK, page=16, num_pages=9, sm=0.1, ws=pl.workspace_bytes)
    a.update(change)
    got = lib.nsg_prefix_attn_run(C.byref(pl), OK, a["q"], OK, OK, None, a["out"], a["idx"],
                                  a["page"], a["num_pages"], a["sm"], 1, OK, a["ws"], None)
    assert got == rc and match in lib.nsg_last_error().decode()
