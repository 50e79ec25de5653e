"""Writes into and reads from the 8-bit KV pool against the 64-bit definition.

Codes and scale bytes are whole numbers and have to be equal; so are the
values read back, which bf16 holds exactly."""
import numpy as np
import pytest
import torch

from oracle import kv_fp8
from tests import _fp8_cases as fc

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _kernels():
    from nanosglang_amd import kernels
    return kernels


def _empty_pool(pages, P, Hkv, D, fill=0x55):
    kc = torch.full((pages, P, Hkv, D), fill, dtype=torch.uint8, device="cuda")
    return kc.view(FP8), kc.clone().view(FP8), torch.full((pages, Hkv, 2, P), fill,
                                                          dtype=torch.uint8, device="cuda")


def _expected(k, v, slots, pages, P, Hkv, D, fill=0x55):
    kc = np.full((pages * P, Hkv, D), fill, np.uint8)
    vc = kc.copy()
    sc = np.full((pages, Hkv, 2, P), fill, np.uint8)
    for x, pool, which in ((k, kc, 0), (v, vc, 1)):
        codes, e = kv_fp8.quantise(x, bool(which))
        for t, s in enumerate(slots):
            if 0 <= s < pages * P:
                pool[s] = codes[t]
                sc[s // P, :, which, s % P] = e[t]
    shape = (pages, P, Hkv, D)
    return kc.reshape(shape), vc.reshape(shape), sc


def _check_pool(got, want):
    for name, g, w in zip(("k", "v", "scale"), got, want):
        g = g.view(torch.uint8).cpu().numpy()
        at = np.argwhere(g != w)
        assert not len(at), f"{name}: {len(at)} differ, first {at[0]}: " \
                            f"{g[tuple(at[0])]} != {w[tuple(at[0])]}"


@pytest.mark.parametrize("T,Hkv,D,P", [(1, 2, 64, 16), (37, 2, 64, 16), (160, 8, 128, 16),
                                       (301, 1, 128, 1), (77, 3, 64, 2), (130, 16, 64, 64),
                                       (9, 5, 128, 8)])
def test_write_matches_the_definition(T, Hkv, D, P):
    rng = np.random.default_rng(T)
    pages = -(-T // P) + 3
    slots = rng.permutation(pages * P)[:T].astype(np.int64)
    if T > 5:
        slots[[1, 4]] = -1
        slots[5] = pages * P + 3                       # past the pool: skipped too
    k, v = (fc.rows(rng, T, Hkv, D, spread=3.0) for _ in range(2))
    # strided views of a fused projection, k and v of different token strides
    kt = torch.zeros(T, (2 + Hkv + 1) * D, device="cuda", dtype=torch.bfloat16)
    vt = torch.zeros(T, (Hkv + 8) * D, device="cuda", dtype=torch.bfloat16)
    kt[:, 2 * D:(2 + Hkv) * D] = torch.from_numpy(k.reshape(T, -1)).cuda().bfloat16()
    vt[:, 8 * D:] = torch.from_numpy(v.reshape(T, -1)).cuda().bfloat16()
    pool = _empty_pool(pages, P, Hkv, D)
    _kernels().kv_write_fp8(kt[:, 2 * D:(2 + Hkv) * D].view(T, Hkv, D),
                            vt[:, 8 * D:].view(T, Hkv, D), torch.from_numpy(slots).cuda(), *pool)
    _check_pool(pool, _expected(k, v, slots, pages, P, Hkv, D))


def test_write_at_the_edges_of_the_range():
    """Zero rows, the smallest and largest magnitudes, both sides of 448, rows
    on a tie, NaN and infinities."""
    D, Hkv, P = 64, 1, 16
    tiny, big = 2.0 ** -133, 3.3895313892515355e38      # bf16's smallest and largest
    tops = [0.0, tiny, 3 * tiny, 2.0 ** -126, 448 * 2.0 ** -126, 449 * 2.0 ** -126, 448.0, 450.0,
            446.0, 1.75, 1.7578125, 1.0, big, big / 2, np.inf, -np.inf, np.nan]
    rng = np.random.default_rng(0)
    x = np.zeros((len(tops), Hkv, D))
    for i, top in enumerate(tops):
        if np.isfinite(top):
            x[i] = fc.bf16(top * rng.uniform(-1, 1, (Hkv, D)))
        else:
            x[i] = rng.standard_normal((Hkv, D))
            x[i] = fc.bf16(x[i])
        x[i, 0, rng.integers(D)] = top
    x[6, 0, 1:9] = [1.0625, 1.1875, 17, 19, 0.0009765625, 0.0029296875, -0.0, 2.0 ** -20]  # ties
    x = fc.bf16(x)          # what the kernel gets (449 * 2^-126 is no bf16 value)
    v = np.roll(x, 3, 0)
    pool = _empty_pool(2, P, Hkv, D)
    slots = torch.arange(len(tops)).cuda()
    k_t, v_t = (torch.from_numpy(a).cuda().bfloat16() for a in (x, v))
    _kernels().kv_write_fp8(k_t, v_t, slots, *pool)
    want = _expected(x, v, range(len(tops)), 2, P, Hkv, D)
    _check_pool(pool, want)
    # and back: exactly the values, NaN rows NaN throughout
    k, v = _kernels().kv_read_fp8(slots, *pool)
    for got, val in zip((k, v), fc.values(*want)):
        val = val.reshape(-1, Hkv, D)[:len(tops)]
        # below bf16's smallest the value rounds: half of 2^-133
        assert np.array_equal(np.isnan(got.float().cpu().numpy()), np.isnan(val))
        d = np.abs(got.double().cpu().numpy() - val)
        assert np.nanmax(d) <= 2.0 ** -134
        assert (np.nan_to_num(d)[np.abs(np.nan_to_num(val)) >= 2.0 ** -120] == 0).all()


@pytest.mark.parametrize("T,Hkv,D,P", [(1, 2, 64, 16), (333, 8, 128, 16), (50, 3, 64, 1),
                                       (129, 1, 128, 32)])
def test_read_gives_the_values_exactly_and_zeros_for_padding(T, Hkv, D, P):
    rng = np.random.default_rng(T + 1)
    pages = -(-T // P) + 2
    kc, vc, sc, kval, vval = fc.pool(rng, pages, P, Hkv, D)
    slots = rng.permutation(pages * P)[:T].astype(np.int64)
    if T > 3:
        slots[2], slots[3] = -1, pages * P
    k, v = _kernels().kv_read_fp8(torch.from_numpy(slots).cuda(), *fc.on_gpu(kc, vc, sc))
    ok = (slots >= 0) & (slots < pages * P)
    for got, val in ((k, kval), (v, vval)):
        want = np.where(ok[:, None, None], val.reshape(-1, Hkv, D)[np.where(ok, slots, 0)], 0.0)
        assert np.array_equal(got.double().cpu().numpy(), want)


@pytest.mark.parametrize("T,Hq,Hkv,D,P", [(1, 14, 2, 64, 16), (160, 14, 2, 64, 16),
                                          (213, 32, 8, 128, 16), (33, 4, 4, 128, 1),
                                          (700, 16, 16, 64, 8)])
def test_rope_write_is_the_bf16_ropes_rows_quantised(T, Hq, Hkv, D, P):
    """q bit for bit that of rope_kv_write; the pool what the definition makes
    of the K and V rows that rope_kv_write stores."""
    K = _kernels()
    rng = np.random.default_rng(T)
    pages = -(-T // P) + 3
    qkv = torch.from_numpy(fc.rows(rng, T, (Hq + 2 * Hkv), D)).cuda().bfloat16()
    wide = torch.zeros(T, (Hq + 2 * Hkv) * D + 24, device="cuda", dtype=torch.bfloat16)
    wide[:, :(Hq + 2 * Hkv) * D] = qkv.view(T, -1)
    x = wide[:, :(Hq + 2 * Hkv) * D]
    pos = torch.from_numpy(rng.integers(0, 500, T)).cuda()
    a = torch.outer(torch.arange(500.), 1e4 ** (-torch.arange(0, D, 2) / D))
    cos, sin = a.cos().cuda(), a.sin().cuda()
    slots = torch.from_numpy(rng.permutation(pages * P)[:T]).cuda()
    if T > 4:
        slots[3] = -1
    kb = torch.zeros(pages, P, Hkv, D, device="cuda", dtype=torch.bfloat16)
    vb = torch.zeros_like(kb)
    q_ref = K.rope_kv_write(x, Hq, Hkv, D, pos, cos, sin, slots, kb, vb)
    pool = _empty_pool(pages, P, Hkv, D)
    q = K.rope_kv_write_fp8(x, Hq, Hkv, D, pos, cos, sin, slots, *pool)
    assert torch.equal(q, q_ref)
    at = slots.clamp_min(0).cpu()
    k, v = (b.view(-1, Hkv, D)[at].double().cpu().numpy() for b in (kb, vb))
    _check_pool(pool, _expected(k, v, slots.tolist(), pages, P, Hkv, D))
    # without slots: q alone
    assert torch.equal(K.rope_kv_write_fp8(x, Hq, Hkv, D, pos, cos, sin, None, None, None, None),
                       q_ref)


def test_empty_calls_and_int32_slots():
    K = _kernels()
    pool = _empty_pool(2, 16, 2, 64)
    before = [t.clone() for t in pool]
    e = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    K.kv_write_fp8(e, e, none, *pool)
    assert K.kv_read_fp8(none, *pool)[0].shape == (0, 2, 64)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, before))
    x = torch.randn(3, 2, 64, device="cuda").bfloat16()
    K.kv_write_fp8(x, x, torch.tensor([4, 9, 31], dtype=torch.int32, device="cuda"), *pool)
    k, v = K.kv_read_fp8(torch.tensor([4, 9, 31], dtype=torch.int32, device="cuda"), *pool)
    assert torch.equal(k, v) and (k.float() - x.float()).abs().max() <= 2.0 ** -4 * x.abs().max()


def test_writes_and_reads_replay_in_a_graph_on_another_stream():
    """Captured once, replayed with other rows in the same buffers; eager work
    and synchronisations between the replays."""
    K = _kernels()
    rng = np.random.default_rng(9)
    T, Hq, Hkv, D, P = 40, 4, 2, 64, 16
    pool = _empty_pool(4, P, Hkv, D)
    qkv = torch.zeros(T, (Hq + 2 * Hkv) * D, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(T).cuda()
    a = torch.outer(torch.arange(64.), 1e4 ** (-torch.arange(0, D, 2) / D))
    cos, sin = a.cos().cuda(), a.sin().cuda()
    slots = torch.from_numpy(rng.permutation(4 * P)[:T]).cuda()

    def step():
        q = K.rope_kv_write_fp8(qkv, Hq, Hkv, D, pos, cos, sin, slots, *pool)
        return (q, *K.kv_read_fp8(slots, *pool))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(3):
        qkv.copy_(torch.randn(T, qkv.shape[1], device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), f"replay {i}"
