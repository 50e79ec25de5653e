"""torch.ops.nsg.* of the 8-bit pool and of shared prefixes run the kernels of
the host wrappers: results equal the wrappers' bit for bit, and theirs are
checked against 64-bit references elsewhere."""
import numpy as np
import pytest
import torch

from nanosglang_amd import kernels, ops
from tests import _fp8_cases as fc

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
OP = torch.ops.nsg


def _empty(pages, P, Hkv, D):
    kc = torch.zeros(pages, P, Hkv, D, dtype=torch.uint8, device="cuda")
    return kc.view(FP8), kc.clone().view(FP8), torch.zeros(pages, Hkv, 2, P, dtype=torch.uint8,
                                                           device="cuda")


def _same_pool(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("T,slots_type", [(1, torch.int64), (37, torch.int32), (0, torch.int64)])
def test_writes_and_reads(T, slots_type):
    g = torch.Generator().manual_seed(T)
    Hq, Hkv, D, P, pages = 14, 2, 64, 16, 9
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).bfloat16().cuda()
    k, v = (qkv[:, (Hq + i * Hkv) * D:][:, :Hkv * D].view(T, Hkv, D) for i in range(2))
    slots = torch.randperm(pages * P, generator=g)[:T].to(slots_type).cuda()
    pos = torch.randint(0, 128, (T,), generator=g).cuda()
    ang = torch.rand(128, D // 2, generator=g).cuda()
    a, b = _empty(pages, P, Hkv, D), _empty(pages, P, Hkv, D)
    kernels.kv_write_fp8(k, v, slots, *a)
    OP.kv_write_fp8(k, v, slots, *b)
    assert _same_pool(a, b)
    for x, y in zip(kernels.kv_read_fp8(slots, *a), OP.kv_read_fp8(slots, *b)):
        assert torch.equal(x, y)
    a, b = _empty(pages, P, Hkv, D), _empty(pages, P, Hkv, D)
    cos, sin = ang.cos(), ang.sin()
    q = kernels.rope_kv_write_fp8(qkv, Hq, Hkv, D, pos, cos, sin, slots, *a)
    assert torch.equal(q, OP.rope_kv_write_fp8(qkv, Hq, Hkv, D, pos, cos, sin, slots, *b))
    assert _same_pool(a, b)


def _batch(seed, Hq, Hkv, D, P, q_lens, prefix, own):
    """A pool, its CSR arrays with one prefix of `prefix` tokens before all."""
    rng = np.random.default_rng(seed)
    lens = [prefix] + own
    pages = sum(-(-n // P) for n in lens) + 2
    pool = fc.pool(rng, pages, P, Hkv, D)
    tabs = fc.tables(rng, lens, P, pages)
    qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(qo[-1]), Hq, D))).cuda().bfloat16()
    return pool, tabs, lens, qo, q


def _csr(tabs, lens, P, device="cuda"):
    return [torch.from_numpy(x).to(device) for x in fc.csr(tabs, lens, P)]


@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 64), (32, 8, 128)])
def test_attention_equals_the_wrapper_and_replays(Hq, Hkv, D):
    P, q_lens, own = 16, [1, 5, 2], [40, 700, 16]
    pool, tabs, lens, qo, q = _batch(1, Hq, Hkv, D, P, q_lens, 1, own)
    kc, vc, sc = fc.on_gpu(*pool[:3])
    ptr, idx, last = _csr(tabs[1:], own, P)
    qo_d = torch.from_numpy(qo).cuda()
    w = kernels.BatchPrefillWithPagedKVCacheWrapper(
        torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan(qo, ptr, idx, last, Hq, Hkv, D, P, kv_data_type=FP8)
    want = w.run(q, (kc, vc), kv_scale=sc)
    assert torch.equal(OP.verify_attention_fp8(q, kc, vc, sc, qo_d, ptr, idx, last), want)
    rec, work = OP.verify_attention_plan_fp8(torch.from_numpy(qo), ptr.cpu(), last.cpu(), Hq, Hkv, D, P)
    ws = torch.zeros(max(1, ops.plan_workspace_bytes(rec)), dtype=torch.uint8, device="cuda")
    out, work, q_s = torch.empty_like(q), work.cuda(), q.clone()
    run = lambda: OP.verify_attention_run_fp8(rec, work, q_s, kc, vc, sc, idx, D ** -0.5, True, ws,
                                              out)
    run()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run()
    for rep in range(3):
        q_s.copy_(torch.randn(q.shape, device="cuda").bfloat16())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w.run(q_s, (kc, vc), kv_scale=sc)), rep
    with pytest.raises(ValueError, match="as planned"):
        OP.verify_attention_run_fp8(rec, work, q[:-1].contiguous(), kc, vc, sc, idx, 0.1, True, ws,
                                    out[:-1].contiguous())
    with pytest.raises(ValueError, match="kv_scale"):
        OP.verify_attention_fp8(q, kc, vc, sc[1:], qo_d, ptr, idx, last)
    with pytest.raises(ValueError, match="page ids"):
        OP.verify_attention_fp8(q, kc, vc, sc, qo_d, ptr, idx[:-1], last)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("prefix", [0, 300])
def test_shared_prefix_equals_the_wrapper(fp8, prefix):
    Hq, Hkv, D, P, own = 14, 2, 64, 16, [9, 1, 33, 70]
    pool, tabs, lens, qo, q = _batch(2, Hq, Hkv, D, P, [1, 1, 5, 2], prefix, own)
    if fp8:
        kc, vc, sc = fc.on_gpu(*pool[:3])
    else:
        kc, vc = (torch.from_numpy(x).cuda().bfloat16() for x in pool[3:])
        sc = None
    pre, rest = _csr(tabs[:1], [prefix], P), _csr(tabs[1:], own, P)
    grp = torch.tensor([0, 4], dtype=torch.int32)
    w = kernels.SharedPrefixAttentionWrapper(torch.empty(64 << 20, dtype=torch.uint8,
                                                         device="cuda"))
    w.plan(qo, grp, *pre, *rest, Hq, Hkv, D, P, kv_data_type=FP8 if fp8 else torch.bfloat16)
    want = w.run(q, (kc, vc), kv_scale=sc)
    got = OP.shared_prefix_attention(q, kc, vc, sc, torch.from_numpy(qo), grp, *pre, *rest)
    assert torch.equal(got, want)
    with pytest.raises(ValueError, match="rows"):
        OP.shared_prefix_attention(q[:-1].contiguous(), kc, vc, sc, torch.from_numpy(qo), grp,
                                   *pre, *rest)
    with pytest.raises(ValueError, match="batch or groups"):
        OP.shared_prefix_attention(q, kc, vc, sc, torch.from_numpy(qo), grp, *pre, rest[0][:-1],
                                   *rest[1:])
