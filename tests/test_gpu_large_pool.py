"""Pools whose rows lie past 32-bit byte offsets, and empty batches, for the
8-bit pool and for shared prefixes (bf16 and 8-bit)."""
import numpy as np
import pytest
import torch

from nanosglang_amd import kernels
from tests import _fp8_cases as fc

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16
Hq, Hkv, D, P = 32, 8, 128, 16
PAGES = (1 << 32) // (P * Hkv * D) + 1200       # codes past 4 GiB, bf16 rows past 8


def _ws(mb=256):
    return torch.empty(mb << 20, dtype=torch.uint8, device="cuda")


def _far(small):
    """A pool of PAGES pages whose last ones are the small pool's."""
    big = torch.empty((PAGES,) + tuple(small.shape[1:]), dtype=torch.uint8 if small.dtype == FP8
                      else small.dtype, device="cuda")
    big[PAGES - small.shape[0]:] = small.view(big.dtype)
    return big.view(small.dtype)


@pytest.fixture(scope="module")
def pools():
    rng = np.random.default_rng(0)
    n = 600
    p = fc.pool(rng, n, P, Hkv, D)
    small = fc.on_gpu(*p[:3])
    bf = tuple(torch.from_numpy(x).cuda().bfloat16() for x in p[3:])
    big = tuple(_far(t) for t in small)
    big_bf = tuple(_far(t) for t in bf)
    yield dict(n=n, small=small, big=big, bf=bf, big_bf=big_bf)
    torch.cuda.empty_cache()


def test_writes_and_reads_past_4_gib(pools):
    print("case: 8-bit pool past 4 GiB, write and read", flush=True)
    big, T = pools["big"], 37
    assert big[0].numel() > 1 << 32
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(T, Hkv, D, generator=g).bfloat16().cuda() for _ in range(2))
    far = torch.arange(T, device="cuda") * 3 + (PAGES - 400) * P
    near = torch.arange(T, device="cuda") * 3 + (pools["n"] - 400) * P
    small = [t.clone() for t in pools["small"]]
    kernels.kv_write_fp8(k, v, far, *big)
    kernels.kv_write_fp8(k, v, near, *small)
    for a, b in zip(kernels.kv_read_fp8(far, *big), kernels.kv_read_fp8(near, *small)):
        assert torch.equal(a, b) and a.any()
    for a, b in zip(big, small):                           # nothing else moved
        assert torch.equal(a[PAGES - pools["n"]:].view(torch.uint8), b.view(torch.uint8))
        a[PAGES - pools["n"]:] = pools["small"][0 if a is big[0] else 1 if a is big[1] else 2]


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 5, 2], [300, 640, 17]),       # KV groups
                                            ([9] * 12, [700] * 12),             # split items
                                            ([300, 200], [2000, 900])])         # 256-row tiles
def test_attention_past_4_gib(pools, q_lens, kv_lens):
    rng = np.random.default_rng(2)
    tabs = fc.tables(rng, kv_lens, P, pools["n"])
    ptr, idx, last = fc.csr(tabs, kv_lens, P)
    qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(qo[-1]), Hq, D))).cuda().bfloat16()
    outs = []
    for pool, shift in ((pools["small"], 0), (pools["big"], PAGES - pools["n"])):
        w = kernels.BatchPrefillWithPagedKVCacheWrapper(_ws())
        w.plan(qo, ptr, idx + np.int32(shift), last, Hq, Hkv, D, P, kv_data_type=FP8)
        outs.append(w.run(q, pool[:2], kv_scale=pool[2]))
        assert w.check_flags() == 0
    assert torch.equal(*outs)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,q,prefix", [(6, 1, 900), (40, 5, 600), (40, 9, 6000)])
def test_shared_prefixes_past_4_gib(pools, fp8, n, q, prefix):
    rng = np.random.default_rng(3)
    own = [int(x) for x in rng.integers(q, 60, n)]
    tabs = fc.tables(rng, [prefix] + own, P, pools["n"])
    qo = np.arange(n + 1, dtype=np.int32) * q
    x = torch.from_numpy(rng.standard_normal((n * q, Hq, D))).cuda().bfloat16()
    outs = []
    for name, shift in (("", 0), ("big", PAGES - pools["n"])):
        pool = pools[name or "small"] if fp8 else (*pools["big_bf" if name else "bf"], None)
        pre, rest = fc.csr(tabs[:1], [prefix], P), fc.csr(tabs[1:], own, P)
        w = kernels.SharedPrefixAttentionWrapper(_ws())
        w.plan(qo, np.asarray([0, n]), pre[0], pre[1] + np.int32(shift), pre[2], rest[0],
               rest[1] + np.int32(shift), rest[2], Hq, Hkv, D, P,
               kv_data_type=FP8 if fp8 else BF16)
        outs.append(w.run(x, pool[:2], kv_scale=pool[2]))
        assert w.check_flags() == 0
    assert torch.equal(*outs)


def test_empty_batches(pools):
    pool, i32 = pools["small"], lambda *a: np.asarray(a, np.int32)
    q = torch.empty(0, Hq, D, dtype=BF16, device="cuda")
    w = kernels.BatchPrefillWithPagedKVCacheWrapper(_ws(1))
    w.plan(i32(0), i32(0), i32(), i32(), Hq, Hkv, D, P, kv_data_type=FP8)
    assert w.run(q, pool[:2], kv_scale=pool[2]).shape == (0, Hq, D)
    w = kernels.SharedPrefixAttentionWrapper(_ws(1))
    for grp, pre in ((i32(0), (i32(0), i32(), i32())), (i32(0, 0), (i32(0, 1), i32(3), i32(5)))):
        w.plan(i32(0), grp, *pre, i32(0), i32(), i32(), Hq, Hkv, D, P, kv_data_type=FP8)
        assert w.run(q, pool[:2], kv_scale=pool[2]).shape == (0, Hq, D)
    # requests without query tokens among others
    w.plan(i32(0, 0, 1, 1), i32(0, 3), i32(0, 1), i32(7), i32(9), i32(0, 1, 2, 3), i32(1, 2, 3),
           i32(4, 5, 6), Hq, Hkv, D, P, kv_data_type=FP8)
    x = torch.randn(1, Hq, D, device="cuda").bfloat16()
    got = w.run(x, pool[:2], kv_scale=pool[2])
    k, v = fc.values(*(t.view(torch.uint8).cpu().numpy() for t in pool))
    span = tuple(np.concatenate([a[7].reshape(P, Hkv, D)[:9], a[2].reshape(P, Hkv, D)[:5]])
                 for a in (k, v))
    fc.check(got, *fc.attention(x.double().cpu().numpy(), [span], [1]))
