"""The 8-bit pool's and the shared prefix's torch operators, and the 8-bit
pool's users, on a host without a GPU: schemas, shapes, refusals."""
import numpy as np
import pytest
import torch

from nanosglang_amd import kernels, ops  # noqa: F401  (ops loads the operators)
from nanosglang_amd.engine.paged_kv_cache import BlockManager, PagedKVCache

FP8 = torch.float8_e4m3fn
POOL = ["k_cache", "v_cache", "kv_scale"]
PAGES = ["paged_kv_indptr", "paged_kv_indices", "paged_kv_last_page_len"]


@pytest.mark.parametrize("name,args,written", [
    ("kv_write_fp8", ["k", "v", "slots"] + POOL, set(POOL)),
    ("kv_read_fp8", ["slots"] + POOL, set()),
    ("rope_kv_write_fp8", ["qkv", "num_qo_heads", "num_kv_heads", "head_dim", "positions",
                           "cos_table", "sin_table", "slots"] + POOL, set(POOL)),
    ("verify_attention_fp8", ["q"] + POOL + ["qo_indptr"] + PAGES + ["causal", "sm_scale"], set()),
    ("verify_attention_plan_fp8", ["qo_indptr", "paged_kv_indptr", "paged_kv_last_page_len",
                                   "num_qo_heads", "num_kv_heads", "head_dim", "page_size",
                                   "causal", "num_cus"], set()),
    ("verify_attention_run_fp8", ["plan", "work", "q"] + POOL + [
        "paged_kv_indices", "sm_scale", "causal", "workspace", "out"], {"workspace", "out"}),
    ("shared_prefix_attention", ["q"] + POOL + [
        "qo_indptr", "group_indptr", "prefix_kv_indptr", "prefix_kv_indices",
        "prefix_kv_last_page_len"] + PAGES + ["causal", "sm_scale"], set()),
])
def test_schemas_and_kernels(name, args, written):
    schema = getattr(torch.ops.nsg, name).default._schema
    assert [a.name for a in schema.arguments] == args
    assert {a.name for a in schema.arguments
            if a.alias_info is not None and a.alias_info.is_write} == written
    for key in ("CUDA", "CPU"):
        assert torch._C._dispatch_has_kernel_for_dispatch_key(f"nsg::{name}", key), key


@pytest.mark.parametrize("batch,q,lo,hi", [(64, 9, 2048, 8192), (300, 1, 500, 4000),
                                           (4, 5, 100, 640)])
def test_plans_of_the_8_bit_pool_cut_contexts_half_as_often(batch, q, lo, hi):
    """The same tiles, in fewer and longer items; short contexts (several KV
    groups a workgroup) are not cut differently."""
    rng = np.random.default_rng(batch)
    kv = rng.integers(lo, hi, batch)
    ptr = np.concatenate([[0], np.cumsum(-(-kv // 16))]).astype(np.int32)
    args = [torch.from_numpy(x) for x in ((np.arange(batch + 1) * q).astype(np.int32), ptr,
                                          ((kv - 1) % 16 + 1).astype(np.int32))]
    plans = [ops.plan_from_record(op(*args, 32, 8, 128, 16)[0])[0] for op in (
        torch.ops.nsg.verify_attention_plan, torch.ops.nsg.verify_attention_plan_fp8)]
    a, b = plans
    assert (a.num_groups, a.row_tiles, a.kv_groups) == (b.num_groups, b.row_tiles, b.kv_groups)
    if a.kv_groups > 1:
        assert bytes(a) == bytes(b)
    else:
        assert batch <= b.num_work < a.num_work and b.max_splits < a.max_splits
        assert b.workspace_bytes < a.workspace_bytes


def _step_items(lib, kv8):
    """Work items of each attention call of a filled step, whose plans have to be
    the pool's own planner's."""
    import ctypes as C
    from nanosglang_amd._native import NSG_ATTN_WORK_INTS, AttnPlan
    from tests import test_step_fill as sf
    B, k, P, pages = 6, 3, 16, 300
    tab = np.arange(B * pages, dtype=np.int32).reshape(B, pages)
    starts = np.asarray([4000, 90, 2500, 17, 4700, 3333], np.int64)
    npg = ((starts + k + P) // P).astype(np.int32)
    st = sf._Staging(lib, B, k, 0, ids_stride=B * pages)
    st.bufs.kv8 = kv8
    assert sf._fill(lib, st, tab, np.arange(B, dtype=np.int32), npg, starts,
                    np.zeros(B, np.int64), B, k, P, B * pages - 1, 0) == 0, lib.nsg_last_error()
    items = []
    for a in range(k + 1):
        ql = 1 if a < k else k + 1
        L = starts + (a + 1 if a < k else k + 1)
        ptr = np.concatenate([[0], np.cumsum(-(-L // P))]).astype(np.int32)
        qo, last = (np.arange(B + 1) * ql).astype(np.int32), ((L - 1) % P + 1).astype(np.int32)
        mw, mm, pl = C.c_int32(0), C.c_int32(0), AttnPlan()
        assert lib.nsg_attn_fixed_capacity(B, ql, sf.Hq, sf.Hkv, sf.CUS, 0, C.byref(mw),
                                           C.byref(mm)) == 0
        n = (mw.value + mm.value) * NSG_ATTN_WORK_INTS
        work = np.zeros(n, np.int32)
        plan = lib.nsg_attn_plan_fixed_fp8 if kv8 else lib.nsg_attn_plan_fixed
        assert plan(qo.ctypes.data, ptr.ctypes.data, last.ctypes.data, B, sf.Hq, sf.Hkv, sf.D, P,
                    1, sf.CUS, ql, 0, mw.value, mm.value, work.ctypes.data,
                    n // NSG_ATTN_WORK_INTS, C.byref(pl)) == 0
        np.testing.assert_array_equal(st.work[a * st.sw:a * st.sw + n], work)
        assert bytes(st.plans[a]) == bytes(pl)
        items.append(int((work.reshape(-1, NSG_ATTN_WORK_INTS)[:mw.value, 1] > 0).sum()))
    assert all(i > B for i in items)                     # split
    return items


def test_step_fill_plans_for_its_pool(lib):
    """Long contexts (no bound: split plans), in fewer items over the 8-bit pool."""
    assert all(x < y for x, y in zip(_step_items(lib, 1), _step_items(lib, 0)))


def _args(device):
    i32 = dict(dtype=torch.int32, device=device)
    pool = [torch.empty(8, 16, 2, 64, device=device, dtype=FP8) for _ in range(2)]
    pool.append(torch.empty(8, 2, 2, 16, device=device, dtype=torch.uint8))
    csr = [torch.empty(3, **i32), torch.empty(5, **i32), torch.empty(2, **i32)]
    row = lambda *s: torch.empty(*s, device=device, dtype=torch.bfloat16)
    slots = torch.empty(6, device=device, dtype=torch.int64)
    tab = torch.empty(64, 32, device=device)
    qo = torch.empty(3, **i32)
    return dict(
        kv_write_fp8=[row(6, 2, 64), row(6, 2, 64), slots, *pool],
        kv_read_fp8=[slots, *pool],
        rope_kv_write_fp8=[row(6, 18 * 64), 14, 2, 64, slots, tab, tab, slots, *pool],
        verify_attention_fp8=[row(6, 14, 64), *pool, qo, *csr],
        verify_attention_run_fp8=[qo, qo, row(6, 14, 64), *pool, csr[1], 0.125, True, slots,
                                  row(6, 14, 64)],
        shared_prefix_attention=[row(6, 14, 64), *pool, qo, torch.empty(2, **i32),
                                 torch.empty(2, **i32), torch.empty(4, **i32),
                                 torch.empty(1, **i32), *csr])


def test_shapes_without_a_gpu():
    a = _args("meta")
    op = torch.ops.nsg
    for x in op.kv_read_fp8(*a["kv_read_fp8"]):
        assert (x.shape, x.dtype) == ((6, 2, 64), torch.bfloat16)
    for name in ("rope_kv_write_fp8", "verify_attention_fp8", "shared_prefix_attention"):
        x = getattr(op, name)(*a[name])
        assert (x.shape, x.dtype) == ((6, 14, 64), torch.bfloat16), name
    assert op.kv_write_fp8(*a["kv_write_fp8"]) is None


@pytest.mark.parametrize("name", list(_args("meta")))
def test_operators_refuse_host_tensors(name):
    with pytest.raises(RuntimeError, match="GPU tensor"):
        getattr(torch.ops.nsg, name)(*_args("cpu")[name])


def test_block_manager_of_an_8_bit_pool():
    bm = BlockManager(6, 16, 3, 2, 64, FP8, "cpu", row_scales=True)
    assert [t.dtype for t in bm.caches] == [FP8, FP8, torch.uint8]
    assert bm.kv_scale.shape == (3, 6, 2, 2, 16)
    assert bm.memory_bytes == 3 * 6 * 16 * 2 * (2 * 64 + 2)
    t = PagedKVCache(bm).allocate_for_request(40)
    z = torch.zeros(2, 5, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensor"):        # no CPU path
        bm.write_kv(t.block_indices[0], 0, 3, z, z)
    with pytest.raises(ValueError, match="do not fit"):          # the next block's slots
        bm.write_kv(t.block_indices[0], 0, 12, z, z)
    for dtype in (torch.bfloat16, FP8):                          # caches of any type, as before
        plain = BlockManager(6, 16, 3, 2, 64, dtype, "cpu")
        plain.write_kv(2, 1, 3, z + 1, z + 2)
        k, v = plain.read_kv([2], 1, 8)
        assert plain.kv_scale is None and len(plain.caches) == 2
        assert (k[:, 3:].float() == 1).all() and (v[:, 3:].float() == 2).all()
    with pytest.raises(ValueError, match="row_scales"):
        BlockManager(6, 16, 3, 2, 64, torch.bfloat16, "cpu", row_scales=True)


def test_bf16_writers_refuse_the_8_bit_pool(monkeypatch):
    """They would write two bytes for each of the pool's one."""
    monkeypatch.setattr(kernels, "_require_gpu", lambda *a: None)
    pool = torch.zeros(4, 16, 2, 64, dtype=FP8)
    bf = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    z = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    x, w = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(256, 64, dtype=torch.bfloat16)
    s = torch.zeros(3, dtype=torch.int64)
    for k, v in ((pool, pool), (bf, pool), (pool, bf)):
        with pytest.raises(TypeError):
            kernels.kv_write(z, z, s, k, v)
        with pytest.raises(TypeError, match="8-bit pool"):
            kernels.rope_kv_write(torch.zeros(3, 512, dtype=torch.bfloat16), 4, 2, 64, s, s, s, s,
                                  k, v)
        with pytest.raises(TypeError, match="8-bit pool"):
            kernels.linear_rope_kv(x, w, None, 0, 2, 64, s, s, s, s, k, v)
        with pytest.raises(TypeError, match="8-bit pool"):
            kernels.kv_clear_slots(s, k[None], v[None])


def test_projection_into_the_8_bit_pool_refuses(monkeypatch):
    monkeypatch.setattr(kernels, "_require_gpu", lambda *a: None)
    x, w = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(512, 64, dtype=torch.bfloat16)
    s, tab = torch.zeros(3, dtype=torch.int64), torch.zeros(8, 32)
    pool = torch.zeros(4, 16, 2, 64, dtype=FP8)
    sc = torch.zeros(4, 2, 2, 16, dtype=torch.uint8)
    bf = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    call = lambda *a, **kw: kernels.linear_rope_kv(x, w, None, 4, 2, 64, s, tab, tab, *a,
                                                   force=True, **kw)
    with pytest.raises(TypeError, match="float8_e4m3fn"):
        call(s, bf, bf, kv_scale=sc)
    with pytest.raises(ValueError, match="kv_scale must be"):
        call(s, pool, pool, kv_scale=sc[1:])
    with pytest.raises(ValueError, match="do not match"):
        call(s, pool[:, :, :1].contiguous(), pool[:, :, :1].contiguous(), kv_scale=sc)
    with pytest.raises(ValueError, match="without slots"):
        call(None, None, None, kv_scale=sc)
