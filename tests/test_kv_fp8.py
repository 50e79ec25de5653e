"""The 8-bit KV pool without a GPU: the oracle's own definition, the C entry
points' argument checks, the wrappers' refusals."""
import ctypes as C

import numpy as np
import pytest
import torch

from nanosglang_amd import kernels
from nanosglang_amd._native import AttnPlan
from oracle import kv_fp8


def test_oracle_codes_are_torchs_e4m3():
    """encode / decode against torch's float8_e4m3fn on every bf16 value up to
    448 and every code."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16).float()
    x = x[torch.isfinite(x) & (x.abs() <= 448)]
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kv_fp8.encode(x.double().numpy()), want)
    codes = np.arange(256, dtype=np.uint8)
    back = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv_fp8.decode(codes), back, equal_nan=True)


def test_oracle_scale_is_the_smallest_that_holds_the_row():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 8)) * 2.0 ** rng.uniform(-130, 120, (500, 1))
    _, e = kv_fp8.quantise(x, False)
    top = np.abs(x).max(1)
    s = 2.0 ** (e.astype(float) - 127)
    assert (top <= 448 * s).all() and ((top > 224 * s) | (e == 1)).all()
    codes, e = kv_fp8.quantise(np.array([[0.0, -0.0], [1.0, np.nan], [np.inf, 0]]), True)
    assert e.tolist() == [1, 255, 255] and not codes[1:].any()


# a row's relative error is at most 2^-4 while its code is normal: a value at
# least 2^-6 of the scale, that is 2^-14 of the row's largest
def test_oracle_rounding_error():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((200, 64))
    codes, e = kv_fp8.quantise(x, False)
    back = kv_fp8.dequantise(codes, e)
    big = np.abs(x) >= np.abs(x).max(1, keepdims=True) * 2.0 ** -14
    assert (np.abs(back - x)[big] <= 2.0 ** -4 * np.abs(x)[big]).all()


OK = 0x1000        # an aligned address that no refused call touches


@pytest.mark.parametrize("change,match", [
    (dict(num_tokens=-1), "num_tokens"), (dict(k=None), "null"), (dict(slots=None), "null"),
    (dict(kv_scale=None), "null"), (dict(head_dim=96), "head_dim"), (dict(page=12), "page_size"),
    (dict(page=0), "page_size"), (dict(num_slots=40), "whole pages"), (dict(heads=0), "kv_heads"),
    (dict(ks=100), "strides"), (dict(vs=130), "strides"), (dict(k=OK + 8), "aligned"),
    (dict(k_cache=OK + 4), "aligned"), (dict(num_tokens=2**31 - 1, heads=64), "one launch")])
def test_write_refuses(lib, change, match):
    a = dict(k=OK, ks=128, v=OK, vs=128, slots=OK, num_tokens=5, k_cache=OK, v_cache=OK,
             kv_scale=OK, heads=2, head_dim=64, page=16, num_slots=160)
    a.update(change)
    if a["heads"] == 64:
        a.update(ks=4096, vs=4096)
    rc = lib.nsg_kv_write_fp8(a["k"], a["ks"], a["v"], a["vs"], a["slots"], a["num_tokens"],
                              a["k_cache"], a["v_cache"], a["kv_scale"], a["heads"],
                              a["head_dim"], a["page"], a["num_slots"], None)
    assert rc in (1, 2) and match in lib.nsg_last_error().decode()


@pytest.mark.parametrize("change,match", [
    (dict(num_tokens=-1), "num_tokens"), (dict(qkv=None), "null"), (dict(q_out=None), "null"),
    (dict(head_dim=32), "head_dim"), (dict(stride=380), "stride"), (dict(stride=388), "stride"),
    (dict(max_position=0), "max_position"), (dict(page=3), "page_size"),
    (dict(k_cache=None), "null"), (dict(qkv=OK + 2), "aligned"), (dict(q_out=OK + 8), "aligned")])
def test_rope_write_refuses(lib, change, match):
    a = dict(qkv=OK, stride=384, max_position=100, slots=OK, num_tokens=5, head_dim=64, page=16,
             q_out=OK, k_cache=OK)
    a.update(change)
    rc = lib.nsg_rope_kv_write_fp8(a["qkv"], a["stride"], OK, OK, OK, a["max_position"],
                                   a["slots"], a["num_tokens"], 2, 2, a["head_dim"], a["page"],
                                   a["q_out"], a["k_cache"], OK, OK, 160, None, None)
    assert rc in (1, 2) and match in lib.nsg_last_error().decode()


@pytest.mark.parametrize("change,match", [
    (dict(num_tokens=-3), "num_tokens"), (dict(slots=None), "null"), (dict(k=None), "null"),
    (dict(head_dim=256), "head_dim"), (dict(page=-16), "page_size"), (dict(k=OK + 8), "aligned")])
def test_read_refuses(lib, change, match):
    a = dict(slots=OK, num_tokens=5, head_dim=128, page=16, k=OK)
    a.update(change)
    rc = lib.nsg_kv_read_fp8(a["slots"], a["num_tokens"], OK, OK, OK, 2, a["head_dim"], a["page"],
                             160, a["k"], OK, None)
    assert rc in (1, 2) and match in lib.nsg_last_error().decode()


def _plan_of(lib, P=16):
    qo, kvp, last = (np.asarray(x, np.int32) for x in ([0, 1], [0, 3], [5]))
    work = np.zeros(8 * 64, np.int32)
    pl = AttnPlan()
    assert lib.nsg_attn_plan(qo.ctypes.data, kvp.ctypes.data, last.ctypes.data, 1, 4, 2, 64, P, 1,
                             256, work.ctypes.data, 64, C.byref(pl)) == 0
    return pl


@pytest.mark.parametrize("change,rc,match", [
    (dict(kv_scale=None), 1, "null"), (dict(page=24), 1, "page_size"),
    (dict(num_pages=0), 1, "num_pages"), (dict(sm=0.0), 1, "sm_scale"), (dict(q=OK + 4), 1, "align"),
    (dict(ws=10), 3, "workspace")])
def test_attention_refuses(lib, change, rc, match):
    pl = _plan_of(lib)
    a = dict(q=OK, kv_scale=OK, page=16, num_pages=9, sm=0.1, ws=pl.workspace_bytes)
    a.update(change)
    got = lib.nsg_attn_run_fp8(C.byref(pl), OK, a["q"], OK, OK, a["kv_scale"], OK, OK, a["page"],
                               a["num_pages"], a["sm"], 1, OK, a["ws"], None)
    assert got == rc and match in lib.nsg_last_error().decode()


def test_wrappers_refuse_host_tensors_and_other_types():
    z = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.float8_e4m3fn)
    sc = torch.zeros(4, 2, 2, 16, dtype=torch.uint8)
    s = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.kv_write_fp8(z, z, s, pool, pool, sc)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.kv_read_fp8(s, pool, pool, sc)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        kernels.rope_kv_write_fp8(z.view(3, 128), 1, 1, 64, s, s, s, s, pool, pool, sc)
    with pytest.raises(NotImplementedError, match="kv_data_type"):
        kernels._kv_dtype(torch.float16)
