"""Seeded 8-bit KV pools and their 64-bit attention, for the CPU and GPU tests."""
import numpy as np
import torch

from oracle import kv_fp8

FP8 = torch.float8_e4m3fn


def bf16(x):
    """Values rounded to bf16, as float64."""
    return torch.from_numpy(np.asarray(x, np.float32)).to(torch.bfloat16).double().numpy()


def rows(rng, *shape, spread=0.5):
    """K or V rows with a magnitude of their own each."""
    return bf16(rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[:-1] + (1,))))


def pool(rng, pages, P, Hkv, D):
    """(k codes, v codes, scale bytes, k values, v values) of a layer's pool."""
    out, e = [], []
    for is_v in (False, True):
        c, b = kv_fp8.quantise(rows(rng, pages, P, Hkv, D), is_v)
        out.append(c)
        e.append(b)
    scale = np.stack(e, 2).transpose(0, 3, 2, 1)         # (pages, Hkv, 2, P)
    return out[0], out[1], np.ascontiguousarray(scale), *values(out[0], out[1], scale)


def values(kc, vc, scale):
    e = scale.transpose(2, 0, 3, 1)                      # (2, pages, P, Hkv)
    return kv_fp8.dequantise(kc, e[0]), kv_fp8.dequantise(vc, e[1])


def on_gpu(kc, vc, scale):
    d = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (kc, vc, scale)]
    return d[0].view(FP8), d[1].view(FP8), d[2]


def tables(rng, kv_lens, P, pages):
    need = [-(-n // P) for n in kv_lens]
    perm = rng.permutation(pages)[:sum(need)]
    return [t.tolist() for t in np.split(perm, np.cumsum(need)[:-1])]


def csr(tabs, kv_lens, P):
    ptr = np.concatenate([[0], np.cumsum([len(t) for t in tabs])]).astype(np.int32)
    idx = np.asarray([i for t in tabs for i in t], np.int32)
    last = np.asarray([(n - 1) % P + 1 if n else 0 for n in kv_lens], np.int32)
    return ptr, idx, last


def attention(q, spans, q_lens, causal=True, scale=None):
    """64-bit attention and the bound on a kernel's error.

    q (T, Hq, D) float64; spans[b] = (k, v), each (L_b, Hkv, D) float64: request
    b's context in order; bottom-right causal.  Returns (out, bound).  The bound
    counts: probabilities rounded to bf16 (2^-8 of each), the output's rounding
    (2^-8), and the fp32 score, D products and a few more roundings of 2^-24 of
    their magnitude, which moves a probability by as much relative to itself,
    the row's sum again by as much."""
    T, Hq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    out, bound = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    t0 = 0
    for (k, v), n in zip(spans, q_lens):
        L, Hkv = k.shape[:2]
        G = Hq // Hkv
        seen = L - n + np.arange(n) if causal else np.full(n, L - 1)
        hide = np.arange(L)[None] > seen[:, None]
        for h in range(Hq):
            qq, kk, vv = q[t0:t0 + n, h], k[:, h // G], v[:, h // G]
            s = np.where(hide, -np.inf, qq @ kk.T * scale)
            mag = np.where(hide, 0, np.abs(qq) @ np.abs(kk).T * scale).max(1)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            vz = np.nan_to_num(vv)          # masked rows may be NaN
            o = np.where(np.isnan(p @ np.where(np.isnan(vv), 1.0, 0)), np.nan, p @ vz)
            o = np.where((p @ np.isnan(vv).astype(float)) > 0, np.nan, o)
            eps = 2.0 ** -8 + 2 * (D + 8 + L / 64) * 2.0 ** -24 * (1 + mag)
            out[t0:t0 + n, h] = o
            bound[t0:t0 + n, h] = p @ np.abs(vz) * eps[:, None] + np.abs(o) * 2.0 ** -8 + 1e-30
        t0 += n
    return out, bound


def ramp(rng, n, Hkv, D, slope):
    """K rows that every positive query scores slope * (j / n) higher or lower
    with position j: n rows of one direction, exact in e4m3 with their scale."""
    a = np.round(slope * np.arange(n) / n * 4) / 4
    return bf16(np.repeat(a[:, None, None], Hkv, 1) * np.ones(D))


def check(got, want, bound):
    """got (bf16 tensor) within bound of want; where want is NaN got is."""
    g = got.double().cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(g), nan), "NaN where none is due, or the reverse"
    over = np.where(nan, 0, np.abs(g - want) / bound)
    assert over.max(initial=0) <= 1, f"error {over.max():.3f} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
