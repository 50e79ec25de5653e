"""The 8-bit KV cache and the shared-prefix attention: plain forms, the
framework's calls, and the sizes they are measured at.

The 8-bit pool of a layer holds e4m3 codes (pages, P, Hkv, D) for K and for V
and one power-of-two scale per token, KV head and K / V, an E8M0 byte e
(value 2^(e - 127)) in (pages, Hkv, 2, P).  A row is stored with the smallest
e >= 1 for which its largest magnitude is at most 448 * 2^(e - 127); its codes
are the row times 2^(127 - e), rounded to nearest even.

Kinds of cases: ``write`` (K / V rows into slots), ``rope`` (rotary embedding of
a fused projection, then the same write), ``read`` (slots back as bf16 rows),
``attn`` (ragged multi-query attention over the 8-bit pool, bottom-right
causal), ``prefix`` (the same attention where groups of requests share the first
part of their context; bf16 or 8-bit pool).  ``layers`` calls are made one
after the other over pools of their own, as in a model; the calls of a decode
or verify step (``graph``) are captured once and replayed, as the engine does.
Lengths follow from the case alone (``lens``), every value from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
FP8 = torch.float8_e4m3fn
SMALL = {"hq": 14, "hkv": 2, "d": 64}     # the 0.5B shape's heads
LARGE = {"hq": 32, "hkv": 8, "d": 128}    # the 8B shape's heads
MHA = {"hq": 16, "hkv": 16, "d": 64}      # no grouping
MQA = {"hq": 8, "hkv": 1, "d": 128}       # one KV head


def listed():
    return [
        # the K / V write of a verify step: 32 requests x 5 rows, every layer
        {"name": "rope_step", "kind": "rope", **SMALL, "tokens": 160, "page": 16, "layers": 24,
         "pad": 0, "graph": True},
        # the write of a prefill batch's prompts
        {"name": "rope_prefill", "kind": "rope", **LARGE, "tokens": 16384, "page": 16, "layers": 1,
         "pad": 0, "graph": False},
        # rows out of a fused projection, some of them padding (slot -1)
        {"name": "write_ragged", "kind": "write", **LARGE, "tokens": 1003, "page": 16, "layers": 1,
         "pad": 40, "graph": False},
        # a cached prompt read back for a dense pass over it
        {"name": "read_prompt", "kind": "read", **LARGE, "tokens": 2500, "page": 16, "layers": 1,
         "pad": 0, "graph": False},
        # a batch's whole cache read back (moved to another pool)
        {"name": "read_batch", "kind": "read", **LARGE, "tokens": 65000, "page": 16, "layers": 1,
         "pad": 17, "graph": False},
        # one request's decode step: launches and latency
        {"name": "attn_decode_1", "kind": "attn", **SMALL, "batch": 1, "q": 1, "lo": 300, "hi": 400,
         "lens": 1, "page": 16, "layers": 24, "graph": True},
        # the verify step of 32 requests, 4 drafts and the bonus token
        {"name": "attn_verify_32", "kind": "attn", **SMALL, "batch": 32, "q": 5, "lo": 100,
         "hi": 640, "lens": 2, "page": 16, "layers": 24, "graph": True},
        # verify over long contexts, 8 drafts: the KV stream
        {"name": "attn_verify_long", "kind": "attn", **LARGE, "batch": 64, "q": 9, "lo": 2048,
         "hi": 8192, "lens": 3, "page": 16, "layers": 1, "graph": False},
        # chunks of long prompts over what is cached of them
        {"name": "attn_chunk", "kind": "attn", **LARGE, "batch": 4, "q": 1000, "lo": 2048,
         "hi": 8192, "lens": 4, "page": 16, "layers": 1, "graph": False},
        # two prompts sampled a few times each: short prefixes, few rows
        {"name": "prefix_few", "kind": "prefix", **SMALL, "batch": 6, "groups": 2, "q": 5,
         "plo": 700, "phi": 1100, "lo": 20, "hi": 200, "lens": 5, "page": 16, "layers": 24,
         "fp8": False, "graph": True},
        # decode of 32 requests behind one system prompt
        {"name": "prefix_decode_32", "kind": "prefix", **LARGE, "batch": 32, "groups": 1, "q": 1,
         "plo": 4001, "phi": 4001, "lo": 50, "hi": 500, "lens": 6, "page": 16, "layers": 4,
         "fp8": False, "graph": True},
        # verify of 64 requests behind one long document, 8-bit pool
        {"name": "prefix_verify_64", "kind": "prefix", **LARGE, "batch": 64, "groups": 1, "q": 9,
         "plo": 8192, "phi": 8192, "lo": 100, "hi": 1000, "lens": 7, "page": 16, "layers": 1,
         "fp8": True, "graph": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attn", "attn", "attn", "prefix", "prefix",
                       "prefix"])
    heads = rng.choice([SMALL, LARGE, SMALL, LARGE, MHA, MQA])
    page = rng.choice([16, 16, 32, 8, 1, 64])
    lens = rng.randrange(1 << 20)
    if kind in ("rope", "write", "read"):
        tokens = _log_int(rng, 1, 65000 if kind == "read" else 16384)
        layers = 4 if tokens < 300 and kind != "read" else 1
        return {"kind": kind, **heads, "tokens": tokens, "page": page, "layers": layers,
                "pad": rng.choice([0, 0, rng.randint(1, 20)]), "graph": layers > 1}
    if kind == "attn":
        if rng.random() < 0.25:               # a chunk of each prompt, or all of it
            hi = _log_int(rng, 32, 8192)
            q = _log_int(rng, 16, min(hi, 1000))
            batch = _log_int(rng, 1, max(1, min(64, 4000 // q)))
            return {"kind": "attn", **heads, "batch": batch, "q": q, "lo": max(q, hi // 4),
                    "hi": hi, "lens": lens, "page": page, "layers": 1, "graph": False}
        batch, lo = _log_int(rng, 1, 64), _log_int(rng, 9, 2048)
        hi = min(8192, int(lo * rng.uniform(1, 5)))
        layers = min(8, 300_000_000 // (batch * hi * heads["hkv"] * heads["d"]))
        return {"kind": "attn", **heads, "batch": batch, "q": rng.choice([1, 1, 2, 3, 5, 9]),
                "lo": lo, "hi": hi, "lens": lens, "page": page, "layers": max(1, layers),
                "graph": layers > 3}
    groups = rng.choice([1, 1, 2, 3])
    batch = max(groups, _log_int(rng, 2, 64))
    lo = _log_int(rng, 9, 300)
    plo = _log_int(rng, 50, 4000)
    layers = rng.choice([1, 4])
    return {"kind": "prefix", **heads, "batch": batch, "groups": groups,
            "q": rng.choice([1, 1, 2, 5, 9]), "plo": plo, "phi": int(plo * rng.uniform(1, 2)),
            "lo": lo, "hi": int(lo * rng.uniform(1, 3.3)), "lens": lens, "page": page,
            "layers": layers, "fp8": rng.random() < 0.5, "graph": layers > 1}


# ---------------------------------------------------------------- sizes

def _lens(case):
    """(query lengths, own KV lengths, group of each request, prefix lengths);
    for ``attn`` the prefixes are empty."""
    r = random.Random(case["lens"])
    n, q = case["batch"], case["q"]
    kv = [max(r.randint(case["lo"], case["hi"]), q) for _ in range(n)]
    if case["kind"] == "attn":
        return [q] * n, kv, [0] * n, [0]
    g = case["groups"]
    cuts = sorted(r.sample(range(1, n), g - 1)) if g > 1 else []
    group = [sum(b >= c for c in cuts) for b in range(n)]
    return [q] * n, kv, group, [r.randint(case["plo"], case["phi"]) for _ in range(g)]


def work(case):
    hq, hkv, d, L = case["hq"], case["hkv"], case["d"], case["layers"]
    if case["kind"] in ("rope", "write", "read"):
        t, kv = case["tokens"], 2 * case["tokens"] * hkv
        b = kv * d * 3 + kv + 8 * t
        if case["kind"] == "rope":
            b += t * (4 * hq * d + 8) + 4 * d * min(t, 8192)
        return {"bytes": b * L, "flops": (2 * kv + 3 * (case["kind"] == "rope") * t * hq) * d * L}
    ql, kl, group, pl = _lens(case)
    row = 2 * d + 2 if case["kind"] == "attn" or case["fp8"] else 4 * d
    pairs = sum(q * (k + pl[g]) - q * (q - 1) // 2 for q, k, g in zip(ql, kl, group))
    return {"bytes": L * ((sum(kl) + sum(pl)) * hkv * row + 4 * sum(ql) * hq * d),
            "flops": L * 4 * pairs * hq * d}


# ---------------------------------------------------------------- inputs

def _normal(g, *shape, std=1.0):
    out = torch.empty(*shape, dtype=BF16, device=DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV) * std
    return out


def _kv_rows(g, *shape):
    """K or V rows: some channels several times wider than others, and a
    token's magnitude of its own."""
    x = _normal(g, *shape)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV)).to(BF16)
    x *= torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=g, device=DEV)).to(BF16)
    return x


def _quantised(x):
    """Rows as the 8-bit pool holds them: (codes, exponents as integers)."""
    x = x.to(F32)
    amax = x.abs().amax(-1)
    m, p = torch.frexp(amax)                  # amax = m 2^p, 1/2 <= m < 1; 448 = 7/8 2^9
    e = (p - 9 + (m > 0.875).to(p.dtype) + 127).clamp_min(1)
    e = torch.where(amax > 0, e, torch.ones_like(e))
    codes = torch.ldexp(x, (127 - e).unsqueeze(-1)).to(FP8)
    return codes, e


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    hq, hkv, d, P, L = case["hq"], case["hkv"], case["d"], case["page"], case["layers"]
    s = {"case": case}
    if case["kind"] in ("rope", "write", "read"):
        T, pad = case["tokens"], case["pad"]
        pages = -(-T // P) + 9
        slots = torch.randperm(pages * P, generator=cpu)[:T]
        if pad:
            slots[torch.randperm(T, generator=cpu)[:min(pad, T - 1)]] = -1
        s["slots"] = slots.to(DEV)
        s["kept"] = (slots >= 0).nonzero().flatten().to(DEV)
        codes, e = _quantised(_kv_rows(g, L, 2, pages * P, hkv, d))
        s["kc"], s["vc"] = (codes[:, i].reshape(L, pages, P, hkv, d).contiguous() for i in (0, 1))
        s["sc"] = (e.view(L, 2, pages, P, hkv).permute(0, 2, 4, 1, 3).to(torch.uint8)
                   .contiguous())
        if case["kind"] != "read":
            s["qkv"] = torch.cat([_normal(g, L, T, hq * d), _kv_rows(g, L, T, 2 * hkv, d)
                                  .view(L, T, -1)], -1)
        if case["kind"] == "rope":
            n = 8192
            f = 1e6 ** (-torch.arange(0, d, 2, dtype=F64) / d)
            a = torch.outer(torch.arange(n, dtype=F64), f)
            s["cos"], s["sin"] = a.cos().to(F32).to(DEV), a.sin().to(F32).to(DEV)
            s["pos"] = torch.randint(0, n, (T,), generator=cpu).to(DEV)
        return s
    ql, kl, group, pl = _lens(case)
    every = list(kl) + (pl if case["kind"] == "prefix" else [])
    need = [-(-n // P) for n in every]
    pages = sum(need) + 5
    perm = torch.randperm(pages, generator=cpu)[:sum(need)].to(torch.int32)
    tables = list(perm.split(need))
    n = len(kl)
    s["tables"], s["prefix_tables"] = tables[:n], tables[n:]
    s["lens"] = (ql, kl, group, pl)
    s["q"] = _normal(g, L, sum(ql), hq, d)
    if case["kind"] == "prefix" and not case["fp8"]:
        s["kc"], s["vc"] = (_kv_rows(g, L, pages, P, hkv, d) for _ in range(2))
        s["sc"] = None
    else:
        kc, ke = _quantised(_kv_rows(g, L, pages, P, hkv, d))
        vc, ve = _quantised(_kv_rows(g, L, pages, P, hkv, d))
        s["kc"], s["vc"] = kc, vc
        s["sc"] = torch.stack([ke, ve], -1).permute(0, 1, 3, 4, 2).to(torch.uint8).contiguous()
    return s


def _csr(tables, lens, P):
    i32 = torch.int32
    ptr = [0]
    for t in tables:
        ptr.append(ptr[-1] + len(t))
    idx = torch.cat(tables).to(i32) if ptr[-1] else torch.zeros(0, dtype=i32)
    last = [(m - 1) % P + 1 if m else 0 for m in lens]
    return torch.tensor(ptr, dtype=i32), idx, torch.tensor(last, dtype=i32)


def _padded(tables, lens, P):
    """Flat slots (tables, longest length) of every position, short tables
    padded with their own slot 0."""
    out = torch.zeros(len(tables), max(max(lens), 1), dtype=torch.int64)
    for i, (t, m) in enumerate(zip(tables, lens)):
        j = torch.arange(m)
        out[i, :m] = t.long()[j // P] * P + j % P
        out[i, m:] = out[i, 0]
    return out.to(DEV)


def prepare(case, seed):
    s = _inputs(case, seed)
    L, P = case["layers"], case["page"]
    if case["kind"] in ("attn", "prefix"):
        ql, kl, group, pl = s["lens"]
        heads = (case["hq"], case["hkv"], case["d"])
        s["o"] = torch.empty_like(s["q"])
        # index tables of the plain form
        s["rows"], s["kl"] = _padded(s["tables"], kl, P), torch.tensor(kl, device=DEV)
        if case["kind"] == "prefix":
            s["prows"], s["pl"] = (_padded(s["prefix_tables"], pl, P),
                                   torch.tensor(pl, device=DEV))
            size = [group.count(i) for i in range(len(pl))]
            first = [group.index(i) for i in range(len(pl))]
            s["members"] = torch.tensor([[f + min(j, m - 1) for j in range(max(size))]
                                         for f, m in zip(first, size)], device=DEV)
            s["group"] = torch.tensor(group, device=DEV)
            s["place"] = torch.tensor([b - first[x] for b, x in enumerate(group)], device=DEV)
        if own:
            from nanosglang_amd import kernels
            qo = torch.tensor([i * case["q"] for i in range(len(ql) + 1)], dtype=torch.int32)
            ptr, idx, last = _csr(s["tables"], kl, P)
            ws = torch.empty(256 << 20, dtype=torch.uint8, device=DEV)
            if case["kind"] == "attn":
                s["wrapper"] = kernels.BatchPrefillWithPagedKVCacheWrapper(ws, "NHD")
                s["wrapper"].plan(qo, ptr, idx, last, *heads, P, causal=True, kv_data_type=FP8)
            else:
                pptr, pidx, plast = _csr(s["prefix_tables"], pl, P)
                groups = torch.tensor([group.index(i) for i in range(len(pl))] + [len(kl)],
                                      dtype=torch.int32)
                s["wrapper"] = kernels.SharedPrefixAttentionWrapper(ws, "NHD")
                s["wrapper"].plan(qo, groups, pptr, pidx, plast, ptr, idx, last, *heads, P,
                                  causal=True, kv_data_type=FP8 if case["fp8"] else BF16)
    elif case["kind"] == "rope":
        s["o"] = torch.empty(L, case["tokens"], case["hq"], case["d"], dtype=BF16, device=DEV)
    if own and case["graph"]:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _own(s)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["out"] = _own(s)
    return s


# ---------------------------------------------------------------- the framework's calls

def _own(s):
    from nanosglang_amd import kernels
    case = s["case"]
    kind, L, hq, hkv, d = (case[n] for n in ("kind", "layers", "hq", "hkv", "d"))
    if kind == "read":
        return kernels.kv_read_fp8(s["slots"], s["kc"][0], s["vc"][0], s["sc"][0])
    if kind == "write":
        for i in range(L):
            k, v = s["qkv"][i].view(-1, hq + 2 * hkv, d)[:, hq:].split(hkv, 1)
            kernels.kv_write_fp8(k, v, s["slots"], s["kc"][i], s["vc"][i], s["sc"][i])
        return s["kc"], s["vc"], s["sc"]
    if kind == "rope":
        for i in range(L):
            kernels.rope_kv_write_fp8(s["qkv"][i], hq, hkv, d, s["pos"], s["cos"], s["sin"],
                                      s["slots"], s["kc"][i], s["vc"][i], s["sc"][i],
                                      q_out=s["o"][i])
        return s["o"], s["kc"], s["vc"], s["sc"]
    for i in range(L):
        s["wrapper"].run(s["q"][i], (s["kc"][i], s["vc"][i]), out=s["o"][i],
                         kv_scale=None if s["sc"] is None else s["sc"][i])
    return s["o"]


# ---------------------------------------------------------------- plain forms

def _plain_write(s):
    case = s["case"]
    hq, hkv, d, P, L = (case[n] for n in ("hq", "hkv", "d", "page", "layers"))
    x = s["qkv"].view(L, -1, hq + 2 * hkv, d)
    if case["kind"] == "rope":
        # every product and the sum rounded to bf16, as bf16 tensors do
        c, sn = (s[n][s["pos"]].to(BF16).unsqueeze(1) for n in ("cos", "sin"))
        a, b = x[:, :, :hq + hkv].chunk(2, -1)
        x = torch.cat([torch.cat([a * c - b * sn, b * c + a * sn], -1), x[:, :, hq + hkv:]], 2)
        s["o"].copy_(x[:, :, :hq])
    codes, e = _quantised(x[:, s["kept"], hq:])
    at = s["slots"][s["kept"]]
    s["kc"].view(torch.uint8).view(L, -1, hkv, d)[:, at] = codes[:, :, :hkv].view(torch.uint8)
    s["vc"].view(torch.uint8).view(L, -1, hkv, d)[:, at] = codes[:, :, hkv:].view(torch.uint8)
    s["sc"].permute(0, 1, 4, 2, 3)[:, at // P, at % P] = (
        e.view(L, -1, 2, hkv).transpose(2, 3).to(torch.uint8))
    pools = s["kc"], s["vc"], s["sc"]
    return (s["o"], *pools) if case["kind"] == "rope" else pools


def _rows(s, rows):
    """K and V of flat slots (tables, length) in 32 bits:
    (layers, tables, Hkv, length, D) each."""
    L, hkv, d = s["case"]["layers"], s["case"]["hkv"], s["case"]["d"]
    k, v = (s[n].view(torch.uint8 if s["sc"] is not None else BF16).view(L, -1, hkv, d)[:, rows]
            for n in ("kc", "vc"))
    if s["sc"] is not None:
        e = s["sc"].permute(0, 1, 4, 2, 3).flatten(1, 2)[:, rows].to(torch.int32) - 127
        k = torch.ldexp(k.view(FP8).to(F32), e[..., 0].unsqueeze(-1))
        v = torch.ldexp(v.view(FP8).to(F32), e[..., 1].unsqueeze(-1))
    return (x.to(F32).transpose(2, 3).contiguous() for x in (k, v))


def _plain_read(s):
    case = s["case"]
    k, v = _rows(s, s["slots"].clamp_min(0).unsqueeze(0))
    ok = (s["slots"] >= 0).view(-1, 1, 1)
    return tuple(torch.where(ok, x[0, 0].transpose(0, 1), 0.0).to(BF16) for x in (k, v))


def _plain_attn(s):
    case = s["case"]
    L, hq, hkv, d, n, ql = (case[k] for k in ("layers", "hq", "hkv", "d", "batch", "q"))
    G = hq // hkv
    # (layers, requests, KV heads, query tokens x heads of the group, D)
    q = (s["q"].to(F32).view(L, n, ql, hkv, G, d).permute(0, 1, 3, 2, 4, 5)
         .reshape(L, n, hkv, ql * G, d))
    k, v = _rows(s, s["rows"])
    score = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    j = torch.arange(k.shape[3], device=DEV)
    seen = s["kl"].view(n, 1) - ql + torch.arange(ql, device=DEV).repeat_interleave(G)
    score.masked_fill_((j > seen.unsqueeze(-1)).view(1, n, 1, ql * G, -1), -math.inf)
    if case["kind"] == "prefix":
        kp, vp = _rows(s, s["prows"])
        groups, most = s["members"].shape
        # the group's queries side by side: one product with its prefix
        qg = (q[:, s["members"]].transpose(2, 3).reshape(L, groups, hkv, most * ql * G, d))
        sp = torch.matmul(qg, kp.transpose(-1, -2)) * d ** -0.5
        j = torch.arange(kp.shape[3], device=DEV)
        sp.masked_fill_((j >= s["pl"].view(groups, 1)).view(1, groups, 1, 1, -1), -math.inf)
        sp = (sp.view(L, groups, hkv, most, ql * G, -1).transpose(2, 3)[:, s["group"], s["place"]])
        score = torch.cat([score, sp], -1)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :k.shape[3]], v)
    if case["kind"] == "prefix":
        pp = p[..., k.shape[3]:][:, s["members"]].transpose(2, 3)
        op = torch.matmul(pp.reshape(L, groups, hkv, most * ql * G, -1), vp)
        o += (op.view(L, groups, hkv, most, ql * G, d).transpose(2, 3)[:, s["group"], s["place"]])
    o = (o / total).view(L, n, hkv, ql, G, d).permute(0, 1, 3, 2, 4, 5)
    return o.reshape(L, n * ql, hq, d).to(BF16)


def run(state):
    if own:
        if "graph" in state:
            state["graph"].replay()
            return state["out"]
        return _own(state)
    kind = state["case"]["kind"]
    if kind in ("rope", "write"):
        return _plain_write(state)
    return _plain_read(state) if kind == "read" else _plain_attn(state)


# ---------------------------------------------------------------- 64 bits

def _values(codes, exps):
    """What codes and exponents stand for."""
    return codes.to(F32).to(F64) * torch.pow(torch.tensor(2.0, dtype=F64, device=DEV),
                                             exps.to(F64) - 127)


def exact(case, seed):
    s = _inputs(case, seed)
    hq, hkv, d, P, L = (case[n] for n in ("hq", "hkv", "d", "page", "layers"))
    if case["kind"] == "read":
        out = []
        for i, pool in enumerate((s["kc"][0], s["vc"][0])):
            x = _values(pool, s["sc"][0][:, :, i].transpose(1, 2).unsqueeze(-1))
            x = x.reshape(-1, hkv, d)[s["slots"]]
            out.append(torch.where((s["slots"] < 0).view(-1, 1, 1), torch.zeros_like(x), x))
        return tuple(out)
    if case["kind"] in ("rope", "write"):
        x = s["qkv"].to(F64).view(L, -1, hq + 2 * hkv, d)
        if case["kind"] == "rope":
            turned = hq + hkv
            z = torch.complex(x[:, :, :turned, :d // 2], x[:, :, :turned, d // 2:])
            w = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[s["pos"]]
            z = z * w[:, None]
            x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, :, turned:]], 2)
        kept = (s["slots"] >= 0)
        at = s["slots"][kept]
        pools = []
        for i, pool in enumerate((s["kc"], s["vc"])):
            rows = x[:, kept][:, :, hq + i * hkv:hq + (i + 1) * hkv]
            # e4m3 has no 64-bit values: the row over its scale, unrounded
            top = rows.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -118)
            e = torch.ceil(torch.log2(top / 448)).clamp_min(-126)
            p = pool.to(F32).to(F64).view(L, -1, hkv, d)
            p[:, at] = rows * torch.pow(torch.tensor(2.0, dtype=F64, device=DEV), -e)
            pools.append(p.view(pool.shape))
        pools.append(None)
        return (x[:, :, :hq], *pools) if case["kind"] == "rope" else tuple(pools)
    ql, kl, group, pl = s["lens"]
    out = torch.empty(L, sum(ql), hq, d, dtype=F64, device=DEV)
    for i in range(L):
        t0 = 0
        for b, (nq, nk) in enumerate(zip(ql, kl)):
            spans = [(s["tables"][b], nk)]
            if case["kind"] == "prefix":
                spans.insert(0, (s["prefix_tables"][group[b]], pl[group[b]]))
            ks, vs = [], []
            for table, m in spans:
                ids = table.long().to(DEV)
                for j, (pool, to) in enumerate(((s["kc"], ks), (s["vc"], vs))):
                    x = pool[i][ids] if s["sc"] is None else _values(
                        pool[i][ids], s["sc"][i][ids][:, :, j].transpose(1, 2).unsqueeze(-1))
                    to.append(x.to(F64).reshape(-1, hkv, d)[:m])
            k, v = torch.cat(ks), torch.cat(vs)
            sight = k.shape[0] - nq + torch.arange(nq, device=DEV)
            hidden = torch.arange(k.shape[0], device=DEV)[None] > sight[:, None]
            for h in range(hq):
                z = s["q"][i, t0:t0 + nq, h].to(F64) @ k[:, h // (hq // hkv)].T / math.sqrt(d)
                z[hidden] = -math.inf
                out[i, t0:t0 + nq, h] = torch.softmax(z, -1) @ v[:, h // (hq // hkv)]
            t0 += nq
    return out
