"""The 8-bit pool as the model and the speculative engine use it, and a run of
its operators together."""
import numpy as np
import pytest
import torch

from oracle import kv_fp8
from tests import _fp8_cases as fc
from tests.test_gpu_model import TINY, _tiny_models

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
Hq, Hkv, D, P = 4, 2, 64, 16          # TINY's


def _manager(blocks=64, layers=4):
    from nanosglang_amd.engine.paged_kv_cache import BlockManager, PagedKVCache
    bm = BlockManager(blocks, P, layers, Hkv, D, FP8, "cuda", row_scales=True)
    return bm, PagedKVCache(bm)


def _ws(mb=32):
    return torch.empty(mb << 20, dtype=torch.uint8, device="cuda")


def _values(bm, li):
    return fc.values(*(t[li].view(torch.uint8).cpu().numpy() for t in bm.caches))


def test_block_manager_writes_and_reads_rows():
    bm, kv = _manager(layers=2)
    t = kv.allocate_for_request(40)
    rng = np.random.default_rng(0)
    x = [fc.rows(rng, Hkv, 40, D, spread=2.0) for _ in range(2)]
    d = [torch.from_numpy(a).cuda().bfloat16() for a in x]
    for i, at in enumerate(range(0, 40, P)):
        n = min(P, 40 - at)
        bm.write_kv(t.block_indices[i], 1, 0, *(a[:, at:at + n] for a in d))
    kv.write_kv_token(t, 1, 40, *(a[:, :1] for a in d))          # token 40: the first again
    got = kv.get_kv_for_attention(t, 1, 41)
    for a, g, is_v in zip(x, got, (False, True)):
        want = kv_fp8.dequantise(*kv_fp8.quantise(np.concatenate([a, a[:, :1]], 1), is_v))
        assert np.array_equal(g.double().cpu().numpy(), want)
    for g in kv.get_kv_for_attention(t, 0, 41):                  # the other layer: untouched
        assert not g.any()


class _Checked:
    """An attention wrapper that checks every layer's output against 64-bit
    attention over the values that the pool then stands for."""

    def __init__(self, w, tables, q_lens, kv_lens):
        self.w, self.tables, self.q_lens, self.kv_lens, self.runs = w, tables, q_lens, kv_lens, 0

    def run(self, q, cache, kv_scale=None):
        out = self.w.run(q, cache, kv_scale=kv_scale)
        k, v = fc.values(*(t.view(torch.uint8).cpu().numpy() for t in (*cache, kv_scale)))
        spans = [tuple(x[t].reshape(-1, Hkv, D)[:n] for x in (k, v))
                 for t, n in zip(self.tables, self.kv_lens)]
        fc.check(out, *fc.attention(q.double().cpu().numpy(), spans, self.q_lens))
        self.runs += 1
        return out


def _row_bound(x):
    """How far a row of the pool may lie from the bf16 path's row x: e4m3's half
    step (2^-4 of a value, 2^-10 of the scale below its normal range; the scale is
    at most amax / 224), and the projection's sums in another order: one bf16
    step, 2^-7, of each of two products of RoPE and their sum, all below
    sqrt(2) amax, so 6 * 2^-7 amax with room for the quantiser's 2^-4 of it."""
    amax = np.abs(x).max(-1, keepdims=True)
    return 2.0 ** -4 * np.abs(x) + amax * (2.0 ** -10 / 224 + 6 * 2.0 ** -7) + 1e-30


@pytest.mark.parametrize("lens", [(40, 7, 129), (40, 7, 29)])
def test_packed_forward_over_the_8_bit_pool(lens):
    """176 rows take the separate norms, 76 the folded ones; then a decode step.
    Layer 0's rows are the bf16 path's, quantised; every layer's attention is
    checked over what its pool holds."""
    from nanosglang_amd.engine.paged_kv_cache import BlockManager
    from nanosglang_amd.kernels import BatchPrefillWithPagedKVCacheWrapper
    _, gpu = _tiny_models(1.0)
    rng = np.random.default_rng(0)
    bm, kv = _manager()
    ref = BlockManager(64, P, 4, Hkv, D, torch.bfloat16, "cuda")
    tables = [kv.allocate_for_request(n + 1) for n in lens]
    starts = [0] * len(lens)
    for q_lens in (list(lens), [1] * len(lens)):
        ends = [s + n for s, n in zip(starts, q_lens)]
        used = [t.block_indices[:-(-n // P)] for t, n in zip(tables, ends)]
        qo = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        ptr, idx, last = fc.csr(used, ends, P)
        dev = lambda x: torch.from_numpy(np.concatenate(x)).cuda()
        ids = dev([rng.integers(0, 1000, n) for n in q_lens])
        pos = dev([np.arange(s, e) for s, e in zip(starts, ends)])
        slots = dev([np.asarray(kv.slots(t, s, n)) for t, s, n in zip(tables, starts, q_lens)])
        w = BatchPrefillWithPagedKVCacheWrapper(_ws())
        w.plan(qo, ptr, idx, last, Hq, Hkv, D, P, kv_data_type=FP8)
        chk = _Checked(w, used, q_lens, ends)
        got = gpu.forward_packed(ids, pos, bm.caches, chk, slots)
        assert chk.runs == 4 and torch.isfinite(got.float()).all()
        w2 = BatchPrefillWithPagedKVCacheWrapper(_ws())
        w2.plan(qo, ptr, idx, last, Hq, Hkv, D, P)
        gpu.forward_packed(ids, pos, ref.caches, w2, slots)
        s = slots.cpu().numpy()
        for mine, bf in zip(_values(bm, 0), (ref.k_cache, ref.v_cache)):
            x = bf[0].double().cpu().numpy().reshape(-1, Hkv, D)[s]
            assert (np.abs(mine.reshape(-1, Hkv, D)[s] - x) <= _row_bound(x)).all()
        starts = ends


def test_packed_forward_behind_a_shared_prefix():
    """A prompt forward writes the prefix once; two requests then decode behind it."""
    from nanosglang_amd.kernels import (BatchPrefillWithPagedKVCacheWrapper,
                                        SharedPrefixAttentionWrapper)
    _, gpu = _tiny_models(1.0)
    rng = np.random.default_rng(3)
    bm, kv = _manager()
    n = 3 * P
    pre = kv.allocate_for_request(n)
    own = [kv.allocate_for_request(4) for _ in range(2)]
    w = BatchPrefillWithPagedKVCacheWrapper(_ws())
    w.plan(np.asarray([0, n]), *fc.csr([pre.block_indices], [n], P), Hq, Hkv, D, P,
           kv_data_type=FP8)
    gpu.forward_packed(torch.from_numpy(rng.integers(0, 1000, n)).cuda(),
                       torch.arange(n, device="cuda"), bm.caches, w,
                       torch.tensor(kv.slots(pre, 0, n), device="cuda"))
    ws = SharedPrefixAttentionWrapper(_ws(64))
    for step in range(3):
        ids = torch.from_numpy(rng.integers(0, 1000, 2)).cuda()
        pos = torch.full((2,), n + step, device="cuda")
        slots = torch.tensor([kv.slots(t, step, 1)[0] for t in own], device="cuda")
        tabs = [t.block_indices for t in own]
        ws.plan(np.asarray([0, 1, 2]), np.asarray([0, 2]), *fc.csr([pre.block_indices], [n], P),
                *fc.csr(tabs, [step + 1] * 2, P), Hq, Hkv, D, P, kv_data_type=FP8)
        chk = _Checked(ws, [pre.block_indices + t for t in tabs], [1, 1], [n + step + 1] * 2)
        gpu.forward_packed(ids, pos, bm.caches, chk, slots)
        assert chk.runs == 4 and ws.check_flags() == 0


@pytest.mark.parametrize("T,fold", [(1, False), (37, False), (160, False), (400, False),
                                    (1, True), (37, True), (160, True)])   # folds: up to 160
def test_projection_into_the_8_bit_pool(T, fold):
    """linear_rope_kv's pool is the bf16 one's rows, quantised, and its q the same."""
    from nanosglang_amd import kernels
    g = torch.Generator().manual_seed(T)
    K, pages = 256, 30
    x = torch.randn(T, K, generator=g).bfloat16().cuda()
    wt = (torch.randn((Hq + 2 * Hkv) * D, K, generator=g) / 16).bfloat16().cuda()
    pos = torch.randint(0, 64, (T,), generator=g).cuda()
    ang = torch.rand(64, D // 2, generator=g).cuda()
    slots = torch.randperm(pages * P, generator=g)[:T].cuda()
    slots[T // 2] = -1
    kw = dict(sumsq_in=kernels.row_sumsq(x)) if fold else {}
    args = (x, wt, None, Hq, Hkv, D, pos, ang.cos(), ang.sin(), slots)
    bf = [torch.zeros(pages, P, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    q = kernels.linear_rope_kv(*args, *bf, **kw)
    pool = [torch.zeros(pages, P, Hkv, D, dtype=torch.uint8, device="cuda").view(FP8)
            for _ in range(2)] + [torch.zeros(pages, Hkv, 2, P, dtype=torch.uint8, device="cuda")]
    assert torch.equal(q, kernels.linear_rope_kv(*args, *pool[:2], kv_scale=pool[2], **kw))
    vals = fc.values(*(t.view(torch.uint8).cpu().numpy() for t in pool))
    for x_, v in zip(bf, vals):
        want = kv_fp8.dequantise(*kv_fp8.quantise(x_.double().cpu().numpy(), x_ is bf[1]))
        assert np.array_equal(v, want)


@pytest.mark.parametrize("heads", [(14, 2, 64), (32, 8, 128)])
def test_the_operators_together(heads):
    """Prompts written, decode steps rotated and written, attended to behind a
    shared prefix, rolled back, and read again: the q and the pool that each
    operator leaves are the next one's inputs."""
    from nanosglang_amd import kernels
    hq, hkv, d = heads
    rng = np.random.default_rng(hq)
    pages, n_pre, own = 24, 85, [3, 17, 40]
    pool = (torch.zeros(pages, P, hkv, d, dtype=torch.uint8, device="cuda").view(FP8),
            torch.zeros(pages, P, hkv, d, dtype=torch.uint8, device="cuda").view(FP8),
            torch.zeros(pages, hkv, 2, P, dtype=torch.uint8, device="cuda"))
    lens = [n_pre] + [n + 6 for n in own]
    tabs = fc.tables(rng, lens, P, pages)
    slot = lambda t, i: t[i // P] * P + i % P
    for t, n in zip(tabs, [n_pre] + own):
        s = torch.tensor([slot(t, i) for i in range(n)], device="cuda")
        k, v = (torch.from_numpy(fc.rows(rng, n, hkv, d)).cuda().bfloat16() for _ in range(2))
        kernels.kv_write_fp8(k, v, s, *pool)
    ang = torch.from_numpy(rng.uniform(0, 6, (256, d // 2)).astype(np.float32)).cuda()
    w = kernels.SharedPrefixAttentionWrapper(_ws(64))
    for step, q_len in enumerate((1, 5, 2)):             # 5 drafts: all but 1 rolled back after
        ends = [n + q_len for n in own]
        qkv = torch.from_numpy(rng.standard_normal((3 * q_len, (hq + 2 * hkv) * d))).cuda().bfloat16()
        pos = torch.tensor([n_pre + n + i for n in own for i in range(q_len)], device="cuda")
        s = torch.tensor([slot(t, n + i) for t, n in zip(tabs[1:], own) for i in range(q_len)],
                         device="cuda")
        q = kernels.rope_kv_write_fp8(qkv, hq, hkv, d, pos, ang.cos(), ang.sin(), s, *pool)
        w.plan(np.arange(4) * q_len, np.asarray([0, 3]), *fc.csr(tabs[:1], [n_pre], P),
               *fc.csr([t[:-(-n // P)] for t, n in zip(tabs[1:], ends)], ends, P), hq, hkv, d, P,
               kv_data_type=FP8)
        out = w.run(q, pool[:2], kv_scale=pool[2])
        spans = []
        for t, n in zip(tabs[1:], ends):
            at = [slot(tabs[0], i) for i in range(n_pre)] + [slot(t, i) for i in range(n)]
            spans.append([x.double().cpu().numpy() for x in
                          kernels.kv_read_fp8(torch.tensor(at, device="cuda"), *pool)])
        fc.check(out, *fc.attention(q.double().cpu().numpy(), spans, [q_len] * 3))
        own = [n + (1 if q_len == 5 else q_len) for n in own]


def _engine(gpu, **kw):
    from nanosglang_amd.engine.spec_engine import SpecEngine
    return SpecEngine(gpu, draft_layers=2, num_speculative=4, num_blocks=64, max_batch=4,
                      kv_dtype=FP8, **kw)


@pytest.mark.parametrize("graphs", [True, False])
def test_engine_over_the_8_bit_pool(graphs):
    """Every emitted token is the argmax of the step's own verify logits; layer
    0's pool rows are those of one forward over the finished sequences (both
    within the quantiser's bound of the bf16 row, hence twice it of each
    other); pages go back."""
    from nanosglang_amd.engine.paged_kv_cache import BlockManager
    from nanosglang_amd.kernels import BatchPrefillWithPagedKVCacheWrapper
    _, gpu = _tiny_models()
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (20, 33, 5)]
    max_new = [18, 12, 25]
    eng = _engine(gpu, use_graphs=graphs, pipeline=False)
    eng.trace = []
    held = []
    free = eng.kv.free_request
    bm = eng.bm
    eng.kv.free_request = lambda t: (held.append((list(t.block_indices), _values(bm, 0))),
                                     free(t))
    out = eng.generate(prompts, max_new)
    del eng.kv.free_request              # (no cycle that keeps the engine's graphs alive)
    assert [len(o) for o in out] == max_new
    assert eng.bm.num_free_blocks == 64 - graphs
    assert eng.trace
    for rec in eng.trace:
        top = rec["verify_logits"].float().argmax(-1).numpy()
        for b, n in enumerate(rec["num_emitted"]):
            assert np.array_equal(rec["emitted"][b, :n], top[b, :n])
    assert len(held) == 3
    seqs = [p + o[:-1] for p, o in zip(prompts, out)]     # the last token was never fed back
    for pages, vals in held:
        fits = []
        for seq in seqs:
            n = len(seq)
            if len(pages) < -(-n // P):
                continue
            ref = BlockManager(8, P, 4, Hkv, D, torch.bfloat16, "cuda")
            w = BatchPrefillWithPagedKVCacheWrapper(_ws())
            w.plan(np.asarray([0, n]), *fc.csr([list(range(-(-n // P)))], [n], P), Hq, Hkv, D, P)
            gpu.forward_packed(torch.tensor(seq, device="cuda"), torch.arange(n, device="cuda"),
                               ref.caches, w, torch.arange(n, device="cuda"), num_layers=1)
            ok = True
            for mine, bf in zip(vals, (ref.k_cache, ref.v_cache)):
                x = bf[0].double().cpu().numpy().reshape(-1, Hkv, D)[:n]
                ok &= bool((np.abs(mine[pages].reshape(-1, Hkv, D)[:n] - x) <= _row_bound(x)).all())
            fits.append(ok)
        assert any(fits)


@pytest.mark.parametrize("dtype", [torch.bfloat16, FP8])
def test_pipelined_steps_of_eight_drafts(dtype):
    """More attention calls than one gate copies ranges for."""
    from nanosglang_amd.engine.spec_engine import SpecEngine
    _, gpu = _tiny_models(1.0)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (20, 33)]
    outs = [SpecEngine(gpu, draft_layers=4, num_speculative=8, num_blocks=64, max_batch=2,
                       kv_dtype=dtype, pipeline=p).generate(prompts, [40, 25])
            for p in (True, False)]
    assert outs[0] == outs[1]


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_pipelined_steps_over_the_8_bit_pool(temperature):
    _, gpu = _tiny_models(1.0)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 1000, n).tolist() for n in (20, 33, 5)]
    outs = [_engine(gpu, pipeline=p, temperature=temperature, seed=7).generate(prompts, [15, 9, 21])
            for p in (True, False)]
    assert outs[0] == outs[1]


def test_synthetic_contexts_fill_the_8_bit_pool():
    _, gpu = _tiny_models(1.0)
    eng = _engine(gpu)
    eng.prefill([[1] * 40, [2] * 20], synthetic_context=True)
    for x in _values(eng.bm, 3):
        assert 0.9 < x.std() < 1.1


def test_other_types_of_pool_are_refused():
    from nanosglang_amd.engine.spec_engine import SpecEngine
    _, gpu = _tiny_models(1.0)
    with pytest.raises(NotImplementedError, match="kv_data_type"):
        SpecEngine(gpu, draft_layers=2, num_speculative=4, num_blocks=64,
                   kv_dtype=torch.float8_e5m2)
