"""Calls on the paged cache and draft verification that their documentation allows and that lie at its edges: packed tokens that no row
owns, rope tables of any angles and too short ones, what is kept of weights and rotated keys, signed zeros, caches in the
reference mode, refusals. Bounds are the ones at the head of `test_paged.py`, named there term by term."""

import math

import numpy as np
import pytest
import torch

from gdn_hybrid_architecture_ideas_b200 import ops
from gdn_hybrid_architecture_ideas_b200.ops import paged as pg
from tests.test_paged import E4M3, _batch, _check_attention, _dense_attention, _random_cache, _status_clean, _tables, _values


def _poison(shape, value=7.0):
    """Free blocks of the allocator that hold `value`: what an output that nobody writes would show."""
    held = [torch.full(shape, value, dtype=torch.bfloat16, device="cuda") for _ in range(64)]
    torch.cuda.synchronize()
    del held


# ------------------------------------------------------------------------------------------------------------ tokens that no row owns

@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd", [("fp4", 64), ("bf16", 64), ("bf16", 256)])
@pytest.mark.parametrize("lead,tail", [(2, 0), (0, 3), (5, 40), (300, 0)])
def test_tokens_before_the_first_row_are_zeros(fmt, hd, lead, tail):
    """A group of rows beside the whole packed q (as of q_start[lo:hi + 1]): the tokens before and behind the group are zeros as in the statement, the
    group's are what a call that writes into `out` gives, and there the others stay."""
    rows, page = [(20, 1, 0), (33, 3, 4), (0, 0, 0), (9, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, fmt)
    q_start, total = q_start + lead, lead + n + tail
    q = torch.randn(total, 8, hd).bfloat16()
    args = [t.cuda() for t in (pages, q_start, lens)]
    _poison((total, 8, hd))
    got = ops.paged_attention(q.cuda(), cache, *args, start=start.cuda())
    out = torch.full((total, 8, hd), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q.cuda(), cache, *args, start=start.cuda(), out=out)
    mine = slice(lead, lead + n)
    assert torch.equal(got[mine], out[mine]) and bool((out[:lead] == 3).all()) and bool((out[lead + n:] == 3).all())
    assert not got[:lead].any() and not got[lead + n:].any()
    want = ops.paged_attention(q, cpu, pages, q_start, lens, start=start)
    assert not want[:lead].any() and not want[lead + n:].any()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, None, None, page=page, got=got)


@pytest.mark.gpu
@pytest.mark.parametrize("q_start,owned", [([0, 1, 3, 9], [0, 1, 2]), ([2, 4, 0, 1], [0, 2, 3]), ([-3, 1, 3, 4], [1, 2, 3]), ([0, 9, 3, 4], [3]), ([5, 6, 8, 9], [])])
def test_tokens_of_refused_rows_are_zeros(q_start, owned):
    """Ranges out of order, negative or behind the packed tokens: status 301, zeros for every token that no accepted row owns, the others as
    with an `out`, in which the rest stays."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page, n = [(20, 1, 0), (33, 2, 0), (9, 1, 0)], 16, 5
    pages, _, lens, _, _, n_pages = _batch(rows, page)
    cache, _ = _random_cache(n_pages, page, 2, 64, "fp4")
    q = torch.randn(n, 8, 64, device="cuda").bfloat16()
    args = pages.cuda(), torch.tensor(q_start, dtype=torch.int32, device="cuda"), lens.cuda()
    _poison((n, 8, 64))
    got = ops.paged_attention(q, cache, *args)
    with pytest.raises(RuntimeError, match="status 301"):
        native.check_status()
    out = torch.full((n, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(q, cache, *args, out=out)
    with pytest.raises(RuntimeError, match="status 301"):
        native.check_status()
    rest = [j for j in range(n) if j not in owned]
    assert torch.equal(got[owned], out[owned]) and not got[rest].any() and bool((out[rest] == 3).all())
    assert all(bool(got[j].any()) for j in owned)


# ------------------------------------------------------------------------------------------------------------ rope tables

def _any_rows(n, pairs, seed=0):
    """A rope table whose rows are rotations by any angles: nothing relates one to another."""
    ang = torch.rand(n, pairs, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 2 * math.pi
    return ang.cos().float(), ang.sin().float()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("hd,group,rot,cap,page,qdt", [(64, 4, 16, 20, 16, "bf16"), (64, 8, 64, 33, 8, "bf16"), (64, 3, 32, 1, 64, "fp32"), (128, 5, 32, 40, 64, "bf16"),
                                                       (128, 2, 64, 300, 16, "fp32"), (256, 8, 64, 100, 16, "bf16"), (256, 1, 16, 7, 32, "bf16")])
def test_capped_scores_take_the_tables_rows_as_they_are(fmt, hd, group, rot, cap, page, qdt):
    """R(p)q . R(t)k with the table's rows at p and t, R(C)q . k beyond the cap, whatever the rows are."""
    rows = [(0, 1, 0), (37, 5, 9), (0, 0, 0), (250, 1, 0), (15, 4, 17), (0, 21, 0), (300, 2, 290)]
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, seed=group)
    cache, cpu = _random_cache(n_pages, page, 2, hd, fmt, seed=rot)
    q = (torch.randn(n, 2 * group, hd) * 1.5).to({"bf16": torch.bfloat16, "fp32": torch.float32}[qdt])
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, _any_rows(310, rot // 2), cap, page=page)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd,new", [("fp4", 64, 2), ("fp4", 128, 1), ("bf16", 64, 1), ("bf16", 256, 3)])
def test_capped_scores_over_many_ctas(fmt, hd, new):
    """The same where rows are cut over many CTAs."""
    rows, page = [(5000, new, 0), (3, new, 0), (2777, new, 1201)], 64
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 1, hd, fmt)
    q = torch.randn(n, 2, hd).bfloat16()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, _any_rows(5100, 16), 700, page=page)


@pytest.mark.parametrize("cap", [None, 7])
def test_capped_statement_takes_the_tables_rows_as_they_are_cpu(cap):
    rows, page, hd = [(37, 5, 9), (0, 1, 0)], 8, 32
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache = pg.PagedKV(*(torch.randn(n_pages, 1, page, hd, dtype=torch.float64) for _ in range(2)))
    cos, sin = (t.double() for t in _any_rows(50, 8))
    q = torch.randn(n, 2, hd, dtype=torch.float64)
    got = ops.paged_attention(q, cache, pages, q_start, lens, start=start, rope=(cos, sin), cap=cap)
    for b, (a, m, c) in enumerate(rows):
        for i in range(m):
            j = int(q_start[b]) + i
            ids, slots = zip(*[(int(pages[b, p // page]), p % page) for p in range(c, a + i + 1)])
            for h in range(2):
                want = _dense_attention(q[j, h].numpy(), cache.k.numpy()[ids, 0, slots], cache.v.numpy()[ids, 0, slots], a + i, c, cos.numpy(), sin.numpy(), cap, hd ** -0.5)[0]
                assert np.abs(got[j, h].numpy() - want).max() < 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd", [("fp4", 64), ("bf16", 64), ("bf16", 128), ("fp4", 256)])
@pytest.mark.parametrize("cap", [None, 10])
@pytest.mark.parametrize("before", [20, 5000])
def test_queries_behind_the_rope_table_are_zeros(fmt, hd, cap, before):
    """Three new tokens of which the last two lie behind the table, a row behind it whole, one inside: status 305; zeros for those, the others
    as with a table that is long enough (rows of 5000 positions are cut over CTAs)."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page = [(before, 3, 0), (before + 30, 1, 0), (9, 1, 0), (before + 30, 1, 40)], 64
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, _ = _random_cache(n_pages, page, 2, hd, fmt)
    q = torch.randn(n, 8, hd, device="cuda").bfloat16()
    args = [t.cuda() for t in (pages, q_start, lens)]
    rope = tuple(t.cuda() for t in _tables(before + 40, 16))
    whole = ops.paged_attention(q, cache, *args, start=start.cuda(), rope=rope, cap=cap)
    _status_clean()
    got = ops.paged_attention(q, cache, *args, start=start.cuda(), rope=tuple(t[:before + 1].contiguous() for t in rope), cap=cap)
    with pytest.raises(RuntimeError, match="status 305"):
        native.check_status()
    assert not got[[1, 2, 3]].any() and torch.equal(got[[0, 4, 5]], whole[[0, 4, 5]])


# ------------------------------------------------------------------------------------------------------------ what is kept of weights and keys

def _bound(o, mass, big, cap):
    """bfloat16 pages: probabilities in two parts 2^-16, queries and rotated keys in two parts 2^-16 each (sqrt 2 for a rotated pair),
    float32 sums and exp2 2^-18; the output's own rounding 2^-8."""
    d = 2.0 ** -16 + big * (2.0 ** -16 * 1.42 * (1 if cap is None else 2) + 2.0 ** -18) + 2.0 ** -18
    return 2.0 ** -8 * np.abs(o) + (math.exp(2 * d) - 1) * 2 * mass * (1 + 2.0 ** -8) + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("odd", [False, True])
def test_bfloat16_pages_keep_the_weights_in_two_parts(hd, odd):
    """Values that cancel in the weighted sum: an error of the weights stands out there. odd: a later token of the row holds NaN, so that its
    tile is summed position by position."""
    for before in (1, 9, 23, 200):
        rows, page = [(before, 2 if odd else 1, 0)], 16
        pages, q_start, lens, start, n, n_pages = _batch(rows, page)
        _, cpu = _random_cache(n_pages, page, 2, hd, "bf16", seed=before)
        q = torch.randn(n, 2, hd).bfloat16()
        at = [(int(pages[0, p // page]), p % page) for p in range(before + 1)]
        ids, slots = np.array([x for x, _ in at]), np.array([y for _, y in at])
        for h in range(2):           # the likeliest position's value makes the sum (nearly) zero
            k, v = cpu.k.double().numpy()[ids, h, slots], cpu.v.double().numpy()[ids, h, slots]
            s = hd ** -0.5 * k @ q[0, h].double().numpy()
            w = np.exp(s - s.max())
            top = int(w.argmax())
            cpu.v[ids[top], h, slots[top]] = torch.from_numpy(-(w @ v - w[top] * v[top]) / w[top]).bfloat16()
        cache = pg.PagedKV(cpu.k.cuda(), cpu.v.cuda())
        if odd:
            cache.v[int(pages[0, (before + 1) // page]), :, (before + 1) % page] = float("nan")
        got = ops.paged_attention(q.cuda(), cache, *(t.cuda() for t in (pages, q_start, lens)))
        _status_clean()
        for h in range(2):
            k, v = cpu.k.double().numpy()[ids, h, slots], cpu.v.double().numpy()[ids, h, slots]
            o, mass, big = _dense_attention(q[0, h].double().numpy(), k, v, before, 0, None, None, None, hd ** -0.5)
            diff = np.abs(got[0, h].double().cpu().numpy() - o)
            assert (diff <= _bound(o, mass, big, None)).all(), (before, h, diff.max())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_an_infinite_value_gives_an_infinite_output(hd):
    """bfloat16 pages, a value of plus or minus infinity in a place that every query sees: that channel is infinite, the others of the slice are finite."""
    rows, page = [(40, 1, 0), (100, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, "bf16")
    for c in (cache, cpu):
        c.v[int(pages[0, 0]), 0, 5, 3], c.v[int(pages[1, 2]), 1, 5, 40] = float("inf"), float("-inf")
    q = torch.randn(n, 4, hd).bfloat16() * 0.2
    got = ops.paged_attention(q.cuda(), cache, *(t.cuda() for t in (pages, q_start, lens))).cpu()
    want = ops.paged_attention(q, cpu, pages, q_start, lens)
    _status_clean()
    assert int(want.isinf().sum()) == 4 and not want.isnan().any()
    odd = want.isinf()
    assert torch.equal(got[odd], want[odd]) and bool(torch.isfinite(got[~odd]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd,rot,page", [(64, 16, 16), (64, 32, 8), (64, 64, 64), (128, 64, 16), (256, 64, 32), (256, 16, 16)])
def test_bfloat16_pages_keep_rotated_keys_in_two_parts(hd, rot, page):
    """Under a cap the keys are rotated while they are scored: large queries along the rotary channels show what the rotated keys lost."""
    rows, cap = [(60, 2, 0), (130, 1, 21)], 50
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, "bf16")
    q = torch.randn(n, 4, hd) * 0.5
    q[..., :rot] *= 12 * (64 / rot) ** 0.5
    q = q.bfloat16()
    rope = _tables(140, rot // 2)
    got = ops.paged_attention(q.cuda(), cache, *(t.cuda() for t in (pages, q_start, lens)), start=start.cuda(), rope=tuple(t.cuda() for t in rope), cap=cap)
    _status_clean()
    kv = [t.double().numpy() for t in _values(cpu)]
    cs = tuple(t.double().numpy() for t in rope)
    for b, (a, m, c) in enumerate(rows):
        for i in range(m):
            at = [(int(pages[b, p // page]), p % page) for p in range(c, a + i + 1)]
            ids, slots = np.array([x for x, _ in at]), np.array([y for _, y in at])
            j = int(q_start[b]) + i
            for h in range(4):
                o, mass, big = _dense_attention(q[j, h].double().numpy(), kv[0][ids, h // 2, slots], kv[1][ids, h // 2, slots], a + i, c, *cs, cap, hd ** -0.5)
                diff = np.abs(got[j, h].double().cpu().numpy() - o)
                assert (diff <= _bound(o, mass, big, cap)).all(), (b, i, h, diff.max())


# ------------------------------------------------------------------------------------------------------------ zeros and their signs

def _bytes(cache):
    return [t.cpu().view(torch.int16 if t.dtype == torch.bfloat16 else torch.uint8) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("rot", [0, 16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_appended_bytes_equal_the_statements_to_the_sign_of_zero(fmt, rot, dtype):
    """Zeros of both signs, values that round to zero, ordinary ones, rotated (by rows with exact zeros and ones too) or not: every byte of the
    cache is the statement's."""
    rows, page, hkv, hd = [(0, 40, 0), (7, 25, 2)], 16, 2, 64
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cpu = pg.PagedKV.zeros(n_pages, page, hkv, hd, fmt)
    gpu = pg.PagedKV.zeros(n_pages, page, hkv, hd, fmt, "cuda")
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(n, hkv, hd, generator=g).to(dtype) for _ in range(2))
    for t in (k, v):
        what = torch.randint(0, 5, t.shape, generator=g)
        t[what == 0], t[what == 1] = 0.0, -0.0
        t[what == 2] *= 2.0 ** -10
    rope = None
    if rot:
        cos, sin = _tables(64, rot // 2)
        cos[1::4], sin[1::4] = 0.0, 1.0
        cos[2::4], sin[2::4] = -1.0, -0.0
        rope = cos, sin
    ops.paged_append(cpu, k, v, pages, q_start, lens, start=start, rope=rope)
    ops.paged_append(gpu, k.cuda(), v.cuda(), *(t.cuda() for t in (pages, q_start, lens)), start=start.cuda(), rope=rope and tuple(t.cuda() for t in rope))
    _status_clean()
    for got, want in zip(_bytes(gpu), _bytes(cpu)):
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------------------ refusals

@pytest.mark.gpu
def test_reference_mode_checks_a_cache_on_the_gpu():
    """With the reference mode chosen the statements run on CUDA tensors: their caches are checked as on the CPU."""
    x = torch.zeros(4, 2, 16, 64, device="cuda")
    codes, scales = torch.zeros(4, 2, 16, 32, dtype=torch.uint8, device="cuda"), torch.zeros(4, 2, 16, 4, device="cuda").to(E4M3)
    ops.set_mode("reference")
    try:
        for match, bad in {"power of two": (x[:, :, :12].contiguous(),) * 2, "contiguous": (x.transpose(1, 2),) * 2, "one type": (x, x.half()), "come with": (codes, codes),
                           "scales are": (codes, codes, scales.float(), scales.float()), "floating type": (x.to(torch.int32),) * 2}.items():
            with pytest.raises(ValueError, match=match):
                ops.PagedKV(*bad)
        cache = ops.PagedKV(x, x.clone())
        i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")          # noqa: E731
        k = torch.randn(3, 2, 64, device="cuda")
        ops.paged_append(cache, k, -k, i32([[2, 0]]), i32([0, 3]), i32([17 + 3]))
        assert torch.equal(cache.k[0, :, 1:4], k.transpose(0, 1)) and torch.equal(ops.paged_read(cache, i32([[2, 0]]), i32([0, 3]), i32([20]), 3)[1], -k)
    finally:
        ops.set_mode("native")


@pytest.mark.gpu
@pytest.mark.parametrize("fraction,cap,match", [(0.125, None, "8 rotary channels"), (0.125, 96, "8 rotary channels"), (0.75, 96, "48 rotary channels")])
def test_engine_refuses_rotary_widths_that_the_paged_kernels_do_not_take(fraction, cap, match):
    """At construction, not at the first step behind a prefill; the static cache takes them."""
    from gdn_hybrid_architecture_ideas_b200 import config as C
    from gdn_hybrid_architecture_ideas_b200.infer.engine import DecodeEngine
    from gdn_hybrid_architecture_ideas_b200.models import build_model

    cfg = C.hybrid_model_config("60m", full=False)
    cfg.encoder.n_layers, cfg.encoder.nope_global_layers, cfg.vocab_size = 8, (1,), 512
    cfg.encoder.attention.rope_fraction, cfg.encoder.attention.rope_max_distance = fraction, cap
    model = build_model(cfg).cuda().eval()
    for kv in ("paged", "paged_fp4"):
        with pytest.raises(ValueError, match=match):
            DecodeEngine(model, 1, 32, kv_cache=kv)
    DecodeEngine(model, 1, 32)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
def test_a_cache_without_heads_is_refused(device, fmt):
    """(Its group of query heads would be a division by zero.)"""
    with pytest.raises(ValueError, match="one head"):
        ops.PagedKV.zeros(4, 16, 0, 64, fmt, device)


@pytest.mark.gpu
def test_the_first_call_on_a_device_is_not_captured(monkeypatch):
    """The device's status word is allocated by the first call. Inside a capture its zeros would belong to the graph: every replay would clear what other
    calls reported, and until the first replay it would hold anything."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    p = torch.softmax(torch.randn(1, 2, 100, device="cuda"), -1)
    args = p, None, torch.zeros(1, 1, dtype=torch.long, device="cuda"), torch.zeros(1, 1, device="cuda"), torch.zeros(1, device="cuda")
    x = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    want = ops.verify_drafts(*args)
    monkeypatch.setattr(native, "_err", {})
    for call in (lambda: ops.verify_drafts(*args), lambda: ops.PagedKV(x, x)):
        with pytest.raises(RuntimeError, match="before a capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y = args[-1] + 1
                call()
        assert not native._err
    ops.verify_drafts(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.verify_drafts(*args)
        ops.PagedKV(x, x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    native.check_status()


# ------------------------------------------------------------------------------------------------------------ callers

def _rounded(x):
    return pg.fp4_values(*pg.fp4_quantize(x)).to(x.dtype)


@pytest.mark.parametrize("kind", ["full", "plain"])
def test_engine_over_4_bit_pages_is_the_engine_over_rounded_entries_cpu(kind, monkeypatch):
    """Steps over 4-bit pages give the logits of steps over float32 pages whose entries are rounded to the 4-bit values as they are cached."""
    from gdn_hybrid_architecture_ideas_b200.infer import engine
    from tests.helpers import make_model
    from tests.test_paged import _engine_cfg

    model = make_model(_engine_cfg(kind), dtype=torch.float32).eval()
    B, P, steps = 3, 40, 6
    g = torch.Generator().manual_seed(0)
    prompts = torch.randint(0, 256, (B, P), generator=g)
    docs = torch.zeros(B, P, dtype=torch.long)
    docs[1, 11:] = 1
    feed = torch.randint(0, 256, (steps, B), generator=g)

    def logits(kv_cache):
        eng = engine.DecodeEngine(model, B, P + steps + 2, device="cpu", use_graph=False, kv_cache=kv_cache, page_size=8)
        eng.prefill(prompts, docs, rows_per_pass=2)
        out = []
        for t in feed:
            eng.tokens.copy_(t)
            eng.step()
            out.append(eng.logits.clone())
        eng.check_guards()
        return torch.stack(out)
    got, plain = logits("paged_fp4"), logits("paged")
    real = ops.paged_append

    def append(cache, k, v, pages, q_start, lens, start=None, rope=None):
        real(cache, k, v, pages, q_start, lens, start=start, rope=rope)
        k, v = ops.paged_read(cache, pages, q_start, lens, k.shape[0])
        real(cache, _rounded(k), _rounded(v), pages, q_start, lens)
    monkeypatch.setattr(engine.ops, "paged_append", append)
    want = logits("paged")
    assert (got - want).abs().max() < 1e-4 and (want - plain).abs().max() > 1e-2


@pytest.mark.gpu
def test_engine_over_4_bit_pages_is_the_engine_over_rounded_entries_gpu(monkeypatch):
    """The same on the kernels, against bfloat16 pages (which hold the 4-bit values exactly) under a cap: what remains is bfloat16 noise."""
    from gdn_hybrid_architecture_ideas_b200 import config as C
    from gdn_hybrid_architecture_ideas_b200.infer import engine
    from gdn_hybrid_architecture_ideas_b200.models import build_model

    torch.manual_seed(0)
    cfg = C.hybrid_model_config("60m", full=True)
    cfg.encoder.n_layers, cfg.encoder.nope_global_layers, cfg.vocab_size = 8, (1,), 2048
    cfg.encoder.attention.rope_max_distance = 96
    model = build_model(cfg).cuda().eval()
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn_like(p) * 0.02)
    prompts, feed = torch.randint(0, 2048, (4, 256), device="cuda"), torch.randint(0, 2048, (4, 4), device="cuda")

    def logits(kv_cache):
        eng = engine.DecodeEngine(model, 4, 280, use_graph=False, kv_cache=kv_cache)
        eng.prefill(prompts)
        out = []
        for t in feed:
            eng.tokens.copy_(t)
            eng.step()
            out.append(eng.logits.clone())
        return torch.stack(out)
    got, real = logits("paged_fp4"), ops.paged_append

    def append(cache, k, v, *a, rope=None, **kw):
        assert rope is None              # (under a cap, and in layers without positions)
        real(cache, _rounded(k), _rounded(v), *a, **kw)
    monkeypatch.setattr(engine.ops, "paged_append", append)
    want = logits("paged")
    _status_clean()
    assert float((got - want).norm() / want.norm()) < 0.05


@pytest.mark.gpu
def test_loopspec_samples_on_the_gpu_as_the_statement_decides(monkeypatch):
    """Sampled decoding of the looped encoder-decoder on the GPU (its forwards through the reference mode in float32, the verification by the
    kernel): every verification equals the statement's on the same numbers, and the tokens are its."""
    from gdn_hybrid_architecture_ideas_b200.infer import loopspec
    from gdn_hybrid_architecture_ideas_b200.ops import native
    from tests.test_paged import _looped

    model, prompt, doc, dec = _looped()
    model = model.float().cuda()
    seen, real = [], ops.verify_drafts

    def verify(*args):
        ops.set_mode("native")
        try:
            seen.append((args, real(*args)))
        finally:
            ops.set_mode("reference")
        return seen[-1][1]
    monkeypatch.setattr(loopspec.ops, "verify_drafts", verify)
    before = native.launch_count()
    ops.set_mode("reference")
    try:
        toks, stats = loopspec.LoopSpec(model).generate(prompt.cuda(), doc.cuda(), dec.cuda(), 24, greedy=False, generator=torch.Generator(device="cuda").manual_seed(7))
    finally:
        ops.set_mode("native")
    _status_clean()
    assert len(toks) == 24 and stats.steps == len(seen) == native.launch_count() - before == 23 and len(set(stats.flags)) == 2
    for i, (args, (tokens, kept)) in enumerate(seen):
        want = pg.verify_drafts(*(t.cpu() for t in args))
        assert torch.equal(tokens.cpu(), want[0]) and torch.equal(kept.cpu(), want[1]) and toks[i + 1] == int(tokens[0, 0])


# ------------------------------------------------------------------------------------------------------------ ranges out of order

@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("q_start", [[2, 4, 0, 1], [0, 9, 3, 4], [-3, 1, 3, 4], [0, 1, 3, 9], [4, 4, 4, 2]])
@pytest.mark.parametrize("more", [0, 1200])
def test_wrong_ranges_are_reported_by_append_and_read(fmt, q_start, more):
    """Status 301 whichever tokens the search finds a row for (with 1200 rows without tokens behind it does not run in shared memory); a token that gets no
    row is not cached, and stays as it is in an `out`; what is cached or read lies where the accepted rows have it."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page, n = [(20, 1, 0), (33, 2, 0), (9, 1, 0)] + [(3, 0, 0)] * more, 16, 5
    pages, _, lens, _, _, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, 64, fmt)
    tables = pages.cuda(), torch.tensor(q_start + q_start[-1:] * more, dtype=torch.int32, device="cuda"), lens.cuda()

    def reported():
        with pytest.raises(RuntimeError, match="status 301"):
            native.check_status()
    out = tuple(torch.full((n, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.paged_read(cache, *tables, n, out=out)
    reported()
    at = {}                          # packed token -> (page, slot), of the rows whose range is right
    for b in range(3):
        q0, q1 = q_start[b], q_start[b + 1]
        if 0 <= q0 <= q1 <= n:
            for j in range(q0, q1):
                p = int(lens[b]) - (q1 - j)
                at[j] = int(pages[b, p // page]), p % page
    for j in range(n):
        for o, t in zip(out, _values(cpu)):
            kept = bool((o[j] == 3).all())
            assert kept or (j in at and torch.equal(o[j].float().cpu(), t[at[j][0], :, at[j][1]].float()))
    before = [t.clone() for t in _values(cache)]
    k, v = (torch.randn(n, 2, 64, device="cuda").bfloat16() for _ in range(2))
    ops.paged_append(cache, k, v, *tables)
    reported()
    for x, t, new in zip(before, _values(cache), (k, v)):
        want = (_rounded(new.float().cpu()) if fmt == "fp4" else new.cpu()).to(t.dtype)
        for j, (page_id, slot) in at.items():
            got = t[page_id, :, slot]
            assert torch.equal(got, want[j]) or torch.equal(got, x[page_id, :, slot])
            x[page_id, :, slot] = got
        assert torch.equal(x, t)
