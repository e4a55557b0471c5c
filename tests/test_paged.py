"""The paged key/value cache (append with rotation, read, attention over bfloat16 and 4-bit pages) and the verification of
drafted tokens: the PyTorch statements against formulas written out in 64 bits, and the kernels against the statements.

Tolerances. A value rounded to a type is off by at most eps / 2 of it: bf16 2^-8, f16 2^-11, float32 2^-24. Attention: a
relative error delta of every weight (rounded probabilities, scores off by delta) moves an output by at most
(e^{2 delta} - 1) sum w |v - o| <= (e^{2 delta} - 1) 2 sum w |v|; then the output itself is rounded. delta is the sum of

* the probabilities' rounding: 2^-11 (4 bits, f16) or 2^-8 (bfloat16),
* the scores' errors, at most scale * max_t sum_c |q_c k_c| times: 2^-11 (4 bits: queries in f16) or 2^-16 (bfloat16: queries in
  two parts), plus under a cap the rotated keys' rounding, 2^-11 or 2^-8 (a rotated pair's rounding is relative to its norm: a
  factor sqrt 2 on both), plus 2^-18 for float32 sums, products with the tables and exp2 (|score| * 2^-22 among it).
"""

import math

import numpy as np
import pytest
import torch

from gdn_hybrid_architecture_ideas_b200 import ops
from gdn_hybrid_architecture_ideas_b200.ops import paged as pg

E4M3 = torch.float8_e4m3fn


def _tables(n, half, theta=1e4, device="cpu", dtype=torch.float32):
    ang = torch.arange(n, dtype=torch.float64)[:, None] * theta ** (-torch.arange(half, dtype=torch.float64) / half)
    return ang.cos().to(dtype).to(device), ang.sin().to(dtype).to(device)


def _batch(rows, page, spare=3, seed=0, device="cpu", width_extra=1):
    """rows: [(positions before, new, start)]. (pages, q_start, lens, start, n, n_pages) with shuffled page ids."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + n for a, n, _ in rows]
    need = [-(-t // page) for t in lens]
    n_pages = sum(need) + spare
    ids = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(rows), max(need + [0]) + width_extra), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = ids[at:at + m]
        at += m
    q_start = [0]
    for _, n, _ in rows:
        q_start.append(q_start[-1] + n)
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=device)       # noqa: E731
    return table.to(device), mk(q_start), mk(lens), mk([c for _, _, c in rows]), q_start[-1], n_pages


def _dense_attention(q, k, v, pos, first, cos, sin, cap, scale):
    """One query head in numpy, 64 bits: q (hd,), k, v (T, hd) from position `first` on, the query at `pos`; returns
    (output, sum w |v|, the largest scale * sum |q k|)."""
    def turn(x, i):
        h = cos.shape[1]
        y = x.copy()
        y[:h] = x[:h] * cos[i] - x[h:2 * h] * sin[i]
        y[h:2 * h] = x[h:2 * h] * cos[i] + x[:h] * sin[i]
        return y
    n = pos - first + 1
    if n <= 0:
        return np.zeros_like(q), np.zeros_like(q), 0.0
    s, big = np.empty(n), 0.0
    for j in range(n):
        a, b = q, k[j]
        if cos is not None:
            d = n - 1 - j
            if cap is None:
                a = turn(q, n - 1)
            elif d <= cap:
                a, b = turn(q, n - 1), turn(k[j], j)
            else:
                a = turn(q, cap)
        s[j] = scale * a @ b
        big = max(big, scale * np.abs(a) @ np.abs(b))
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v[:n], w @ np.abs(v[:n]), big


# ------------------------------------------------------------------------------------------------------------ 4 bits

def test_fp4_is_the_nearest_value_with_ties_to_even():
    """Every block's scale is the E4M3 value nearest max / 6 and every code the E2M1 value nearest x / s, by a search in 64
    bits; ties at the even code; saturation, zeros, infinities and NaN as described."""
    torch.manual_seed(0)
    x = torch.randn(400, 16) * 10.0 ** torch.empty(400, 1).uniform_(-4, 3)
    x[0] = 0
    x[1] = torch.tensor([6.0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0])       # scale 1: every tie
    x[2] = 1e-6                                                                                                             # no scale
    x[3, 0], x[3, 1:] = 1e30, 1.0
    x[4, 0], x[4, 1], x[4, 2:] = float("inf"), float("-inf"), 0.5
    x[5, 3] = float("nan")
    codes, scales = pg.fp4_quantize(x)
    assert codes.shape == (400, 8) and scales.shape == (400, 1) and codes.dtype == torch.uint8 and scales.dtype == E4M3
    got = pg.fp4_values(codes, scales).double()
    grid4 = torch.tensor(pg.E2M1_GRID, dtype=torch.float64)
    grid8 = torch.arange(127, dtype=torch.uint8).view(E4M3).double()

    def nearest(a, grid):
        d = (grid - a).abs()
        best = torch.nonzero(d == d.min()).flatten().tolist()
        return grid[[i for i in best if i % 2 == 0][0] if len(best) > 1 else best[0]]
    want = torch.zeros(400, 16, dtype=torch.float64)
    for i in range(400):
        row = torch.nan_to_num(x[i].double(), nan=0.0).clamp(-2688, 2688)
        s = nearest(row.abs().max() / 6, grid8)
        assert float(scales[i, 0].double()) == float(s)
        if s > 0:
            for j in range(16):
                want[i, j] = torch.sign(row[j]) * nearest(min(row[j].abs() / s, torch.tensor(6.0, dtype=torch.float64)), grid4) * s
    assert torch.equal(got, want)
    assert got[1, 1:8].tolist() == [0, 1, 1, 2, 2, 4, 4] and float(got[4, 0]) == 2688 and float(got[4, 1]) == -2688
    assert torch.equal(got, got.bfloat16().double())                       # a code times a scale is exact in bfloat16


def test_fp4_agrees_with_the_frameworks_nvfp4_up_to_its_tensor_scale():
    from gdn_hybrid_architecture_ideas_b200.ops.lowp import nvfp4_fake

    x = torch.randn(64, 64, generator=torch.Generator().manual_seed(3))
    x[0, 0] = 2688.0                                       # amax 2688: the tensor scale is 1
    assert torch.equal(pg.fp4_values(*pg.fp4_quantize(x)), nvfp4_fake(x))


# ------------------------------------------------------------------------------------------------------------ statements (CPU)

ROWS = [[(0, 1, 0)], [(5, 3, 2), (0, 0, 0), (16, 1, 16), (7, 9, 0)], [(0, 33, 0), (31, 2, 30), (0, 0, 0)]]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("fmt", ["fp64", "fp4"])
@pytest.mark.parametrize("rot", [0, 8, 16])
def test_append_and_read_cpu(rows, fmt, rot):
    hkv, hd, page = 2, 32, 8
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache = pg.PagedKV.zeros(n_pages, page, hkv, hd, fmt)
    dt = torch.float64 if fmt == "fp64" else torch.float32
    k, v = torch.randn(n + 2, hkv, hd, dtype=dt), torch.randn(n + 2, hkv, hd, dtype=dt)
    rope = _tables(64, rot // 2, dtype=dt) if rot else None
    ops.paged_append(cache, k, v, pages, q_start, lens, start=start, rope=rope)
    ko, vo = ops.paged_read(cache, pages, q_start, lens, n + 2)
    want = k.double().clone()
    for b, (a, m, c) in enumerate(rows):
        for i in range(m):
            if rot:
                z = torch.complex(want[q_start[b] + i, :, :rot // 2], want[q_start[b] + i, :, rot // 2:rot])
                z = z * torch.complex(rope[0][a + i - c].double(), rope[1][a + i - c].double())
                want[q_start[b] + i, :, :rot] = torch.cat([z.real, z.imag], -1)
    if fmt == "fp64":
        assert (ko[:n] - want[:n]).abs().max() < 1e-14 and torch.equal(vo[:n], v[:n])
    else:
        assert torch.equal(ko[:n], pg.fp4_values(*pg.fp4_quantize(want[:n].float())).bfloat16())
        assert torch.equal(vo[:n], pg.fp4_values(*pg.fp4_quantize(v[:n])).bfloat16())
    assert not ko[n:].any() and not vo[n:].any()           # packed tokens behind the last row
    touched = {(int(pages[b, p // page]), p % page) for b, (a, m, _) in enumerate(rows) for p in range(a, a + m)}
    for page_id in range(n_pages):
        for slot in range(page):
            if (page_id, slot) not in touched:
                assert not cache.k[page_id, :, slot].any()
    out = tuple(torch.full((n + 2, hkv, hd), 7.0, dtype=ko.dtype) for _ in range(2))
    ops.paged_read(cache, pages, q_start, lens, n + 2, out=out)
    assert torch.equal(out[0][:n], ko[:n]) and bool((out[1][n:] == 7).all())


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("rot,cap", [(0, None), (8, None), (8, 1), (16, 4), (16, 40)])
def test_attention_cpu(rows, rot, cap):
    hq, hkv, hd, page = 6, 2, 32, 8
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, seed=1)
    cache = pg.PagedKV.zeros(n_pages, page, hkv, hd, "fp64")
    cache.k.normal_(), cache.v.normal_()
    q = torch.randn(n + 1, hq, hd, dtype=torch.float64)
    rope = _tables(64, rot // 2, dtype=torch.float64) if rot else None
    got = ops.paged_attention(q, cache, pages, q_start, lens, start=start, rope=rope, cap=cap, scale=0.3)
    assert not got[n:].any()
    cs = (None, None) if rope is None else tuple(t.numpy() for t in rope)
    for b, (a, m, c) in enumerate(rows):
        keys = torch.stack([cache.k[int(pages[b, p // page]), :, p % page] for p in range(c, a + m)]).numpy() if a + m > c else None
        vals = torch.stack([cache.v[int(pages[b, p // page]), :, p % page] for p in range(c, a + m)]).numpy() if a + m > c else None
        for i in range(m):
            for h in range(hq):
                if keys is None:
                    assert not got[q_start[b] + i].any()
                    continue
                want, _, _ = _dense_attention(q[q_start[b] + i, h].numpy(), keys[:, h // 3], vals[:, h // 3], a + i, c, *cs, cap, 0.3)
                assert np.abs(got[q_start[b] + i, h].numpy() - want).max() < 1e-12


def test_attention_ignores_what_is_masked_cpu():
    """Entries behind the length, before the start and other tokens' future hold NaN and infinities: nothing of it shows."""
    rows = [(3, 3, 2)]
    pages, q_start, lens, start, n, n_pages = _batch(rows, 8)
    q = torch.randn(3, 2, 16, dtype=torch.float64)
    clean = pg.PagedKV.zeros(n_pages, 8, 1, 16, "fp64")
    clean.k.normal_(), clean.v.normal_()
    dirty = pg.PagedKV(clean.k.clone(), clean.v.clone())
    keep = torch.zeros(n_pages, 1, 8, 1, dtype=torch.bool)
    keep[int(pages[0, 0]), :, 2:4] = True
    dirty.k.masked_fill_(~keep, float("nan")), dirty.v.masked_fill_(~keep, float("inf"))
    a = ops.paged_attention(q, clean, pages, q_start, lens, start=start)
    b = ops.paged_attention(q, dirty, pages, q_start, lens, start=start)
    assert torch.allclose(a[0], b[0], rtol=0, atol=1e-13)      # the first new token sees positions 2 and 3 alone
    assert not torch.isfinite(b[1:]).any()


def test_refusals_cpu():
    rows = [(5, 3, 0), (2, 1, 0)]
    pages, q_start, lens, start, n, n_pages = _batch(rows, 8)
    cache = pg.PagedKV.zeros(n_pages, 8, 2, 32, "fp32")
    k = torch.randn(n, 2, 32)
    rope = _tables(32, 8)
    edit = lambda t, i, x: torch.where(torch.arange(t.numel()).view(t.shape) == i, torch.full_like(t, x), t)       # noqa: E731
    cases = {
        "q_start": dict(q_start=edit(q_start, 1, 9)), "q_start of row 1": dict(q_start=edit(q_start, 2, 2)), "cached positions": dict(lens=edit(lens, 0, 2)),
        "pages hold": dict(lens=edit(lens, 1, 1000)), "is not in 0": dict(start=edit(start, 0, 9)), "start -1": dict(start=edit(start, 0, -1)),
        "page id": dict(pages=edit(pages, 0, n_pages)), "page id -1": dict(pages=edit(pages, 0, -1)), "int32": dict(lens=lens.long()),
        "one batch": dict(lens=lens[:1]),
    }
    for match, change in cases.items():
        args = {"pages": pages, "q_start": q_start, "lens": lens, "start": start, **change}
        with pytest.raises(ValueError, match=match):
            ops.paged_append(cache, k, k, args["pages"], args["q_start"], args["lens"], start=args["start"])
        with pytest.raises(ValueError, match=match):
            ops.paged_attention(torch.randn(n, 4, 32), cache, args["pages"], args["q_start"], args["lens"], start=args["start"])
    with pytest.raises(ValueError, match="rope table"):
        ops.paged_append(cache, k, k, pages, q_start, lens, rope=_tables(7, 8))
    with pytest.raises(ValueError, match="before its start"):
        ops.paged_append(cache, k, k, pages, q_start, lens, start=edit(start, 0, 6), rope=rope)
    with pytest.raises(ValueError, match="pairs"):
        ops.paged_append(cache, k, k, pages, q_start, lens, rope=_tables(32, 17))
    with pytest.raises(ValueError, match="paged_append: k, v"):
        ops.paged_append(cache, k[:, :1], k[:, :1], pages, q_start, lens)
    with pytest.raises(ValueError, match="a multiple of 2"):
        ops.paged_attention(torch.randn(n, 3, 32), cache, pages, q_start, lens)
    for bad in (dict(cap=4), dict(cap=0, rope=rope)):
        with pytest.raises(ValueError, match="cap"):
            ops.paged_attention(torch.randn(n, 4, 32), cache, pages, q_start, lens, **bad)
    with pytest.raises(ValueError, match="rope table"):
        ops.paged_attention(torch.randn(n, 4, 32), cache, pages, q_start, lens, rope=rope, cap=32)
    with pytest.raises(ValueError, match="out is"):
        ops.paged_attention(torch.randn(n, 4, 32), cache, pages, q_start, lens, out=torch.empty(n, 4, 16))
    z = torch.zeros
    for match, make in {
        "page size": lambda: pg.PagedKV.zeros(2, 12, 1, 32, "bf16"), "fmt": lambda: pg.PagedKV.zeros(2, 8, 1, 32, "int8"), "blocks": lambda: pg.PagedKV.zeros(2, 8, 1, 40, "fp4"),
        "scales are": lambda: pg.PagedKV(z(2, 1, 8, 16, dtype=torch.uint8), z(2, 1, 8, 16, dtype=torch.uint8), z(2, 1, 8, 2), z(2, 1, 8, 2)),
        "come with": lambda: pg.PagedKV(z(2, 1, 8, 16, dtype=torch.uint8), z(2, 1, 8, 16, dtype=torch.uint8)),
        "one type": lambda: pg.PagedKV(z(2, 1, 8, 16), z(2, 1, 8, 32)), "contiguous": lambda: pg.PagedKV(z(2, 1, 16, 8).transpose(2, 3), z(2, 1, 16, 8).transpose(2, 3)),
        "floating type": lambda: pg.PagedKV(z(2, 1, 8, 16, dtype=torch.int32), z(2, 1, 8, 16, dtype=torch.int32)),
    }.items():
        with pytest.raises(ValueError, match=match):
            make()


# ------------------------------------------------------------------------------------------------------------ drafts (CPU)

def test_verified_tokens_are_distributed_as_the_target():
    """One draft over 4 tokens, its token and both uniform numbers integrated on a grid: the first emitted token follows p_0
    and, where the draft was kept, the second follows p_1, to the grid's step."""
    p = torch.tensor([[[0.1, 0.5, 0.4, 0.0], [0.25, 0.25, 0.0, 0.5]]], dtype=torch.float64)
    for q in (torch.tensor([0.3, 0.3, 0.2, 0.2], dtype=torch.float64), p[0, 0], torch.tensor([0.0, 0.0, 0.0, 1.0], dtype=torch.float64)):
        K = 50
        u = (torch.arange(K) + 0.5) / K
        first, second, kept_mass = torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.float64), 0.0
        for x in range(4):
            if q[x] == 0:
                continue
            ua, us = (t.reshape(-1) for t in torch.meshgrid(u, u, indexing="ij"))
            B = K * K
            tokens, kept = ops.verify_drafts(p.expand(B, 2, 4), q.view(1, 1, 4).expand(B, 1, 4), torch.full((B, 1), x), ua[:, None], us)
            first += q[x] * torch.bincount(tokens[:, 0], minlength=4).double() / B
            on = kept == 1
            second += q[x] * torch.bincount(tokens[on, 1], minlength=4).double() / B
            kept_mass += q[x] * on.double().mean()
            assert bool((tokens[~on, 1] == -1).all())
        assert (first - p[0, 0]).abs().max() <= 2 / K
        if kept_mass > 0:
            assert (second / kept_mass - p[0, 1]).abs().max() <= 2 / K
        assert abs(float(kept_mass) - float(torch.minimum(p[0, 0], q).sum())) <= 2 / K


def test_verify_edges_and_refusals_cpu():
    p = torch.softmax(torch.randn(2, 3, 7), -1)
    q = p[:, :2].clone()
    d = torch.tensor([[1, 2], [3, 4]])
    one = torch.ones(2)
    # q = p and u = 1: refused though the residual is zero everywhere: drawn from the target
    tokens, kept = ops.verify_drafts(p, q, d, torch.ones(2, 2), one * 0.0)
    assert kept.tolist() == [0, 0] and tokens[:, 0].tolist() == [0, 0] and bool((tokens[:, 1:] == -1).all())
    # u_sample = 1 (outside [0, 1)): the last token of positive weight
    w = p.clone()
    w[:, :, 5:] = 0
    assert ops.verify_drafts(w, None, d, torch.zeros(2, 2), one)[0][:, 2].tolist() == [4, 4]
    # without draft probabilities: u < p(x) keeps, a refusal never draws x
    t0, k0 = ops.verify_drafts(p, None, d, torch.ones(2, 2), torch.tensor([0.3, 0.9]))
    assert k0.tolist() == [0, 0] and int(t0[0, 0]) != 1 and int(t0[1, 0]) != 3
    # no drafts at all, and n_drafts
    assert ops.verify_drafts(p[:, :1], q[:, :0], d[:, :0], torch.ones(2, 0), one * 0)[0].shape == (2, 1)
    assert ops.verify_drafts(p, q, d, torch.zeros(2, 2), one * 0, n_drafts=torch.tensor([0, 1], dtype=torch.int32))[1].tolist() == [0, 1]
    for bad in (dict(drafts=d[:1]), dict(u_accept=torch.ones(2, 3)), dict(draft=q[:, :1])):
        args = {"draft": q, "drafts": d, "u_accept": torch.ones(2, 2), **bad}
        with pytest.raises(ValueError, match="verify_drafts"):
            ops.verify_drafts(p, args["draft"], args["drafts"], args["u_accept"], one)
    with pytest.raises(ValueError, match="n_drafts"):
        ops.verify_drafts(p, q, d, torch.zeros(2, 2), one, n_drafts=torch.tensor([0, 3], dtype=torch.int32))
    with pytest.raises(ValueError, match="vocabulary"):
        ops.verify_drafts(p, q, d + 5, torch.zeros(2, 2), one)


# ------------------------------------------------------------------------------------------------------------ kernels

def _dev():
    return torch.device("cuda")


def _status_clean():
    from gdn_hybrid_architecture_ideas_b200.ops import native
    native.check_status()


def _random_cache(n_pages, page, hkv, hd, fmt, seed=0):
    """A cache on the GPU full of values of unit size, and its twin on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = [torch.randn(n_pages, hkv, page, hd, generator=g) for _ in range(2)]
    if fmt == "bf16":
        cpu = pg.PagedKV(*(t.bfloat16() for t in x))
        return pg.PagedKV(cpu.k.cuda(), cpu.v.cuda()), cpu
    (kc, ks), (vc, vs) = (pg.fp4_quantize(t) for t in x)
    cpu = pg.PagedKV(kc, vc, ks, vs)
    return pg.PagedKV(*(t.cuda() for t in (kc, vc, ks, vs))), cpu


def _values(cache):
    if not cache.fp4:
        return cache.k.cpu(), cache.v.cpu()
    return tuple(pg.fp4_values(c.cpu(), s.cpu()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


MIXED = [(0, 1, 0), (37, 5, 9), (0, 0, 0), (250, 1, 0), (15, 17, 15), (0, 130, 0), (63, 1, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("hd,rot,page,dtype", [(64, 16, 8, "bf16"), (64, 64, 64, "fp32"), (128, 32, 16, "bf16"), (128, 128, 128, "fp32"), (256, 64, 32, "bf16"), (64, 48, 16, "bf16"), (64, 0, 64, "fp32")])
def test_append_and_read_kernels(fmt, hd, rot, page, dtype):
    """The pages after an append equal the statement's on the CPU, value for value (both rotate in 64 bits and round at the
    same places), entries of other positions stay, and reading gives the values back."""
    hkv = 3
    pages, q_start, lens, start, n, n_pages = _batch(MIXED, page, seed=hd)
    cache, cpu = _random_cache(n_pages, page, hkv, hd, fmt)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32}[dtype]
    base_k, base_v = (torch.randn(n + 3, hkv, 2 * hd).to(dt) for _ in range(2))      # the keys: a strided view, as of a fused projection
    base_k[2, 0, 3], base_k[3, 1, 17], base_v[4, 2, 5] = 1e6, 0.0, -1e6
    base_k[:, :, hd:].mul_(3)
    k, v = base_k[:, :, :hd], base_v[:, :, hd:]
    rope = _tables(300, rot // 2) if rot else None
    ops.paged_append(cpu, k, v, pages, q_start, lens, start=start, rope=rope)
    dev = [t.cuda() for t in (pages, q_start, lens, start)]
    ops.paged_append(cache, base_k.cuda()[:, :, :hd], base_v.cuda()[:, :, hd:], dev[0], dev[1], dev[2], start=dev[3], rope=None if rope is None else tuple(t.cuda() for t in rope))
    _status_clean()
    for got, want in zip(_values(cache), _values(cpu)):
        assert torch.equal(got, want)
    got = ops.paged_read(cache, dev[0], dev[1], dev[2], n + 3)
    want = ops.paged_read(cpu, pages, q_start, lens, n + 3)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b) and not a[n:].any()
    out = tuple(torch.full_like(t, 5.0) for t in got)
    ops.paged_read(cache, dev[0], dev[1], dev[2], n + 3, out=out)
    assert torch.equal(out[0][:n], got[0][:n]) and bool((out[0][n:] == 5).all()) and bool((out[1][n:] == 5).all())
    _status_clean()


@pytest.mark.gpu
def test_append_kernel_odd_values_and_unaligned_inputs():
    """NaN, infinities and magnitudes without a scale, from inputs whose rows start off 16-byte boundaries; many rows."""
    page, hkv, hd = 8, 2, 64
    rows = [(b % 5, b % 3, 0) for b in range(1500)]           # more rows than shared memory keeps
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, hkv, hd, "fp4")
    raw = torch.randn(n, hkv, hd + 1) * 10.0 ** torch.empty(n, hkv, 1).uniform_(-5, 4)
    raw[0, 0, 5], raw[1, 1, 6], raw[2, 0, 7], raw[2, 1] = float("nan"), float("inf"), float("-inf"), 0.0
    k = raw[:, :, 1:]
    ops.paged_append(cpu, k, k, pages, q_start, lens)
    kc = raw.cuda()[:, :, 1:]
    ops.paged_append(cache, kc, kc, *(t.cuda() for t in (pages, q_start, lens)))
    _status_clean()
    for got, want in zip(_values(cache), _values(cpu)):
        assert torch.equal(got, want)


def _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, rope, cap, scale=None, page=16, got=None):
    """Every output of the kernel within the bound of the module's head."""
    n, hq, hd = q.shape
    hkv = cpu.n_kv_heads
    fp4 = cpu.fp4
    sc = hd ** -0.5 if scale is None else scale
    if got is None:
        dev = [t.cuda() for t in (pages, q_start, lens, start)]
        got = ops.paged_attention(q.cuda(), cache, dev[0], dev[1], dev[2], start=dev[3], rope=None if rope is None else tuple(t.cuda() for t in rope), cap=cap, scale=scale)
    _status_clean()
    assert got.dtype == torch.bfloat16
    kv = [t.double().numpy() for t in _values(cpu)]
    cs = (None, None) if rope is None else tuple(t.double().numpy() for t in rope)
    worst = 0.0
    for b, (a, m, c) in enumerate(rows):
        for i in range(m):
            j = int(q_start[b]) + i
            if a + i < c:
                assert not got[j].any()
                continue
            at = [(int(pages[b, p // page]), p % page) for p in range(c, a + i + 1)]
            ids, slots = np.array([x for x, _ in at]), np.array([y for _, y in at])
            for h in range(hq):
                o, mass, big = _dense_attention(q[j, h].double().numpy(), kv[0][ids, h * hkv // hq, slots], kv[1][ids, h * hkv // hq, slots], a + i, c, *cs, cap, sc)
                d = (2.0 ** -11 if fp4 else 2.0 ** -8) + big * ((2.0 ** -11 if fp4 else 2.0 ** -16) * 1.42 + (0 if cap is None else (2.0 ** -11 if fp4 else 2.0 ** -8) * 1.42) + 2.0 ** -18) + 2.0 ** -18
                bound = 2.0 ** -8 * np.abs(o) + (math.exp(2 * d) - 1) * 2 * mass * (1 + 2.0 ** -8)
                diff = np.abs(got[j, h].double().cpu().numpy() - o)
                worst = max(worst, float((diff / (bound + 1e-30)).max()))
                assert (diff <= bound + 1e-30).all(), (b, i, h, diff.max(), worst)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("hd,group,rot,cap,page,qdt", [
    (64, 1, 16, None, 8, "bf16"), (64, 4, 16, 20, 16, "bf16"), (64, 3, 64, 33, 64, "fp32"), (64, 8, 32, 1, 32, "bf16"), (64, 20, 0, None, 16, "bf16"),
    (128, 4, 32, None, 16, "fp32"), (128, 5, 32, 40, 64, "bf16"), (128, 2, 128, None, 16, "bf16"), (256, 8, 64, None, 16, "bf16"), (256, 1, 64, 100, 16, "fp32")])
def test_attention_kernels(fmt, hd, group, rot, cap, page, qdt):
    """Ragged rows: empty, one position, starts inside pages, several new tokens, a start behind the query, a prompt."""
    rows = [(0, 1, 0), (37, 5, 9), (0, 0, 0), (250, 1, 0), (15, 4, 17), (0, 21, 0), (300, 2, 290)]
    hkv = 2
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, seed=group)
    cache, cpu = _random_cache(n_pages, page, hkv, hd, fmt, seed=rot)
    q = (torch.randn(n, hkv * group, hd) * 1.5).to({"bf16": torch.bfloat16, "fp32": torch.float32}[qdt])
    rope = _tables(320, rot // 2) if rot else None
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, rope, cap, page=page)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("hd,group,rot", [(64, 6, 16), (64, 7, 64), (128, 4, 32), (128, 3, 64), (256, 4, 64), (256, 3, 16)])
@pytest.mark.parametrize("cap", [None, 25])
def test_attention_kernels_many_query_rows(fmt, hd, group, rot, cap):
    """More query rows than one block of 8: several blocks, partly used ones, several units, rows with different counts."""
    rows, page = [(30, 9, 0), (100, 1, 70), (64, 2, 0), (0, 4, 1), (3, 14, 0)], 8
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, fmt)
    q = torch.randn(n, 2 * group, hd).bfloat16()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, _tables(110, rot // 2), cap, page=page)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd,new", [("fp4", 64, 1), ("fp4", 128, 3), ("bf16", 64, 2), ("bf16", 256, 1), ("fp4", 256, 9)])
def test_attention_kernels_long_rows(fmt, hd, new):
    """Rows long enough to be cut over many CTAs and joined; one of them short, so that borders fall inside units."""
    rows, page = [(5000, new, 0), (3, new, 0), (2777, new, 1201)], 64
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 1, hd, fmt)
    q = torch.randn(n, 2, hd).bfloat16()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, _tables(5100, 16), 700, page=page)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
def test_attention_kernel_extreme_queries(fmt):
    """Query rows of very different sizes in one tile (a power of two per row brings them to one), zeros, and one with a NaN."""
    rows, page = [(40, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 1, 64, fmt)
    q = torch.randn(1, 8, 64) * torch.tensor([1e-20, 1e-3, 1.0, 30.0, 0.0, 1e-8, 3.0, 1.0])[None, :, None]
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, None, None, page=page)
    q[0, 3, 0] = float("nan")
    got = ops.paged_attention(q.cuda(), cache, *(t.cuda() for t in (pages, q_start, lens)))
    assert bool(got[0, 3].isnan().all()) and bool(torch.isfinite(got[0, [0, 1, 2, 4, 5, 6, 7]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_kernel_ignores_what_is_masked(fmt, hd):
    """Everything a row does not see is NaN (bfloat16) or bytes of ones (4 bits: NaN scales): free pages, slots behind the length,
    positions before the start; with bfloat16 also infinities and NaN in later tokens of the same row."""
    rows, page = [(21, 3, 5), (0, 2, 0), (64, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, hd, fmt)
    seen = torch.zeros(n_pages, page, dtype=torch.bool)
    for b, (a, m, c) in enumerate(rows):
        for p in range(c, a + m):
            seen[int(pages[b, p // page]), p % page] = True
    hide = (~seen)[:, None, :, None].cuda()
    for t in (cache.k, cache.v):
        t.masked_fill_(hide, 255 if fmt == "fp4" else float("nan"))
    if fmt == "fp4":
        for t in (cache.k_scale, cache.v_scale):
            t.view(torch.uint8).masked_fill_(hide, 255)
    q = torch.randn(n, 8, hd).bfloat16()
    rope = _tables(80, 16)
    got = _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, rope, 10, page=page)
    if fmt == "bf16":
        last = (int(pages[0, 23 // page]), 23 % page)
        cache.v[last[0], :, last[1], ::3] = float("inf")
        cache.v[last[0], :, last[1], 1::3] = float("nan")
        cache.k[last[0], :, last[1]] = float("nan")
        args = [t.cuda() for t in (pages, q_start, lens)]
        again = ops.paged_attention(q.cuda(), cache, *args, start=start.cuda(), rope=tuple(t.cuda() for t in rope), cap=10)
        keep = [0, 1, 3, 4, 5]
        assert bool(torch.isfinite(again[keep]).all()) and bool(again[2].isnan().all())
        # (the tile with the odd values is summed position by position: another order of float32 sums, at most one rounding away)
        assert (again[keep].float() - got[keep].float()).abs().max() <= 2.0 ** -7 * got[keep].float().abs().max()


@pytest.mark.gpu
def test_padding_outputs_and_strided_queries():
    rows, page = [(20, 1, 0), (33, 2, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, cpu = _random_cache(n_pages, page, 2, 64, "fp4")
    wide = torch.randn(n + 2, 8, 128, dtype=torch.bfloat16)
    args = [t.cuda() for t in (pages, q_start, lens)]
    q = wide.cuda()[:, :, 64:]                                    # as of a projection with the gate interleaved
    got = ops.paged_attention(q, cache, *args)
    assert not got[n:].any()
    out = torch.full((n + 2, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    assert ops.paged_attention(q, cache, *args, out=out) is out
    assert torch.equal(out[:n], got[:n]) and bool((out[n:] == 3).all())
    assert torch.equal(ops.paged_attention(q.contiguous(), cache, *args)[:n], got[:n])
    empty = torch.zeros(0, 8, 64, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(empty, cache, args[0], none, args[2]).shape == (0, 8, 64)
    ops.paged_append(cache, empty[:, :2], empty[:, :2], args[0], none, args[2])
    assert ops.paged_read(cache, args[0], none, args[2], 0)[0].shape == (0, 2, 64)
    # rows without new tokens everywhere, packed tokens that are padding alone
    assert not ops.paged_attention(q, cache, args[0], none, args[2]).any()
    _status_clean()


@pytest.mark.gpu
def test_wrong_tables_are_reported_on_the_device():
    """Values that the host cannot see: the kernels leave the access out, write the status word and keep the other rows right."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page = [(20, 1, 0), (33, 2, 0), (9, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, _ = _random_cache(n_pages, page, 2, 64, "fp4")
    rope = tuple(t.cuda() for t in _tables(64, 8))
    q = torch.randn(n, 4, 64, dtype=torch.bfloat16, device="cuda")
    good = ops.paged_attention(q, cache, *(t.cuda() for t in (pages, q_start, lens)), start=start.cuda(), rope=rope)
    _status_clean()

    def edit(t, i, x):
        t = t.clone()
        t.view(-1)[i] = x
        return t
    for code, change, row in ((304, dict(pages=edit(pages, 0, n_pages)), 0), (304, dict(pages=edit(pages, 0, -7)), 0), (302, dict(lens=edit(lens, 0, 0)), 0),
                              (302, dict(lens=edit(lens, 2, 4000)), 2), (303, dict(start=edit(start, 0, 22)), 0), (303, dict(start=edit(start, 0, -1)), 0)):
        a = {"pages": pages, "q_start": q_start, "lens": lens, "start": start, **change}
        a = {k: v.cuda() for k, v in a.items()}
        got = ops.paged_attention(q, cache, a["pages"], a["q_start"], a["lens"], start=a["start"], rope=rope)
        with pytest.raises(RuntimeError, match=f"status {code}"):
            native.check_status()
        others = [j for j in range(n) if not int(q_start[row]) <= j < int(q_start[row + 1])]
        assert torch.equal(got[others], good[others])
        before = [t.clone() for t in (cache.k, cache.v, cache.k_scale.view(torch.uint8), cache.v_scale.view(torch.uint8))]
        if code != 304:                                          # (the bad page of that row is not the one its new token goes to)
            k = torch.randn(n, 2, 64, dtype=torch.bfloat16, device="cuda")
            only = a["q_start"].clone()
            only[:row + 1], only[row + 1:] = 0, int(q_start[row + 1] - q_start[row])
            ops.paged_append(cache, k, k, a["pages"], only, a["lens"], start=a["start"], rope=rope)
            with pytest.raises(RuntimeError, match=f"status {code}"):
                native.check_status()
            assert all(torch.equal(x, y) for x, y in zip(before, (cache.k, cache.v, cache.k_scale.view(torch.uint8), cache.v_scale.view(torch.uint8))))
    dev = [t.cuda() for t in (pages, q_start, lens)]
    ops.paged_attention(q, cache, dev[0], edit(q_start, 1, 9).cuda(), dev[2])
    with pytest.raises(RuntimeError, match="status 301"):
        native.check_status()
    ops.paged_append(cache, q[:, :2], q[:, :2], *dev, rope=tuple(t[:16] for t in rope))
    with pytest.raises(RuntimeError, match="status 305"):
        native.check_status()
    ops.paged_read(cache, edit(pages, 0, 10 ** 6).cuda(), dev[1], edit(lens, 0, 5).cuda(), n)
    with pytest.raises(RuntimeError, match="status 304"):
        native.check_status()


@pytest.mark.gpu
def test_refusals_of_the_cuda_entries():
    rows, page = [(20, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, device="cuda")
    cache, _ = _random_cache(n_pages, page, 2, 64, "fp4")
    q = torch.randn(n, 4, 64, dtype=torch.bfloat16, device="cuda")
    k = q[:, :2]
    r = lambda half, n=64: tuple(t.cuda() for t in _tables(n, half))          # noqa: E731
    for match, call in {
        "multiple of 2": lambda: ops.paged_attention(q[:, :3], cache, pages, q_start, lens),
        "float32": lambda: ops.paged_attention(q.half(), cache, pages, q_start, lens),
        "int32": lambda: ops.paged_attention(q, cache, pages.long(), q_start, lens),
        "one batch": lambda: ops.paged_attention(q, cache, pages, q_start[:1], lens),
        "under a cap": lambda: ops.paged_attention(q, cache, pages, q_start, lens, rope=r(24), cap=5),
        "inside the rope table": lambda: ops.paged_attention(q, cache, pages, q_start, lens, rope=r(8), cap=64),
        "multiple of 16": lambda: ops.paged_append(cache, k, k, pages, q_start, lens, rope=r(4)),
        "unit inner stride": lambda: ops.paged_attention(torch.randn(n, 64, 4, device="cuda").transpose(1, 2), cache, pages, q_start, lens),
        "cache's device": lambda: ops.paged_attention(q.cpu(), cache, pages, q_start, lens),
        "on the cache's device": lambda: ops.paged_append(cache, k, k, pages.cpu(), q_start, lens),
        "out is": lambda: ops.paged_attention(q, cache, pages, q_start, lens, out=torch.empty(n, 4, 64, device="cuda")),
        "bfloat16 or float32": lambda: ops.paged_append(cache, k.half(), k.half(), pages, q_start, lens),
        "head dimension 32": lambda: ops.paged_append(pg.PagedKV.zeros(4, 16, 2, 32, "bf16", "cuda"), k[..., :32], k[..., :32], pages, q_start, lens),
        "out holds": lambda: ops.paged_read(cache, pages, q_start, lens, 4, out=(k, k)),
    }.items():
        with pytest.raises((RuntimeError, ValueError), match=match):
            call()
    with pytest.raises(ValueError, match="cap"):
        ops.paged_attention(q, cache, pages, q_start, lens, cap=4)


@pytest.mark.gpu
def test_captured_steps_and_other_streams():
    """Append + attention captured once and replayed while lengths and pages move on, beside a second captured graph and a
    call on another stream: every result equals the eager call's."""
    B, page, hkv, hd, steps = 5, 16, 2, 64, 6
    rows = [(10 + 13 * b, 1, 0) for b in range(B)]
    pages, q_start, lens, start, n, n_pages = _batch([(a + steps, 1, 0) for a, _, _ in rows], page, device="cuda")
    lens0 = torch.tensor([a + 1 for a, _, _ in rows], dtype=torch.int32, device="cuda")
    eager, _ = _random_cache(n_pages, page, hkv, hd, "fp4")
    caught = pg.PagedKV(eager.k.clone(), eager.v.clone(), eager.k_scale.view(torch.uint8).clone().view(E4M3), eager.v_scale.view(torch.uint8).clone().view(E4M3))
    rope = tuple(t.cuda() for t in _tables(128, 8))
    q, k, v = (torch.randn(steps, n, h, hd, dtype=torch.bfloat16, device="cuda") for h in (8, hkv, hkv))
    sq, sk, sv, sl = torch.empty_like(q[0]), torch.empty_like(k[0]), torch.empty_like(v[0]), lens0.clone()

    def step(cache, qq, kk, vv, ll):
        ops.paged_append(cache, kk, vv, pages, q_start, ll, rope=rope)
        return ops.paged_attention(qq, cache, pages, q_start, ll, rope=rope)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t, src in ((sq, q), (sk, k), (sv, v)):
            t.copy_(src[0])
        step(caught, sq, sk, sv, sl)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(caught, sq, sk, sv, sl))
        graphs.append(gr)
    for i in range(steps):
        want = step(eager, q[i], k[i], v[i], lens0 + i)
        for t, src in ((sq, q), (sk, k), (sv, v)):
            t.copy_(src[i])
        sl.copy_(lens0 + i)
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        ll = lens0 + i
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.paged_attention(q[i], eager, pages, q_start, ll, rope=rope)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)
    _status_clean()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """A cache of over 2^32 bytes of keys: pages at its end are written and read."""
    page, hkv, hd = 64, 2, 256
    n_pages = 68000                                             # 64 KB a page and side: 4.4 GB each
    cache = pg.PagedKV(*(torch.empty(n_pages, hkv, page, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    rows = [(0, 70, 0), (3, 1, 0)]
    pages = torch.tensor([[n_pages - 1, 66000], [n_pages - 2, 0]], dtype=torch.int32, device="cuda")
    q_start = torch.tensor([0, 70, 71], dtype=torch.int32, device="cuda")
    lens = torch.tensor([70, 4], dtype=torch.int32, device="cuda")
    cache.k[n_pages - 2].zero_(), cache.v[n_pages - 2].zero_()
    k, v, q = (torch.randn(71, h, hd, dtype=torch.bfloat16, device="cuda") for h in (2, 2, 4))
    ops.paged_append(cache, k, v, pages, q_start, lens)
    got = ops.paged_read(cache, pages, q_start, lens, 71)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    assert torch.equal(cache.k[n_pages - 1, :, 5], k[5]) and torch.equal(cache.v[66000, :, 3], v[67])
    small = pg.PagedKV(*(torch.stack([t[n_pages - 1], t[66000], t[n_pages - 2]]).contiguous() for t in (cache.k, cache.v)))
    want = ops.paged_attention(q, small, torch.tensor([[0, 1], [2, 0]], dtype=torch.int32, device="cuda"), q_start, lens)
    assert torch.equal(ops.paged_attention(q, cache, pages, q_start, lens), want)
    _status_clean()


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,V,dtype,with_draft", [(1, 3, 32768, "float32", True), (7, 4, 9001, "float32", True), (33, 2, 130, "bfloat16", True), (5, 0, 64000, "float32", True),
                                                    (4, 40, 17, "float32", True), (6, 3, 20000, "float32", False), (3, 1, 1, "float32", True), (9, 5, 8192, "bfloat16", False)])
def test_verify_kernel(B, N, V, dtype, with_draft):
    """Tokens and counts equal the statement's exactly, over many random numbers; ragged drafts; NaN behind a row's last draft."""
    dt = getattr(torch, dtype)
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(B, N + 1, V, generator=g) * 2
    target = torch.softmax(logits, -1)
    target[:, :, ::7] = 0 if V > 7 else target[:, :, ::7]
    draft = torch.softmax(logits[:, :N] + 0.6 * torch.randn(B, N, V, generator=g), -1)
    drafts = torch.multinomial(draft.reshape(B * N, V), 1, generator=g).view(B, N) if N else torch.zeros(B, 0, dtype=torch.long)
    target, draft = target.to(dt), draft.to(dt)
    n = torch.randint(0, N + 1, (B,), generator=g).to(torch.int32)
    for b in range(B):
        target[b, int(n[b]) + 1:] = float("nan")
        draft[b, int(n[b]):] = float("nan")
    wide = torch.zeros(B, N + 2, V + 3, dtype=dt)
    wide[:, :N + 1, 1:V + 1] = target
    dev = wide.cuda()[:, :N + 1, 1:V + 1]                       # strided, not 16-byte aligned
    for trial in range(4):
        ua, us = torch.rand(B, N, generator=g), torch.rand(B, generator=g)
        if trial == 2:
            us[:] = 0
        if trial == 3:
            us[:], ua[:] = 1 - 2.0 ** -24, 0
        want = ops.verify_drafts(target, draft if with_draft else None, drafts, ua, us, n)
        for tgt in (target.cuda(), dev):
            got = ops.verify_drafts(tgt, draft.cuda() if with_draft else None, drafts.cuda(), ua.cuda(), us.cuda(), n.cuda())
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]), trial
    _status_clean()


@pytest.mark.gpu
def test_verify_kernel_edges_and_reports():
    from gdn_hybrid_architecture_ideas_b200.ops import native

    V = 12000
    p = torch.softmax(torch.randn(2, 3, V), -1)
    d = torch.tensor([[1, 2], [3, 4]])
    one = torch.ones(2)
    cpu = (p, p[:, :2].clone(), d, torch.ones(2, 2), one * 0.4)
    want = ops.verify_drafts(*cpu)                               # q = p, u = 1: the residual is zero everywhere
    got = ops.verify_drafts(*(t.cuda() for t in cpu))
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]) and want[1].tolist() == [0, 0]
    w = p.clone()
    w[:, :, 11000:] = 0
    assert ops.verify_drafts(w.cuda(), None, d.cuda(), torch.zeros(2, 2).cuda(), one.cuda())[0][:, 2].tolist() == [10999, 10999]
    assert ops.verify_drafts((p * 0).cuda(), None, d.cuda(), torch.ones(2, 2).cuda(), one.cuda())[0].tolist() == [[0, -1, -1]] * 2
    assert ops.verify_drafts(p[:0].cuda(), None, d[:0].cuda(), torch.ones(0, 2).cuda(), one[:0].cuda())[0].shape == (0, 3)
    _status_clean()
    ops.verify_drafts(p.cuda(), None, d.cuda(), torch.zeros(2, 2).cuda(), one.cuda() * 0, n_drafts=torch.tensor([5, 1], dtype=torch.int32).cuda())
    with pytest.raises(RuntimeError, match="status 306"):
        native.check_status()
    t, k = ops.verify_drafts(p.cuda(), None, (d + V).cuda(), torch.zeros(2, 2).cuda(), one.cuda() * 0)
    with pytest.raises(RuntimeError, match="status 307"):
        native.check_status()
    assert k.tolist() == [0, 0]
    for match, bad in (("int64", dict(drafts=d.int())), ("draft bfloat16|of target's type", dict(draft=p[:, :2].bfloat16())), ("u_accept", dict(u=torch.zeros(2, 2).double()))):
        a = {"draft": p[:, :2], "drafts": d, "u": torch.zeros(2, 2), **bad}
        with pytest.raises(RuntimeError, match=match):
            ops.verify_drafts(p.cuda(), a["draft"].cuda(), a["drafts"].cuda(), a["u"].cuda(), one.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "fp4"])
def test_the_operators_together(fmt):
    """Two rounds of drafted decoding as a server runs them, ragged rows: prompts enter the cache, drafted tokens are appended and
    scored in one pass, the scores become probabilities and are verified, the lengths fall back to what was kept. Against
    the statements on the CPU with the same cache contents."""
    torch.manual_seed(5)
    B, hq, hkv, hd, page, N, V = 3, 8, 2, 64, 16, 3, 500
    prompt = [40, 7, 65]
    room = [p + 16 for p in prompt]
    pages, _, _, _, _, n_pages = _batch([(r, 0, 0) for r in room], page)
    rope = _tables(128, 8)
    cpu = pg.PagedKV.zeros(n_pages, page, hkv, hd, fmt)
    gpu = pg.PagedKV.zeros(n_pages, page, hkv, hd, fmt, "cuda")
    head = torch.randn(hq * hd, V) * 0.3
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)          # noqa: E731

    def both(fn, *tensors, **kw):
        return fn(cpu, *tensors), fn(gpu, *(t.cuda() for t in tensors))

    n = sum(prompt)
    qs, lens = i32([0, 40, 47, 112]), i32(prompt)
    k, v = torch.randn(n, hkv, hd).bfloat16(), torch.randn(n, hkv, hd).bfloat16()
    both(lambda c, k, v, p, s, l, co, si: ops.paged_append(c, k, v, p, s, l, rope=(co, si)), k, v, pages, qs, lens, *rope)
    for rnd in range(2):
        m = N + 1
        lens = lens + m
        qs = i32([0, m, 2 * m, 3 * m])
        q, k, v = (torch.randn(B * m, h, hd).bfloat16() for h in (hq, hkv, hkv))
        both(lambda c, k, v, p, s, l, co, si: ops.paged_append(c, k, v, p, s, l, rope=(co, si)), k, v, pages, qs, lens, *rope)
        oc, og = both(lambda c, q, p, s, l, co, si: ops.paged_attention(q, c, p, s, l, rope=(co, si)), q, pages, qs, lens, *rope)
        # bf16 outputs of the two, each at most (2^-8 + 2^-8) of the weighted values off (the module's head): well within
        assert (oc.float() - og.float().cpu()).abs().max() <= 2.0 ** -5 * oc.float().abs().max()
        target = torch.softmax((oc.float().reshape(B, m, -1) @ head), -1)
        draft = torch.softmax((oc.float().reshape(B, m, -1) @ head)[:, :N] + 0.5 * torch.randn(B, N, V), -1)
        drafts = torch.multinomial(draft.reshape(-1, V), 1).view(B, N)
        ua, us = torch.rand(B, N), torch.rand(B)
        tc, kc = ops.verify_drafts(target, draft, drafts, ua, us)
        tg, kg = ops.verify_drafts(*(t.cuda() for t in (target, draft, drafts, ua, us)))
        assert torch.equal(tc, tg.cpu()) and torch.equal(kc, kg.cpu())
        lens = (lens - (N - kc)).to(torch.int32)
        for a, b in zip(_values(cpu), _values(gpu)):
            assert torch.equal(a, b)
    _status_clean()


# ------------------------------------------------------------------------------------------------------------ callers: the decode engine, LoopSpec

def _engine_cfg(kind):
    from gdn_hybrid_architecture_ideas_b200 import config as C

    cfg = C.tiny_full_config() if kind == "full" else C.tiny_control_config()
    cfg.encoder.attention.head_dim = 16
    return cfg


@pytest.mark.parametrize("kind", ["full", "plain"])
def test_engine_over_pages_matches_prefill_and_extend_cpu(kind):
    """The decode engine on paged keys and values equals the model's own cached forward (with the distance cap, position-free
    layers, a document that starts inside a row; and rotated keys without a cap)."""
    from gdn_hybrid_architecture_ideas_b200.infer.engine import DecodeEngine
    from tests.helpers import make_model
    from tests.test_decode_engine import _oracle

    model = make_model(_engine_cfg(kind), dtype=torch.float32).eval()
    B, P, steps = 3, 40, 6
    g = torch.Generator().manual_seed(0)
    prompts = torch.randint(0, 256, (B, P), generator=g)
    docs = torch.zeros(B, P, dtype=torch.long)
    docs[1, 11:] = 1
    want = _oracle(model, prompts, docs, steps)
    eng = DecodeEngine(model, B, P + steps + 2, device="cpu", use_graph=False, kv_cache="paged", page_size=8)
    assert torch.equal(eng.prefill(prompts, docs, rows_per_pass=2), want[:, 0].argmax(-1))
    for i in range(1, steps):
        eng.step()
        assert (eng.logits - want[:, i]).abs().max() < 2e-4
    eng.check_guards()


def test_engine_over_4_bit_pages_cpu():
    """The first attention layer's pages hold the static engine's keys and values in 4 bits; steps run, no guard is touched,
    the cache takes 4.5 / 32 of the float32 bytes."""
    from gdn_hybrid_architecture_ideas_b200.infer.engine import DecodeEngine
    from tests.helpers import make_model

    model = make_model(_engine_cfg("full"), dtype=torch.float32).eval()
    prompts = torch.randint(0, 256, (2, 30), generator=torch.Generator().manual_seed(1))
    kw = dict(device="cpu", use_graph=False)
    eng, static = DecodeEngine(model, 2, 48, kv_cache="paged_fp4", page_size=16, **kw), DecodeEngine(model, 2, 48, **kw)
    eng.prefill(prompts), static.prefill(prompts)
    li = next(i for i, st in enumerate(eng.layers) if "paged" in st)
    c = eng.layers[li]["paged"]
    q_start = torch.tensor([0, 30, 60], dtype=torch.int32)
    k, v = ops.paged_read(c, eng.pages, q_start, eng.lens, 60)
    for got, name in ((k, "k"), (v, "v")):
        x = static.layers[li][name][:, :30].flatten(0, 1)
        assert torch.equal(got, pg.fp4_values(*pg.fp4_quantize(x)).bfloat16())
    for _ in range(4):
        eng.step()
    assert torch.isfinite(eng.logits).all()
    eng.check_guards()
    attn = lambda e: sum(st["paged"].bytes() if "paged" in st else st["k"].numel() * 8 for st in e.layers if "paged" in st or "k" in st)       # noqa: E731
    assert attn(eng) * 32 == attn(static) * 4.5


def test_engine_refuses_paged_grid_and_unknown_caches():
    from gdn_hybrid_architecture_ideas_b200.infer.engine import DecodeEngine
    from tests.helpers import make_model
    from tests.test_decode_engine import _cfg

    with pytest.raises(ValueError, match="grid"):
        DecodeEngine(make_model(_cfg("grid"), dtype=torch.float32), 1, 16, device="cpu", use_graph=False, kv_cache="paged")
    with pytest.raises(ValueError, match="kv_cache"):
        DecodeEngine(make_model(_cfg("full"), dtype=torch.float32), 1, 16, device="cpu", use_graph=False, kv_cache="fp8")


@pytest.mark.gpu
@pytest.mark.parametrize("kv_cache", ["paged", "paged_fp4"])
@pytest.mark.parametrize("cap", [96, None])
def test_engine_over_pages_gpu(kv_cache, cap):
    """The captured step equals the eager one token for token; with bfloat16 pages the logits agree with the static cache's
    (the same cached values, rotated and scored by another kernel: bfloat16 noise), with 4 bits they stay near."""
    from gdn_hybrid_architecture_ideas_b200 import config as C
    from gdn_hybrid_architecture_ideas_b200.infer.engine import DecodeEngine
    from gdn_hybrid_architecture_ideas_b200.models import build_model

    torch.manual_seed(0)
    cfg = C.hybrid_model_config("60m", full=True)
    cfg.encoder.n_layers, cfg.encoder.nope_global_layers, cfg.vocab_size = 8, (1,), 2048
    cfg.encoder.attention.rope_max_distance = cap
    model = build_model(cfg).cuda().eval()
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn_like(p) * 0.02)
    B, P, steps = 4, 256, 8
    prompts = torch.randint(0, 2048, (B, P), device="cuda")
    mk = lambda graph, kv: DecodeEngine(model, B, P + steps + 4, use_graph=graph, kv_cache=kv)          # noqa: E731
    graph, eager, static = mk(True, kv_cache), mk(False, kv_cache), mk(False, "static")
    assert torch.equal(graph.generate(prompts, steps), eager.generate(prompts, steps))
    _status_clean()
    graph.check_guards(), eager.check_guards()
    eager.prefill(prompts), static.prefill(prompts)
    eager.tokens.copy_(static.tokens)
    eager.step(), static.step()
    rel = float((eager.logits - static.logits).norm() / static.logits.norm())
    assert rel < (0.05 if kv_cache == "paged" else 0.5), rel


def _looped():
    from gdn_hybrid_architecture_ideas_b200 import config as C
    from gdn_hybrid_architecture_ideas_b200.models import build_model

    torch.manual_seed(0)
    cfg = C.tiny_looped_config()
    model = build_model(cfg).double().eval()
    g = torch.Generator().manual_seed(2)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn(p.shape, generator=g, dtype=p.dtype) * 0.05)
    prompt = torch.randint(0, cfg.vocab_size, (1, 14), generator=g)
    doc, dec = torch.zeros_like(prompt), torch.zeros_like(prompt, dtype=torch.bool)
    dec[0, 9:] = True
    return model, prompt, doc, dec


def test_loopspec_samples_by_the_acceptance_rule(monkeypatch):
    """Every step's decision is the rule's on the distributions of the model's own forwards at that prefix: the target's of two
    passes, the draft head's of one; a draft head equal to the target is always kept."""
    from gdn_hybrid_architecture_ideas_b200.infer import loopspec

    model, prompt, doc, dec = _looped()
    seen = []
    real = ops.verify_drafts
    monkeypatch.setattr(loopspec.ops, "verify_drafts", lambda *a, **k: seen.append((a, real(*a, **k))) or seen[-1][1])
    toks, stats = loopspec.LoopSpec(model).generate(prompt, doc, dec, 10, greedy=False, generator=torch.Generator().manual_seed(7))
    assert len(toks) == 10 and stats.steps == len(seen) == 9 and stats.flags == [bool(k[0]) for _, (_, k) in seen] and len(set(stats.flags)) == 2
    for i, ((target, draft, drafted, ua, us), (tokens, kept)) in enumerate(seen):
        prefix = torch.cat([prompt, torch.tensor([toks[:i + 1]])], 1)
        mask = torch.cat([dec, torch.ones(1, i + 1, dtype=torch.bool)], 1)
        with torch.no_grad():
            two = model(prefix, torch.zeros_like(prefix), mask, T=2, capacity=int(mask.sum())).logits[0, prefix.shape[1] - 1]
        p = torch.softmax(two.float(), -1)
        assert (target[0, 0] - p).abs().max() < 1e-6
        x, q = int(drafted), draft[0, 0].double()
        keep = float(ua) * float(q[x]) < float(target[0, 0, x])
        assert bool(kept[0]) == keep and toks[i + 1] == int(tokens[0, 0])
        if keep:
            assert toks[i + 1] == x
        else:
            w = (target[0, 0].double() - q).clamp(min=0)
            assert toks[i + 1] == int((w.cumsum(0) > float(us) * w.sum()).nonzero()[0])
    again, _ = loopspec.LoopSpec(model).generate(prompt, doc, dec, 10, greedy=False, generator=torch.Generator().manual_seed(7))
    assert again == toks
    with torch.no_grad():                    # a second pass that changes nothing
        model.readout_norms[0].weight.copy_(model.decoder_norm.weight)
        for layer in model.decoder_layers:
            layer.residual_scale = 0.0
        model.injection.A_log.fill_(-30.0)
        model.injection.B.zero_()
        model.loop_embedding.zero_()
    _, stats = loopspec.LoopSpec(model).generate(prompt, doc, dec, 8, greedy=False, generator=torch.Generator().manual_seed(3))
    assert stats.acceptance == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_kernel_scales_that_are_no_numbers_reach_only_who_sees_them(hd):
    """4 bits: one value scale of a row's last new token is NaN. Its own query gets NaN in that block of 16 channels; the two before it, which
    do not see it (their weights there are zero before and after), and every other channel keep what they had."""
    rows, page, block = [(21, 3, 5), (40, 1, 0)], 16, 2
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    cache, _ = _random_cache(n_pages, page, 2, hd, "fp4")
    q = torch.randn(n, 8, hd, device="cuda").bfloat16()
    args = (q, cache, *(t.cuda() for t in (pages, q_start, lens)))
    before = ops.paged_attention(*args, start=start.cuda())
    cache.v_scale.view(torch.uint8)[int(pages[0, 23 // page]), 1, 23 % page, block] = 0x7f
    got = ops.paged_attention(*args, start=start.cuda())
    hit = torch.zeros(n, 8, hd, dtype=torch.bool, device="cuda")
    hit[2, 4:, 16 * block:16 * block + 16] = True               # query heads 4 .. 7 read key head 1
    assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], before[~hit])
    cache.v_scale.view(torch.uint8)[int(pages[0, 8 // page]), 0, 8 % page, 0] = 0xff          # in a place that all of the row's queries see
    got = ops.paged_attention(*args, start=start.cuda())
    assert bool(got[:3, :4, :16].isnan().all()) and torch.equal(got[3], before[3]) and bool(torch.isfinite(got[:3, :4, 16:]).all())
    _status_clean()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,hd", [("fp4", 64), ("bf16", 128)])
def test_more_rows_than_a_block_has_threads(fmt, hd):
    """1100 ragged rows (the tables' search leaves shared memory, the attention's prefix sum takes several steps), every third without new
    tokens, pairs of rows over the same pages."""
    page = 8
    rows = [((7 * b) % 31, 0 if b % 3 == 2 else 1 + b % 2, 0) for b in range(1100)]
    pages, q_start, lens, start, n, n_pages = _batch(rows, page)
    for b in range(0, 1100, 6):
        total, new = rows[b][0] + rows[b][1], rows[b + 1][1]
        if total >= new:
            pages[b + 1], rows[b + 1], lens[b + 1] = pages[b], (total - new, new, 0), total
    cache, cpu = _random_cache(n_pages, page, 1, hd, fmt)
    q = torch.randn(n, 2, hd).bfloat16()
    _check_attention(q, cache, cpu, rows, pages, q_start, lens, start, _tables(64, 8), None, page=page)
    dev = [t.cuda() for t in (pages, q_start, lens)]
    back = ops.paged_read(cache, *dev, n)
    for x, y in zip(back, ops.paged_read(cpu, pages, q_start, lens, n)):
        assert torch.equal(x.cpu(), y)
    _status_clean()


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,V,dtype,with_draft", [(140, 2, 4100, "float32", True), (700, 1, 1003, "float32", True), (170, 3, 6001, "bfloat16", False), (2, 2, 3, "float32", True),
                                                    (60, 2, 12288, "bfloat16", True), (3, 1, 5, "bfloat16", True)])
def test_verify_kernel_at_every_split_of_a_row(B, N, V, dtype, with_draft):
    """Batches that take 8, 4 and 2 CTAs a row, of 8 and of 16 warps, and vocabularies of less than a group of four."""
    test_verify_kernel(B, N, V, dtype, with_draft)


@pytest.mark.gpu
def test_forward_only_and_refused_caches():
    rows, page = [(20, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, device="cuda")
    cache, _ = _random_cache(n_pages, page, 2, 64, "fp4")
    q = torch.randn(n, 4, 64, device="cuda", requires_grad=True)
    k = torch.randn(n, 2, 64, device="cuda", requires_grad=True)
    for call in (lambda: ops.paged_attention(q, cache, pages, q_start, lens), lambda: ops.paged_append(cache, k, k.detach(), pages, q_start, lens),
                 lambda: ops.paged_append(cache, k.detach(), k, pages, q_start, lens)):
        with pytest.raises(RuntimeError, match="forward only"):
            call()
    with torch.no_grad():
        assert not ops.paged_attention(q, cache, pages, q_start, lens).requires_grad
    big = torch.zeros(5 * 2 * 16 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    x = big[:-8].view(5, 2, 16, 64)
    for match, bad in {"power of two": (x[:, :, :12].contiguous(),) * 2, "32-byte": (big[8:].view(5, 2, 16, 64),) * 2, "contiguous": (x.transpose(1, 2),) * 2, "one type": (x, x.float()),
                       "bfloat16, or uint8": (x.half(), x.half()), "alone": (cache.k, cache.v), "float8": (cache.k, cache.v, cache.k_scale.float(), cache.v_scale.float())}.items():
        with pytest.raises(ValueError, match=match):
            ops.PagedKV(*bad)
    with pytest.raises(RuntimeError, match="16-byte"):
        t = torch.zeros(65 * 8 + 4, device="cuda")[1:521].view(65, 8)
        ops.paged_attention(q.detach(), cache, pages, q_start, lens, rope=(t, t))


@pytest.mark.gpu
def test_two_caches_on_two_streams_at_once():
    """Attention over two caches launched side by side on two streams, many times: each equals its own result alone."""
    rows, page = [(900, 1, 0), (77, 2, 5)], 32
    tabs = _batch(rows, page, device="cuda")
    caches = [_random_cache(tabs[5], page, 2, 64, f, seed=i)[0] for i, f in enumerate(("fp4", "bf16"))]
    q = torch.randn(tabs[4], 8, 64, device="cuda").bfloat16()
    alone = [ops.paged_attention(q, c, *tabs[:3], start=tabs[3]) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    outs = [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, caches)):
            with torch.cuda.stream(s):
                outs[i].append(ops.paged_attention(q, c, *tabs[:3], start=tabs[3]))
    torch.cuda.synchronize()
    for o, want in zip(outs, alone):
        assert all(torch.equal(x, want) for x in o)
    _status_clean()


@pytest.mark.gpu
def test_empty_tables_and_tokens_without_a_rotation():
    """A rope table without positions is refused; a batch of no rows leaves zeros; a token behind the rope table is left out whole, its value as
    well as its key, however its heads are spread over threads."""
    from gdn_hybrid_architecture_ideas_b200.ops import native

    rows, page = [(20, 1, 0)], 16
    pages, q_start, lens, start, n, n_pages = _batch(rows, page, device="cuda")
    cache, _ = _random_cache(n_pages, page, 2, 64, "bf16")
    q = torch.randn(n, 4, 64, device="cuda").bfloat16()
    k = torch.randn(n, 2, 64, device="cuda").bfloat16()
    none = tuple(torch.zeros(0, 8, device="cuda") for _ in range(2))
    for call in (lambda: ops.paged_attention(q, cache, pages, q_start, lens, rope=none), lambda: ops.paged_append(cache, k, k, pages, q_start, lens, rope=none)):
        with pytest.raises(RuntimeError, match="without positions"):
            call()
    before = cache.k.clone(), cache.v.clone()
    no_rows = (pages[:0], q_start[:1], lens[:0])
    assert not ops.paged_attention(q, cache, *no_rows).any() and not ops.paged_read(cache, *no_rows, n)[0].any()
    ops.paged_append(cache, k, k, *no_rows)
    _status_clean()
    ops.paged_append(cache, k, k, pages, q_start, lens, rope=tuple(t.cuda() for t in _tables(20, 8)))          # position 20 needs 21 entries
    with pytest.raises(RuntimeError, match="status 305"):
        native.check_status()
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
