"""A paged key/value cache in bfloat16 or 4 bits, and the PyTorch statements of the ops over it (the CPU path and the
oracle of the kernels in csrc/paged.cu and csrc/paged_attention.cu; the public entry points are in `ops`).

Layout. A pool of pages, each `page_size` positions of every KV head:

    k, v              [n_pages, Hkv, page_size, hd]        the values (bfloat16 on CUDA; any floating type on the CPU)
  or, in 4 bits,
    k, v              [n_pages, Hkv, page_size, hd / 2]    uint8: E2M1 codes, the even channel in the low four bits
    k_scale, v_scale  [n_pages, Hkv, page_size, hd / 16]   float8_e4m3fn: one scale for 16 channels

so the entries of one head in one page are contiguous (a 64-position page of 64 channels: 2 KB of codes, 256 bytes of
scales). 4 bits cost 0.5625 bytes a value against 2: 0.28 of the bytes.

The 4-bit value: s = e4m3(max |x| / 6) over the 16 channels, code = e2m1(x / s), both to nearest with ties to even; read
back as code * s, which is exact in bfloat16 (2 + 4 significant bits). x is held to +-2688 (the largest value, 6 * 448)
before; the format has no infinities and no NaN: an infinity is held as 2688 of its sign and NaN as 0. A block whose
largest magnitude rounds to no scale (below 6 * 2^-10) is held as zeros.

Rows. Every op takes the same description of a batch: `pages` int32 [B, width], the page ids of each row in order of
position (entries past the row's last page are not read); `q_start` int32 [B + 1], row b's NEW tokens are the packed
tokens q_start[b] .. q_start[b + 1]; `lens` int32 [B], the row's cached positions including those, so its packed token j sits
at position lens[b] - (q_start[b + 1] - j); `start` int32 [B] (default 0), the row's first visible position, from which its
rotary positions count. Packed tokens that no row owns (before q_start[0], from q_start[B] on, of a row whose range is refused) are
padding: no op reads or writes for them, except that an op which allocates its own output leaves zeros there. Rows may have
no tokens. What a token does not see may hold anything; a cached value that is infinite or NaN reaches the tokens that see it (on CUDA a
key of that kind makes their outputs NaN).
"""

from __future__ import annotations

import operator

import torch

E2M1_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E4M3 = torch.float8_e4m3fn
BLOCK = 16
LARGEST = 6.0 * 448.0
NATIVE_CHECK = None             # set by `ops`: where the kernels run, checks a cache on a GPU (in the binding, once) and says so


class PagedKV:
    """The cache's tensors (see the module's head for the layout). `PagedKV.zeros` allocates an empty one."""

    __slots__ = ("_k", "_v", "_ks", "_vs", "native")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        self._k, self._v, self._ks, self._vs = k, v, k_scale, v_scale          # (fixed: the binding holds them too)
        self.native = None              # the CUDA binding's form of these tensors (ops/native.py)
        if k.is_cuda and NATIVE_CHECK is not None and NATIVE_CHECK(self):
            return
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"PagedKV: k and v are [pages, kv heads, page size, channels] of one type on one device, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("PagedKV: k and v are contiguous")
        if k.dtype == torch.uint8:
            want = (*k.shape[:3], k.shape[3] // 8)
            if k.shape[3] % 8 or k_scale is None or v_scale is None:
                raise ValueError("PagedKV: uint8 codes come with k_scale and v_scale, for head dimensions that are multiples of 16")
            for s in (k_scale, v_scale):
                if s.dtype != E4M3 or s.shape != want or not s.is_contiguous() or s.device != k.device:
                    raise ValueError(f"PagedKV: scales are contiguous float8_e4m3fn {want} beside the codes, got {tuple(s.shape)} {s.dtype}")
        elif not k.dtype.is_floating_point or k.dtype.itemsize < 2 or k_scale is not None or v_scale is not None:
            raise ValueError(f"PagedKV: uint8 codes with scales, or values of a floating type without, got {k.dtype}")
        if k.shape[1] < 1:
            raise ValueError("PagedKV: at least one head")
        page = k.shape[2]
        if page < 8 or page & (page - 1):
            raise ValueError(f"PagedKV: the page size is a power of two from 8 on, got {page}")

    @classmethod
    def zeros(cls, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, fmt: str = "bf16", device="cpu", make=None) -> "PagedKV":
        """fmt "bf16" (float32 and float64 on the CPU as "fp32" / "fp64") or "fp4". make(name, shape, dtype): where the tensors
        come from (default torch.zeros)."""
        make = make or (lambda name, shape, dtype: torch.zeros(shape, dtype=dtype, device=device))
        lead = (n_pages, n_kv_heads, page_size)
        if fmt == "fp4":
            if head_dim % BLOCK:
                raise ValueError(f"PagedKV: 4-bit entries hold blocks of {BLOCK} channels, got head dimension {head_dim}")
            kv = [make(n, (*lead, head_dim // 2), torch.uint8) for n in ("k", "v")]
            # (float8 has no fill kernel everywhere: the bytes are made and viewed)
            return cls(*kv, *(make(n, (*lead, head_dim // BLOCK), torch.uint8).view(E4M3) for n in ("k_scale", "v_scale")))
        dtypes = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp64": torch.float64}
        if fmt not in dtypes:
            raise ValueError(f"PagedKV: fmt {fmt!r}: 'bf16', 'fp4' (on the CPU also 'fp32', 'fp64')")
        return cls(*(make(n, (*lead, head_dim), dtypes[fmt]) for n in ("k", "v")))

    k, v, k_scale, v_scale = (property(operator.attrgetter(n)) for n in ("_k", "_v", "_ks", "_vs"))

    @property
    def fp4(self) -> bool:
        return self.k.dtype == torch.uint8

    @property
    def n_pages(self) -> int:
        return self.k.shape[0]

    @property
    def n_kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] * (2 if self.fp4 else 1)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None)


# ------------------------------------------------------------------------------------------------------------ 4 bits

def fp4_quantize(x: torch.Tensor):
    """x [..., d] -> (codes uint8 [..., d / 2], scales float8_e4m3fn [..., d / 16])."""
    from .lowp import e2m1_round

    b = torch.nan_to_num(x.float(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST).unflatten(-1, (-1, BLOCK))
    scale = (b.abs().amax(-1) / 6.0).to(E4M3)
    s = scale.float()[..., None]
    y = torch.where(s > 0, b / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(b))
    mag = e2m1_round(y.abs())
    code = torch.searchsorted(torch.tensor(E2M1_GRID, device=x.device), mag).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | (code[..., 1] << 4), scale


def fp4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float32 values of codes [..., d / 2] and scales [..., d / 16]."""
    grid = torch.tensor(E2M1_GRID + tuple(-g for g in E2M1_GRID), device=codes.device)
    x = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
    return (x.unflatten(-1, (-1, BLOCK)) * scales.float()[..., None]).flatten(-2)


# ------------------------------------------------------------------------------------------------------------ rows

def _check_rows(cache: PagedKV, pages, q_start, lens, start, n: int, what: str):
    """The host-side form of the checks that the kernels make per row; returns python lists."""
    B = lens.shape[0]
    if pages.dim() != 2 or pages.shape[0] != B or q_start.shape != (B + 1,) or lens.dim() != 1 or (start is not None and start.shape != (B,)):
        raise ValueError(f"{what}: pages [B, width], q_start [B + 1], lens [B] and start [B] of one batch")
    for name, t in (("pages", pages), ("q_start", q_start), ("lens", lens), ("start", start)):
        if t is not None and t.dtype != torch.int32:
            raise ValueError(f"{what}: {name} is int32, got {t.dtype}")
    qs, ls = q_start.tolist(), lens.tolist()
    st = [0] * B if start is None else start.tolist()
    table = pages.tolist()
    P, room = cache.page_size, pages.shape[1] * cache.page_size
    for b in range(B):
        m = qs[b + 1] - qs[b]
        if qs[b] < 0 or m < 0 or qs[b + 1] > n:
            raise ValueError(f"{what}: q_start of row {b} ({qs[b]} .. {qs[b + 1]}) is not a range of the {n} packed tokens")
        if not m <= ls[b] <= room:
            raise ValueError(f"{what}: row {b} has {ls[b]} cached positions with {m} new ones; its pages hold {room}")
        if not 0 <= st[b] <= ls[b]:
            raise ValueError(f"{what}: start {st[b]} of row {b} is not in 0 .. {ls[b]}")
    return qs, ls, st, table


def _pages_of(cache: PagedKV, table, lo: int, hi: int, b: int, what: str):
    """Page ids that hold positions lo .. hi of row b, as a tensor, checked."""
    P = cache.page_size
    ids = table[b][lo // P:-(-hi // P)]
    bad = [i for i in ids if not 0 <= i < cache.n_pages]
    if bad:
        raise ValueError(f"{what}: page id {bad[0]} of row {b} is not one of the cache's {cache.n_pages} pages")
    return torch.tensor(ids, dtype=torch.long, device=cache.k.device)


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [..., H, hd] by cos, sin [..., half]: channel i with channel i + half, in the wider of the two types."""
    half = cos.shape[-1]
    c, s = cos[..., None, :], sin[..., None, :]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def _check_rope(rope, hd: int, need: int, what: str):
    cos, sin = rope
    if cos.dim() != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > hd:
        raise ValueError(f"{what}: rope is (cos, sin), each [positions, rotary pairs] with at most {hd // 2} pairs")
    if need > cos.shape[0]:
        raise ValueError(f"{what}: rotary position {need - 1} lies behind the rope table's {cos.shape[0]} positions")
    return cos, sin


# ------------------------------------------------------------------------------------------------------------ statements

def paged_append(cache: PagedKV, k, v, pages, q_start, lens, start=None, rope=None) -> None:
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (cache.n_kv_heads, cache.head_dim):
        raise ValueError(f"paged_append: k, v [n, {cache.n_kv_heads}, {cache.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
    qs, ls, st, table = _check_rows(cache, pages, q_start, lens, start, k.shape[0], "paged_append")
    P = cache.page_size
    for b in range(len(ls)):
        m = qs[b + 1] - qs[b]
        if m == 0:
            continue
        lo, hi = ls[b] - m, ls[b]
        ids = _pages_of(cache, table, lo, hi, b, "paged_append")
        pos = torch.arange(lo, hi, device=k.device)
        at, slot = ids[pos // P - lo // P], pos % P
        kb, vb = k[qs[b]:qs[b + 1]], v[qs[b]:qs[b + 1]]
        if rope is not None:
            if lo < st[b]:
                raise ValueError(f"paged_append: row {b} rotates position {lo}, which lies before its start {st[b]}")
            cos, sin = _check_rope(rope, cache.head_dim, hi - st[b], "paged_append")
            # 64 bits, held in 32 (in 64 where the cache is): the 4-bit grid's borders then lie where the formula has them
            kb = _rotate(kb.double(), cos[pos - st[b]].double(), sin[pos - st[b]].double())
            kb = kb if cache.k.dtype == torch.float64 else kb.float()
        if cache.fp4:
            for x, code, scale in ((kb, cache.k, cache.k_scale), (vb, cache.v, cache.v_scale)):
                c, s = fp4_quantize(x)
                code[at, :, slot] = c
                scale.view(torch.uint8)[at, :, slot] = s.view(torch.uint8)
        else:
            cache.k[at, :, slot] = kb.to(cache.k.dtype)
            cache.v[at, :, slot] = vb.to(cache.v.dtype)


def _entries(cache: PagedKV, table, lo: int, hi: int, b: int, what: str):
    """(k, v) [hi - lo, Hkv, hd] of positions lo .. hi of row b (fp4: float32 values)."""
    P = cache.page_size
    ids = _pages_of(cache, table, lo, hi, b, what)
    cut = slice(lo - lo // P * P, hi - lo // P * P)

    def rows(t):
        return t[ids].transpose(1, 2).flatten(0, 1)[cut]
    if not cache.fp4:
        return rows(cache.k), rows(cache.v)
    return tuple(fp4_values(rows(c), rows(s.view(torch.uint8)).contiguous().view(E4M3)) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))


def paged_read(cache: PagedKV, pages, q_start, lens, n: int, out=None):
    qs, ls, _, table = _check_rows(cache, pages, q_start, lens, None, n, "paged_read")
    dt = torch.bfloat16 if cache.fp4 else cache.k.dtype
    shape = (n, cache.n_kv_heads, cache.head_dim)
    if out is None:
        out = tuple(torch.zeros(shape, dtype=dt, device=cache.k.device) for _ in range(2))
    elif any(o.shape != shape or o.dtype != dt for o in out):
        raise ValueError(f"paged_read: out is two {dt} tensors {shape}")
    for b in range(len(ls)):
        m = qs[b + 1] - qs[b]
        if m:
            for o, x in zip(out, _entries(cache, table, ls[b] - m, ls[b], b, "paged_read")):
                o[qs[b]:qs[b + 1]] = x.to(dt)
    return out


def paged_attention(q, cache: PagedKV, pages, q_start, lens, start=None, rope=None, cap=None, scale=None, out=None):
    n, hq, hd = q.shape
    hkv = cache.n_kv_heads
    if hd != cache.head_dim or hq % hkv:
        raise ValueError(f"paged_attention: q [n, a multiple of {hkv}, {cache.head_dim}], got {tuple(q.shape)}")
    if cap is not None and (rope is None or cap < 1):
        raise ValueError("paged_attention: a rotary distance cap is an integer >= 1 beside a rope table")
    qs, ls, st, table = _check_rows(cache, pages, q_start, lens, start, n, "paged_attention")
    scale = hd ** -0.5 if scale is None else scale
    dt = torch.promote_types(torch.promote_types(q.dtype, torch.float32), torch.float32 if cache.fp4 else cache.k.dtype)
    odt = torch.bfloat16 if q.is_cuda or torch.bfloat16 in (q.dtype, cache.k.dtype) else q.dtype
    if out is None:
        out = torch.zeros(n, hq, hd, dtype=odt, device=q.device)
    elif out.shape != q.shape or out.dtype != odt:
        raise ValueError(f"paged_attention: out is a {odt} tensor {tuple(q.shape)}")
    for b in range(len(ls)):
        m = qs[b + 1] - qs[b]
        if m == 0:
            continue
        first, hi = st[b], ls[b]
        qb = q[qs[b]:qs[b + 1]].to(dt)
        p = torch.arange(hi - m, hi, device=q.device)
        if rope is not None:
            cos, sin = _check_rope(rope, hd, max(hi - first, 0 if cap is None else cap + 1), "paged_attention")
        if hi <= first:
            out[qs[b]:qs[b + 1]] = 0
            continue
        k, v = (x.to(dt) for x in _entries(cache, table, first, hi, b, "paged_attention"))
        t = torch.arange(first, hi, device=q.device)

        def scores(qx, kx):
            return torch.einsum("nhgd,thd->hgnt", qx.view(m, hkv, hq // hkv, hd), kx)
        at = (p - first).clamp(min=0)
        if rope is None:
            a = scores(qb, k)
        else:
            near = _rotate(qb, cos[at].to(dt), sin[at].to(dt))
            if cap is None:
                a = scores(near, k)
            else:
                a = scores(near, _rotate(k, cos[t - first].to(dt), sin[t - first].to(dt)))
                far = scores(_rotate(qb, cos[cap].to(dt).expand(m, -1), sin[cap].to(dt).expand(m, -1)), k)
                a = torch.where(p[:, None] - t > cap, far, a)
        seen = t <= p[:, None]
        a = (a * scale).masked_fill(~seen, float("-inf"))
        top = a.amax(-1, keepdim=True)
        w = torch.exp(a - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, torch.zeros_like(w), w / total)
        # a masked entry's value does not enter, whatever it holds
        clean = bool(torch.isfinite(v).all())
        if clean:
            o = torch.einsum("hgnt,thd->nhgd", w, v)
        else:
            o = torch.stack([torch.einsum("hgt,thd->hgd", w[:, :, i, :int(seen[i].sum())], v[:int(seen[i].sum())]) for i in range(m)])
        out[qs[b]:qs[b + 1]] = o.reshape(m, hq, hd).to(odt)
    return out


def verify_drafts(target, draft, drafts, u_accept, u_sample, n_drafts=None):
    B, N1, V = target.shape
    N = N1 - 1
    if drafts.shape != (B, N) or u_accept.shape != (B, N) or u_sample.shape != (B,) or (draft is not None and draft.shape != (B, N, V)) \
            or (n_drafts is not None and n_drafts.shape != (B,)):
        raise ValueError(f"verify_drafts: target [B, N + 1, V], draft [B, N, V], drafts and u_accept [B, N], u_sample and n_drafts [B]; got "
                         f"target {tuple(target.shape)}, drafts {tuple(drafts.shape)}")
    tokens = torch.full((B, N1), -1, dtype=torch.long, device=target.device)
    kept = torch.zeros(B, dtype=torch.long, device=target.device)
    for b in range(B):
        m = N if n_drafts is None else int(n_drafts[b])
        if not 0 <= m <= N:
            raise ValueError(f"verify_drafts: n_drafts[{b}] = {m} is not in 0 .. {N}")
        i = 0
        while i < m:
            x = int(drafts[b, i])
            if not 0 <= x < V:
                raise ValueError(f"verify_drafts: drafted token {x} of row {b} is not in the vocabulary of {V}")
            q = 1.0 if draft is None else float(draft[b, i, x].double())
            if not float(u_accept[b, i].double()) * q < float(target[b, i, x].double()):
                break
            tokens[b, i] = x
            i += 1
        p = target[b, i].double()
        p = torch.where(p > 0, p, torch.zeros_like(p))
        w = p
        if i < m:
            if draft is None:
                w = p.clone()
                w[int(drafts[b, i])] = 0
            else:
                w = p - draft[b, i].double()
                w = torch.where(w > 0, w, torch.zeros_like(w))
            if not float(w.sum()) > 0:
                w = p
        upto = w.cumsum(0)
        over = torch.nonzero(upto > u_sample[b].double() * upto[-1])
        live = torch.nonzero(w > 0)
        tokens[b, i] = int(over[0]) if len(over) else (int(live[-1]) if len(live) else 0)
        kept[b] = i
    return tokens, kept
