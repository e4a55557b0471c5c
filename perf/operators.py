"""The paged serving operators of this framework, as a measurement sees them: appending keys and values to a paged
cache (bfloat16 or 4 bits) with the position rotation on the way, reading cached entries back, attention of one or a
few new tokens a row over such a cache, and the verification of drafted tokens against the target's probabilities.

`run` computes a case in elementary torch operations (32 bits; 64 where a value is about to be rounded to the cache's
grid, and for sums over a vocabulary), or, with `own` set, through the framework's public calls.

The cache: pages of `page` positions, tensors [pages, kv heads, page, ...]. bfloat16 holds the values. The 4-bit form
holds E2M1 codes (two channels a byte, the even channel in the low half) and one E4M3 scale for 16 channels: the block's
largest magnitude / 6, rounded to E4M3; a code is the value / scale rounded to the nearest E2M1 value, ties to even.
Row b owns the packed new tokens q_start[b] .. q_start[b + 1], which are its last cached positions before lens[b].
"""

import math
import random

import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
THETA = 1.0e7


# ------------------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one new token of one row joins a bfloat16 cache (2 key heads of 256 channels, 64 of them rotary): pure latency
        {"name": "append_one_token", "op": "append", "fmt": "bf16", "rows": 1, "before": 777, "new": 1, "even": True, "kv_heads": 2, "head_dim": 256, "page": 64, "rot": 64},
        # a decode step of 64 rows at 32k cached positions: one token a row into the 4-bit cache, and back as stored
        {"name": "append_step_fp4", "op": "append", "fmt": "fp4", "rows": 64, "before": 32767, "new": 1, "even": True, "kv_heads": 4, "head_dim": 64, "page": 64, "rot": 16},
        # ragged prompts enter a bfloat16 cache, some behind a cached prefix (2 key heads of 128 channels)
        {"name": "append_prompts_bf16", "op": "append", "fmt": "bf16", "rows": 9, "before": 500, "new": 4099, "even": False, "kv_heads": 2, "head_dim": 128, "page": 16, "rot": 32},
        # a prefill batch of long ragged prompts enters the 4-bit cache (8 key heads of 64 channels)
        {"name": "append_prompts_fp4", "op": "append", "fmt": "fp4", "rows": 16, "before": 0, "new": 8192, "even": False, "kv_heads": 8, "head_dim": 64, "page": 64, "rot": 16},
        # a short bfloat16 row is read back (a chunk of a prompt attends over what is cached)
        {"name": "read_bf16", "op": "read", "fmt": "bf16", "rows": 3, "before": 0, "new": 1001, "even": False, "kv_heads": 2, "head_dim": 256, "page": 32, "rot": 0},
        # ragged 4-bit rows are read back whole
        {"name": "read_fp4", "op": "read", "fmt": "fp4", "rows": 16, "before": 0, "new": 8192, "even": False, "kv_heads": 8, "head_dim": 64, "page": 64, "rot": 0},
        # one row, one new token, an ordinary context: the latency of a single user's step (8 query heads, 2 key heads of 128)
        {"name": "attend_one_row", "op": "attend", "fmt": "fp4", "rows": 1, "ctx": 4097, "q": 1, "even": True, "heads": 8, "kv_heads": 2, "head_dim": 128, "page": 64, "rot": 32, "cap": 0, "docs": False},
        # a full decode batch: 64 rows of 32k positions, 16 query heads over 4 key heads of 64, rotary distance cap 2048
        {"name": "attend_64x32k", "op": "attend", "fmt": "fp4", "rows": 64, "ctx": 32768, "q": 1, "even": True, "heads": 16, "kv_heads": 4, "head_dim": 64, "page": 64, "rot": 16, "cap": 2048, "docs": False},
        # drafted tokens of ragged rows scored in one pass: up to 5 queries a row, 32 query heads over 8 key heads
        {"name": "attend_drafts", "op": "attend", "fmt": "fp4", "rows": 24, "ctx": 16001, "q": 5, "even": False, "heads": 32, "kv_heads": 8, "head_dim": 64, "page": 32, "rot": 16, "cap": 2048, "docs": True},
        # the bfloat16 cache, wide heads (16 query heads over 2 key heads of 256), ragged rows
        {"name": "attend_bf16", "op": "attend", "fmt": "bf16", "rows": 12, "ctx": 9001, "q": 1, "even": False, "heads": 16, "kv_heads": 2, "head_dim": 256, "page": 16, "rot": 64, "cap": 0, "docs": False},
        # three drafted tokens of one row against a 32k vocabulary: latency
        {"name": "verify_one_row", "op": "verify", "rows": 1, "drafts": 3, "vocab": 32768, "dtype": "float32", "even": True},
        # a batch of ragged drafts against a 64,000-token vocabulary
        {"name": "verify_batch", "op": "verify", "rows": 96, "drafts": 5, "vocab": 64000, "dtype": "float32", "even": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "attend", "verify"])
    if op == "verify":
        rows, drafts = _log(rng, 1, 96), rng.randint(1, 6)
        return {"op": op, "rows": rows, "drafts": drafts, "vocab": _log(rng, 300, 64000), "dtype": rng.choice(["float32", "float32", "bfloat16"]), "even": rng.random() < 0.3}
    fmt = rng.choice(["fp4", "fp4", "bf16"])
    head_dim = rng.choice([64, 64, 128, 256])
    rot = {64: rng.choice([16, 32, 64]), 128: rng.choice([32, 64]), 256: 64}[head_dim]
    page = rng.choice([16, 32, 64, 128])
    if op in ("append", "read"):
        kv = rng.choice([1, 2, 3, 4, 8])
        rows = _log(rng, 1, 64)
        new = rng.choice([1, _log(rng, 2, 8192)])
        new = max(1, min(new, (65536 * 8 * 64) // (rows * kv * head_dim)))
        return {"op": op, "fmt": fmt, "rows": rows, "before": rng.choice([0, _log(rng, 1, 8192)]), "new": new, "even": rng.random() < 0.4, "kv_heads": kv,
                "head_dim": head_dim, "page": page, "rot": rot if op == "append" and rng.random() < 0.8 else 0}
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    q = rng.choice([1, 1, rng.randint(2, 9)])
    ctx = _log(rng, 1, 32768)
    most = 64 * 32768 * 4 * 64
    rows = _log(rng, 1, max(1, min(128, most // (4 * ctx * kv * head_dim))))
    cap = rng.choice([0, rng.choice([1, 96, 1024, 2048])])
    return {"op": op, "fmt": fmt, "rows": rows, "ctx": max(q, ctx), "q": q, "even": rng.random() < 0.4, "heads": kv * group, "kv_heads": kv, "head_dim": head_dim,
            "page": page, "rot": rng.choice([rot, rot, 0]) if not cap else rot, "cap": cap, "docs": rng.random() < 0.4}


def _rows(case):
    """(positions before, new positions, first visible position) of every row, from the case alone."""
    r = random.Random("%s %s" % (case["rows"], case.get("ctx", case.get("new"))))
    out = []
    for _ in range(case["rows"]):
        if case["op"] == "attend":
            n = case["q"] if case["even"] else r.randint(1, case["q"])
            total = case["ctx"] if case["even"] else max(n, int(case["ctx"] * r.uniform(0.05, 1.0)))
            out.append((total - n, n, r.randrange(0, total - n + 1) // 3 if case["docs"] else 0))
        else:
            n = case["new"] if case["even"] else r.randint(1, case["new"])
            out.append((case["before"] if case["even"] else r.randint(0, case["before"]), n, 0))
    return out


# ------------------------------------------------------------------------------------------------------------ inputs

def _quantise(x):
    """x [..., d] float32 -> (codes uint8 [..., d / 2], scales float8_e4m3fn [..., d / 16])."""
    b = x.clamp(-2688.0, 2688.0).unflatten(-1, (-1, 16))
    scale = (b.abs().amax(-1) / 6.0).to(torch.float8_e4m3fn)
    s = scale.float()[..., None]
    y = torch.where(s > 0, b / s, torch.zeros_like(b))
    a = y.abs().clamp(max=6.0)
    a = torch.where(a < 2, torch.round(a * 2) * 0.5, torch.where(a < 4, torch.round(a), torch.round(a * 0.5) * 2))
    grid = torch.tensor(E2M1, device=x.device)
    code = torch.searchsorted(grid, a.contiguous()).to(torch.uint8) + 8 * torch.signbit(y).to(torch.uint8)
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] + 16 * code[..., 1], scale


def _pool(g, n_pages, case):
    """A page pool whose positions all hold earlier tokens: normed keys and values of about unit size."""
    shape = (case["kv_heads"], case["page"], case["head_dim"])
    if case["fmt"] == "bf16":
        return {n: torch.randn(n_pages, *shape, device="cuda", generator=g, dtype=torch.bfloat16) for n in ("k", "v")}
    out = {}
    for n in ("k", "v"):
        codes = torch.empty(n_pages, *shape[:2], shape[2] // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(n_pages, *shape[:2], shape[2] // 16, dtype=torch.float8_e4m3fn, device="cuda")
        step = max(1, (1 << 26) // math.prod(shape))
        for lo in range(0, n_pages, step):
            hi = min(n_pages, lo + step)
            codes[lo:hi], scales[lo:hi] = _quantise(torch.randn(hi - lo, *shape, device="cuda", generator=g))
        out[n], out[n + "_scale"] = codes, scales
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    rows, page = _rows(case), case["page"]
    lens = [a + n for a, n, _ in rows]
    need = [-(-t // page) for t in lens]
    n_pages, width = sum(need) + 3, max(need) + 1
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(rows), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q_start = [0]
    for _, n, _ in rows:
        q_start.append(q_start[-1] + n)
    s = {"case": dict(case), "pages": table, "n": q_start[-1], "n_max": max(n for _, n, _ in rows),
         "q_start": torch.tensor(q_start, dtype=torch.int32, device="cuda"), "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "start": torch.tensor([c for _, _, c in rows], dtype=torch.int32, device="cuda"), "rope": None}
    s.update(_pool(g, n_pages, case))
    if case["rot"]:
        half = case["rot"] // 2
        ang = torch.arange(max(max(lens), case.get("cap", 0) + 1), dtype=torch.float64, device="cuda")[:, None]
        ang = ang * THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        s["rope"] = (ang.cos().float(), ang.sin().float())
    hd = case["head_dim"]
    if case["op"] == "append":
        for n in ("new_k", "new_v"):
            s[n] = torch.randn(s["n"], case["kv_heads"], hd, device="cuda", generator=g, dtype=torch.bfloat16)
    if case["op"] == "attend":
        # normed queries times a learned gain: logits of a spread of about two
        s["q"] = (2.0 * torch.randn(s["n"], case["heads"], hd, device="cuda", generator=g)).to(torch.bfloat16)
    return s


def _prepare_verify(case, g):
    B, N, V, dt = case["rows"], case["drafts"], case["vocab"], getattr(torch, case["dtype"])
    logits = 2.5 * torch.randn(B, N + 1, V, device="cuda", generator=g)
    target = torch.softmax(logits, -1).to(dt)
    draft = torch.softmax(logits[:, :N] + 0.7 * torch.randn(B, N, V, device="cuda", generator=g), -1).to(dt)
    drafts = torch.multinomial(draft.float().reshape(B * N, V), 1, generator=g).view(B, N)
    r = random.Random("%d %d" % (B, N))
    count = [N if case["even"] else r.randint(0, N) for _ in range(B)]
    return {"case": dict(case), "target": target, "draft": draft, "drafts": drafts, "u_accept": torch.rand(B, N, device="cuda", generator=g),
            "u_sample": torch.rand(B, device="cuda", generator=g), "n_drafts": torch.tensor(count, dtype=torch.int32, device="cuda")}


# ------------------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "append":
        return _append(s)
    if op == "read":
        return _read(s)
    if op == "attend":
        return _attend(s)
    return _verify(s)


def _run_own(s):
    from gdn_hybrid_architecture_ideas_b200 import ops

    op = s["case"]["op"]
    if op == "verify":
        return ops.verify_drafts(s["target"], s["draft"], s["drafts"], s["u_accept"], s["u_sample"], n_drafts=s["n_drafts"])
    cache = ops.PagedKV(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
    if op == "append":
        ops.paged_append(cache, s["new_k"], s["new_v"], s["pages"], s["q_start"], s["lens"], rope=s["rope"])
        if s["case"]["fmt"] == "bf16":
            return s["k"], s["v"]
        return ops.paged_read(cache, s["pages"], s["q_start"], s["lens"], s["n"])
    if op == "read":
        return ops.paged_read(cache, s["pages"], s["q_start"], s["lens"], s["n"])
    return ops.paged_attention(s["q"], cache, s["pages"], s["q_start"], s["lens"], start=s["start"], rope=s["rope"], cap=s["case"]["cap"] or None)


def _places(s):
    """(row, position) of every packed token."""
    j = torch.arange(s["n"], device="cuda")
    row = torch.searchsorted(s["q_start"][1:], j.int(), right=True)
    return row, s["lens"][row] - (s["q_start"][row + 1] - j)


def _turn(x, cos, sin):
    """The first 2 * cos.shape[-1] channels of x rotated: channel i with channel i + half."""
    half = cos.shape[-1]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _values(codes, scales):
    """float32 values of 4-bit codes [..., d / 2] and their scales [..., d / 16]."""
    grid = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pair = torch.stack([grid[byte & 15], grid[byte >> 4]], -1)
    x = pair.index_select(0, codes.reshape(-1).int()).view(*codes.shape[:-1], -1)
    return (x.unflatten(-1, (-1, 16)) * scales.float()[..., None]).flatten(-2)


def _append(s):
    page = s["case"]["page"]
    row, pos = _places(s)
    k, v = s["new_k"].double(), s["new_v"].float()
    if s["rope"] is not None:
        k = _turn(k, s["rope"][0][pos].double()[:, None], s["rope"][1][pos].double()[:, None])
    at, slot = s["pages"][row, pos // page], pos % page
    if s["case"]["fmt"] == "bf16":
        s["k"][at, :, slot], s["v"][at, :, slot] = k.float().bfloat16(), s["new_v"]
        return s["k"], s["v"]
    s["k"][at, :, slot], s["k_scale"][at, :, slot] = _quantise(k.float())
    s["v"][at, :, slot], s["v_scale"][at, :, slot] = _quantise(v)
    return _read(s)


def _read(s):
    page = s["case"]["page"]
    row, pos = _places(s)
    at, slot = s["pages"][row, pos // page], pos % page
    if s["case"]["fmt"] == "bf16":
        return s["k"][at, :, slot], s["v"][at, :, slot]
    return tuple(_values(s[n][at, :, slot], s[n + "_scale"].view(torch.uint8)[at, :, slot].view(torch.float8_e4m3fn)).bfloat16() for n in ("k", "v"))


def _gather(s, name):
    """[rows, positions, kv heads, head_dim] float32 of the rows' pages."""
    at = s["pages"].clamp(min=0)
    x = s[name][at]
    x = x.float() if s["case"]["fmt"] == "bf16" else _values(x, s[name + "_scale"].view(torch.uint8)[at].view(torch.float8_e4m3fn))
    return x.transpose(2, 3).flatten(1, 2)


def _attend(s):
    c = s["case"]
    B, N, hkv, hd, G, cap = c["rows"], s["n_max"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"], c["cap"]
    row, pos = _places(s)
    i = torch.arange(s["n"], device="cuda") - s["q_start"][row]
    where = torch.zeros(B, N, dtype=torch.long, device="cuda")
    where[row, i] = pos.long()
    at = (where - s["start"][:, None]).clamp(min=0)

    def padded(q):
        x = torch.zeros(B, N, hkv, G, hd, device="cuda")
        x[row, i] = q.float().view(-1, hkv, G, hd)
        return x

    def scores(q, k):
        return torch.einsum("bnhgd,bthd->bhgnt", q, k)

    q, k = padded(s["q"]), _gather(s, "k")
    t = torch.arange(k.shape[1], device="cuda")
    if s["rope"] is not None:
        cos, sin = s["rope"]
        near = _turn(q, cos[at][:, :, None, None], sin[at][:, :, None, None])
        if cap:
            kt = (t - s["start"][:, None]).clamp(min=0, max=cos.shape[0] - 1)
            a = scores(near, _turn(k, cos[kt][:, :, None], sin[kt][:, :, None]))
            far = (where[:, :, None] - t) > cap
            a = torch.where(far[:, None, None], scores(_turn(q, cos[cap], sin[cap]), k), a)
        else:
            a = scores(near, k)
    else:
        a = scores(q, k)
    del k
    seen = (t <= where[:, :, None]) & (t >= s["start"][:, None, None])
    a = (a * hd ** -0.5).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.einsum("bhgnt,bthd->bnhgd", p, _gather(s, "v"))
    return o[row, i].reshape(-1, c["heads"], hd).bfloat16()


def _verify(s):
    target, draft, drafts, n = s["target"], s["draft"], s["drafts"], s["n_drafts"]
    B, N = drafts.shape
    p = target[:, :N].gather(2, drafts[:, :, None])[:, :, 0].double()
    q = draft.gather(2, drafts[:, :, None])[:, :, 0].double()
    i = torch.arange(N, device="cuda")
    ok = (s["u_accept"].double() * q < p) & (i < n[:, None])
    kept = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device="cuda")
    last = target[b, kept].double()
    rest = (last - draft[b, kept.clamp(max=N - 1)].double()).clamp(min=0)
    rest = torch.where((kept < n)[:, None] & (rest.sum(1, keepdim=True) > 0), rest, last)
    upto = rest.cumsum(1)
    pick = (upto <= s["u_sample"].double()[:, None] * upto[:, -1:]).sum(1)
    pick = torch.minimum(pick, ((rest > 0) * torch.arange(rest.shape[1], device="cuda")).amax(1))
    j = torch.arange(N + 1, device="cuda")
    drafted = torch.cat([drafts, drafts[:, :1]], 1)
    tokens = torch.where(j < kept[:, None], drafted, torch.where(j == kept[:, None], pick[:, None], -1))
    return tokens, kept


# ------------------------------------------------------------------------------------------------------------ what it costs

def work(case):
    if case["op"] == "verify":
        # the row of target and draft probabilities that the last token is drawn from (a bonus token needs the target's alone)
        B, N = case["rows"], case["drafts"]
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": B * (2 * case["vocab"] * size + N * (2 * size + 12) + 16 + 8 * (N + 2)), "flops": 3 * B * case["vocab"]}
    hd, hkv = case["head_dim"], case["kv_heads"]
    entry = hkv * (2 * hd * 2 if case["fmt"] == "bf16" else 2 * (hd // 2 + hd // 16))
    rows = _rows(case)
    n = sum(m for _, m, _ in rows)
    if case["op"] == "append":
        back = 0 if case["fmt"] == "bf16" else entry + 2 * hkv * hd * 2      # what is stored in 4 bits is read back as values
        return {"bytes": n * (2 * hkv * hd * 2 + entry + back + 4 * case["rot"]), "flops": n * hkv * (3 * case["rot"] + 4 * hd)}
    if case["op"] == "read":
        return {"bytes": n * (entry + 2 * hkv * hd * 2), "flops": 2 * n * hkv * hd}
    seen = sum(a + m - c for a, m, c in rows)
    pairs = sum(m * (a - c) + m * (m + 1) // 2 for a, m, c in rows)
    return {"bytes": seen * entry + 2 * n * case["heads"] * hd * 2 + 4 * case["rot"] * min(seen, case["ctx"]), "flops": 4 * pairs * case["heads"] * hd}


# ------------------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify":
        return _exact_verify(s)
    page, rows = case["page"], _rows(case)
    q_start, table = s["q_start"].tolist(), s["pages"].tolist()
    if case["op"] == "append":
        return _exact_append(s, case, rows, q_start, table)
    if case["op"] == "read":
        ks, vs = [], []
        for b, (a, n, _) in enumerate(rows):
            ks.append(_stored(s, "k", table[b], a, a + n, page))
            vs.append(_stored(s, "v", table[b], a, a + n, page))
        return torch.cat(ks), torch.cat(vs)
    hd, hkv, G, cap = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["cap"]
    out = torch.empty(s["n"], case["heads"], hd, dtype=torch.float64, device="cuda")
    for b, (a, n, first) in enumerate(rows):
        k, v = _stored(s, "k", table[b], first, a + n, page), _stored(s, "v", table[b], first, a + n, page)
        for i in range(n):
            m = a + i - first + 1                    # visible positions; the query is the last of them
            q = s["q"][q_start[b] + i].double()
            near, kn = q, k[:m]
            if case["rot"]:
                cos, sin = s["rope"][0].double(), s["rope"][1].double()
                near = _complex_turn(q, cos[m - 1], sin[m - 1])
                if cap:
                    kn = _complex_turn(k[:m], cos[:m, None], sin[:m, None])
            for h in range(case["heads"]):
                z = kn[:, h // G] @ near[h]
                if cap and m - 1 > cap:
                    z[:m - 1 - cap] = k[:m - 1 - cap, h // G] @ _complex_turn(q[h], cos[cap], sin[cap])
                out[q_start[b] + i, h] = torch.softmax(z / math.sqrt(hd), 0) @ v[:m, h // G]
    return out


def _complex_turn(x, cos, sin):
    """Rotation as a product of complex numbers (channel i the real part, channel i + half the imaginary one)."""
    half = cos.shape[-1]
    z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.complex(cos, sin)
    return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)


def _stored(s, name, pages, lo, hi, page):
    """[hi - lo, kv heads, head_dim] float64 of one row's cached positions."""
    first = lo // page
    at = torch.tensor(pages[first:-(-hi // page)], device="cuda")
    x = s[name][at].movedim(1, 2).flatten(0, 1)[lo - first * page:hi - first * page]
    if x.dtype != torch.uint8:
        return x.double()
    sc = s[name + "_scale"].view(torch.uint8)[at].movedim(1, 2).flatten(0, 1)[lo - first * page:hi - first * page].view(torch.float8_e4m3fn).double()
    low, high = (x & 15).double(), (x >> 4).double()

    def value(c):            # E2M1 from its fields: sign, two exponent bits, one mantissa bit
        sign, e, m = torch.floor(c / 8), torch.floor(c % 8 / 2), c % 2
        return (1 - 2 * sign) * torch.where(e > 0, 2.0 ** (e - 1) * (1 + m / 2), m / 2)
    both = torch.stack([value(low), value(high)], -1).flatten(-2)
    return both * sc.repeat_interleave(16, -1)


def _nearest(x, grid):
    """x >= 0 at the nearest value of an ascending grid, a tie at the one of even index."""
    hi = torch.searchsorted(grid, x.contiguous()).clamp(1, len(grid) - 1)
    lo = hi - 1
    below, above = x - grid[lo], grid[hi] - x
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return grid[torch.where(up, hi, lo)]


def _exact_append(s, case, rows, q_start, table):
    k, v = s["new_k"].double(), s["new_v"].double()
    page = case["page"]
    if case["rot"]:
        pos = torch.tensor([a + i for a, n, _ in rows for i in range(n)], device="cuda")
        k = _complex_turn(k, s["rope"][0][pos].double()[:, None], s["rope"][1][pos].double()[:, None])
    if case["fmt"] == "bf16":
        out = {"k": s["k"].double(), "v": s["v"].double()}
        for name, x in (("k", k), ("v", v)):
            for b, (a, n, _) in enumerate(rows):
                pos = torch.arange(a, a + n, device="cuda")
                at = torch.tensor(table[b], device="cuda")[pos // page]
                out[name].transpose(1, 2)[at, pos % page] = x[q_start[b]:q_start[b + 1]]
        return out["k"], out["v"]
    e4m3 = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    e2m1 = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    back = []
    for x in (k, v):
        x = x.float().double().clamp(-2688, 2688)          # the value before the grid is held in 32 bits
        blocks = x.view(*x.shape[:-1], -1, 16)
        sc = _nearest((blocks.abs().amax(-1) / 6), e4m3)[..., None]
        y = torch.where(sc > 0, blocks / torch.where(sc > 0, sc, torch.ones_like(sc)), torch.zeros_like(blocks))
        back.append((torch.sign(y) * _nearest(y.abs().clamp(max=6), e2m1) * sc).view_as(x))
    return tuple(back)


def _exact_verify(s):
    target, draft, drafts, n = s["target"].double(), s["draft"].double(), s["drafts"].tolist(), s["n_drafts"].tolist()
    ua, us = s["u_accept"].double().tolist(), s["u_sample"].double().tolist()
    B, N = len(drafts), len(drafts[0])
    tokens, kept = torch.full((B, N + 1), -1, dtype=torch.long), torch.zeros(B, dtype=torch.long)
    for b in range(B):
        i = 0
        while i < n[b]:
            x = drafts[b][i]
            if not ua[b][i] * float(draft[b, i, x]) < float(target[b, i, x]):
                break
            tokens[b, i] = x
            i += 1
        w = target[b, i]
        if i < n[b]:
            left = (target[b, i] - draft[b, i]).clamp(min=0)
            w = left if float(left.sum()) > 0 else w
        w = w.cpu()
        c = w.cumsum(0)                                    # on the host: one element after the other
        over = torch.nonzero(c > us[b] * c[-1])
        tokens[b, i] = int(over[0]) if len(over) else int(torch.nonzero(w > 0)[-1])
        kept[b] = i
    return tokens.cuda(), kept.cuda()
