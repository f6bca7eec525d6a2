"""The 8-bit key/value cache and the step's page maps: how fast they are, and what they have to give.

Three operators of a serving step, as a program that keeps its cache in 8 bits has them done:

``write``  rotary positions on queries and keys, and keys and values into pages of e4m3 values with one power-of-two scale
           for each (page, kv head): ``ops().rope_kv_write_q8``
``attend`` attention of single tokens and of prompt portions over such pages: ``ops().attention_q8``
``maps``   query starts, positions, cache slots and block tables of a step, on the GPU, out of each request's length and a
           page table that stays there: ``ops().step_maps``

With ``own`` false, ``run`` works them in plain torch, 32 bits throughout.  ``exact`` works them in 64 bits, request by request.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
BF16, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
TOP = 448.0                               # the largest e4m3 value
THETA = 1000000.0

# query heads, kv heads, head size of the benchmark's model shapes
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "14b": (40, 8, 128)}


def listed() -> list[dict]:
    return [
        # one user alone: a decode step's write is all latency
        dict(name="write_single", op="write", size="1.5b", page=64, singles=1, shortest=517, longest=517, portions=0, tokens=0, behind=0),
        # 64 users decode a token each, pages of 16
        dict(name="write_64_singles", op="write", size="7b", page=16, singles=64, shortest=100, longest=4000, portions=0, tokens=0, behind=0),
        # four prompts of odd lengths arrive in portions behind tokens that are there already, beside 13 users who decode
        dict(name="write_portions", op="write", size="7b", page=64, singles=13, shortest=700, longest=2100, portions=4, tokens=1999,
             behind=333),
        # one user with a short chat
        dict(name="attend_single_short", op="attend", size="1.5b", page=64, singles=1, shortest=57, longest=57, portions=0, tokens=0,
             behind=0, window=0),
        # the benchmark's own decode step: eight users at 2,048 tokens
        dict(name="attend_8_singles", op="attend", size="1.5b", page=64, singles=8, shortest=2048, longest=2048, portions=0, tokens=0,
             behind=0, window=0),
        # many users with long contexts of many lengths, pages of 16: what the cache's bytes bound
        dict(name="attend_64_singles", op="attend", size="7b", page=16, singles=64, shortest=4100, longest=8192, portions=0, tokens=0,
             behind=0, window=0),
        # one very long document
        dict(name="attend_single_long", op="attend", size="14b", page=64, singles=1, shortest=100001, longest=100001, portions=0,
             tokens=0, behind=0, window=0),
        # a scheduler's mixed step under a sliding window, heads of 64: 16 users beside a portion of a long prompt
        dict(name="attend_mixed_window", op="attend", size="0.5b", page=16, singles=16, shortest=300, longest=3001, portions=1,
             tokens=495, behind=1500, window=1024),
        # a prompt of 2,048 tokens
        dict(name="attend_prompt", op="attend", size="1.5b", page=64, singles=0, shortest=0, longest=0, portions=1, tokens=2048,
             behind=0, window=0),
        # a long prompt's last portion, at the 7B shape (the largest)
        dict(name="attend_long_prompt", op="attend", size="7b", page=64, singles=0, shortest=0, longest=0, portions=1, tokens=4096,
             behind=4001, window=0),
        # the maps of eight users who decode
        dict(name="maps_8_singles", op="maps", page=64, width=64, groups=1, singles=8, shortest=2048, longest=2048, portions=0, tokens=0,
             behind=0),
        # the maps of a full engine: 128 users with long contexts, pages of 16, beside a prompt portion, two cache groups
        dict(name="maps_full", op="maps", page=16, width=2048, groups=2, singles=128, shortest=500, longest=32000, portions=1, tokens=1920,
             behind=4000),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    op = rng.choice(["write", "attend", "attend", "attend", "maps"])
    c = dict(op=op, page=rng.choice([16, 32, 64]), singles=0, shortest=0, longest=0, portions=0, tokens=0, behind=0)
    if op == "maps":
        c.update(width=2048, groups=rng.choice([1, 2]), singles=_log_int(rng, 1, 128), longest=_log_int(rng, 2, 32000))
        c["shortest"] = rng.randint(1, c["longest"])
        if rng.random() < 0.5:
            c.update(portions=1, tokens=_log_int(rng, 2, 2048), behind=rng.randint(0, 4000))
        return c
    c["size"] = rng.choice(list(HEADS))
    kind = rng.choice(["singles", "portions", "mixed"])
    if op == "write":
        if kind != "portions":
            c.update(singles=_log_int(rng, 1, 128), longest=_log_int(rng, 1, 8192))
            c["shortest"] = rng.randint(1, c["longest"])
        if kind != "singles":
            c.update(portions=rng.randint(1, 4), tokens=_log_int(rng, 2, 1999), behind=rng.choice([0, rng.randint(1, 2000)]))
        return c
    H = HEADS[c["size"]][0]
    c["window"] = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
    if kind != "portions":
        c["longest"] = _log_int(rng, 1, 100001)
        # (no more keys than 64 requests of 6,000)
        c["singles"] = _log_int(rng, 1, max(1, min(128, 380000 // c["longest"])))
        c["shortest"] = rng.randint(max(1, c["longest"] // 4), c["longest"])
    if kind != "singles":
        c.update(portions=rng.choice([1, 1, 2, 3]), behind=rng.choice([0, rng.randint(1, 4000)]))
        # (no more scores than the largest listed case)
        c["tokens"] = max(2, _log_int(rng, 2, 28 * 4096 // H) // c["portions"])
        while c["portions"] * c["tokens"] * (c["tokens"] + c["behind"]) * H > 28 * 4096 * 8097:
            c["tokens"] = max(2, c["tokens"] // 2)
    return c


# -- what a step looks like ------------------------------------------------------------------------------------------------

def _lens(c) -> tuple[list[int], list[int]]:
    """(tokens each request brings, its context after the step): the single tokens, then the portions."""
    n = c["singles"]
    ctx = [c["shortest"] + (c["longest"] - c["shortest"]) * (i * 7 % n) // max(1, n - 1) if n > 1 else c["longest"] for i in range(n)]
    q = [1] * n
    for i in range(c["portions"]):
        q.append(max(2, c["tokens"] - 37 * i))
        ctx.append(c["behind"] + q[-1])
    return q, [min(x, c["longest"]) if i < n else x for i, x in enumerate(ctx)]


def _seen(c, q: list[int], ctx: list[int]) -> int:
    """(query, key) pairs under the mask, of one head."""
    w, total = c.get("window", 0), 0
    for n, s in zip(q, ctx):
        if not w:
            total += n * s - n * (n - 1) // 2
        else:
            lo, hi = s - n + 1, s                         # keys that the first and the last query would see without a window
            a = min(max(w, lo - 1), hi)
            total += (a * (a + 1) - (lo - 1) * lo) // 2 + (hi - a) * w
    return total


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _tables(c, ctx, g):
    """(block tables [B, width], pages of the pool): every request's pages are scattered over the pool; page 0 is nobody's."""
    page = c["page"]
    need = [-(-s // page) for s in ctx]
    width, total = max(need), sum(need) + 1
    ids = (torch.randperm(total - 1, generator=g, device=DEV) + 1).to(I32)
    tables = torch.zeros((len(ctx), width), dtype=I32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at:at + n]
        at += n
    return tables, total


def _power(x):
    """2^x of whole numbers, exactly."""
    return torch.ldexp(torch.ones_like(x, dtype=torch.float32), x)


def _pages(total, KVH, page, D, g):
    """Pages of keys or values in 8 bits: scales of several powers of two, values up to the top of the range."""
    exps = torch.randint(-9, -5, (total, KVH), generator=g, device=DEV)
    x = torch.randn((total, KVH, page, D), generator=g, device=DEV) * 110.0
    return x.clamp_(-TOP, TOP).to(F8), _power(exps)


def prepare(case: dict, seed: int):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    s = SimpleNamespace(case=c, op=c["op"])
    q, ctx = _lens(c)
    B, T = len(q), sum(q)
    s.q_lens, s.ctx, s.B, s.T, s.page = q, ctx, B, T, c["page"]
    if c["op"] == "maps":
        G, W, P = c["groups"], c["width"], c["page"]
        rows = 1 + B + 7
        s.tables = torch.randint(1, 1 << 20, (G, rows, W), generator=g, device=DEV, dtype=I32)
        row = torch.randperm(rows - 1, generator=g, device=DEV)[:B].to(I32)
        s.requests = torch.stack([row, _i32([b - a for a, b in zip(q, ctx)]), _i32(q)])
        # the pages that this step's new tokens begin, in each group
        own_, idx = [], []
        for b in range(B):
            for i in range(-(-(ctx[b] - q[b]) // P), -(-ctx[b] // P)):
                own_.append(b)
                idx.append(i)
        n = len(own_)
        pages = torch.randint(1, 1 << 20, (G * n,), generator=g, device=DEV, dtype=I32)
        of_row = row[torch.tensor(own_, dtype=torch.long, device=DEV)]
        s.updates = torch.stack([_i32([k for k in range(G) for _ in range(n)]), of_row.repeat(G), _i32(idx).repeat(G), pages], 1).contiguous()
        new = lambda *shape: torch.empty(shape, dtype=I32, device=DEV)  # noqa: E731
        s.q_start, s.seq_lens, s.token_request, s.positions = new(B + 1), new(B), new(T), new(T)
        s.slots, s.block_tables = new(G, T), new(G, B, W)
        return s
    s.H, s.KVH, s.D = H, KVH, D = HEADS[c["size"]]
    s.q_start = _i32([sum(q[:b]) for b in range(B + 1)])
    s.seq_lens = _i32(ctx)
    s.singles = c["singles"]
    if c["op"] == "write":
        s.qkv = torch.randn((T, (H + 2 * KVH) * D), generator=g, device=DEV)
        s.qkv *= 2.0 ** (torch.randn((T, 1), generator=g, device=DEV))                  # tokens of several magnitudes
        s.qkv = s.qkv.to(BF16)
        s.q = torch.empty((T, H * D), dtype=BF16, device=DEV)
        at = torch.arange(max(ctx), device=DEV, dtype=torch.float64)[:, None]
        angle = at * THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        s.positions = torch.cat([torch.arange(m - n, m, device=DEV, dtype=I32) for n, m in zip(q, ctx)])
        # only the pages that new tokens go to are kept: the others are not touched
        first = [(m - n) // s.page for n, m in zip(q, ctx)]
        local = [m - f * s.page for m, f in zip(ctx, first)]
        tables, total = _tables(c, local, g)
        slot = [tables[b][(p := torch.arange(local[b] - q[b], local[b], device=DEV)) // s.page] * s.page + p % s.page for b in range(B)]
        s.slots = torch.cat(slot).to(I32)
        s.k, s.ks = _pages(total, KVH, s.page, D, g)
        s.v, s.vs = _pages(total, KVH, s.page, D, g)
        return s
    s.q = torch.randn((T, H * D), generator=g, device=DEV).to(BF16)
    s.tables, total = _tables(c, ctx, g)
    s.k, s.ks = _pages(total, KVH, s.page, D, g)
    s.v, s.vs = _pages(total, KVH, s.page, D, g)
    s.scale, s.window = D ** -0.5, c["window"]
    s.out = torch.empty((T, H * D), dtype=BF16, device=DEV)
    s.step = SimpleNamespace(num_requests=B, num_decode=c["singles"], q_start=s.q_start, seq_lens=s.seq_lens, max_q_len=max(q),
                             max_seq_len=max(ctx), settled=True)
    return s


# -- one pass --------------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"write": _plain_write, "attend": _plain_attend, "maps": _plain_maps}[s.op](s)


def _own(s):
    from turingserve_b200 import kernels

    ops = kernels.ops()
    if s.op == "write":
        ops.rope_kv_write_q8(s.q, s.qkv, s.positions, s.cos, s.sin, s.H, s.KVH, s.D, s.D, s.k, s.v, s.ks, s.vs, s.slots, s.page)
        return {"q": s.q, "k": s.k, "v": s.v, "k_scale": s.ks, "v_scale": s.vs}
    if s.op == "attend":
        ops.attention_q8(s.out, s.q.view(s.T, s.H, s.D), s.k, s.v, s.ks, s.vs, s.tables, s.step, s.KVH, s.page, s.scale, s.window)
        return {"out": s.out}
    ops.step_maps(s.requests, s.updates, s.tables, s.page, s.q_start, s.seq_lens, s.token_request, s.positions, s.slots, s.block_tables)
    return _maps_of(s)


def _maps_of(s):
    return {"q_start": s.q_start, "seq_lens": s.seq_lens, "token_request": s.token_request, "positions": s.positions, "slots": s.slots,
            "block_tables": s.block_tables, "tables": s.tables}


def _plain_block(cache, scale, rows, page_of, at, begins):
    """The rows [T, KVH, D] into their places, in 8 bits.  A page's scale is the least power of two under which its largest value
    fits; rows that were there keep the larger of the two scales, unless the page is begun anew by its first row."""
    pages, KVH = scale.shape
    top = torch.zeros_like(scale).index_reduce_(0, page_of, rows.abs().amax(-1), "amax")
    m, e = torch.frexp(top)
    need = torch.where(top > 0, _power((e - 9 + (m > 0.875).int()).clamp(min=-50)), torch.ones_like(top) * 2.0 ** -50)
    touched = torch.zeros(pages, dtype=torch.bool, device=cache.device).index_fill_(0, page_of, True)
    anew = torch.zeros(pages, dtype=torch.int32, device=cache.device).index_reduce_(0, page_of, begins.int(), "amax").bool()
    held = torch.where(anew[:, None], torch.zeros_like(scale), scale)
    now = torch.where(touched[:, None], torch.maximum(held, need), scale)
    ratio = torch.where(anew[:, None], torch.ones_like(scale), scale / now)
    cache.copy_((cache.float() * ratio[:, :, None, None]).to(F8))
    scale.copy_(now)
    cache[page_of, :, at] = (rows / now[page_of][..., None]).clamp(-TOP, TOP).to(F8)


def _plain_write(s):
    T, H, KVH, D, page = s.T, s.H, s.KVH, s.D, s.page
    x = s.qkv.float().view(T, H + 2 * KVH, D)
    pos = s.positions.long()
    # the tables' rows are taken in the type of the values that they turn
    cos, sin = s.cos[pos].to(BF16).float()[:, None], s.sin[pos].to(BF16).float()[:, None]
    a, b = x[:, :H + KVH, :D // 2], x[:, :H + KVH, D // 2:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    s.q.copy_(turned[:, :H].reshape(T, H * D))
    slots = s.slots.long()
    page_of, at = slots // page, slots % page
    _plain_block(s.k, s.ks, turned[:, H:], page_of, at, at == 0)
    _plain_block(s.v, s.vs, x[:, H + KVH:], page_of, at, at == 0)
    return {"q": s.q, "k": s.k, "v": s.v, "k_scale": s.ks, "v_scale": s.vs}


def _plain_rows(s, q, q_start, seq_lens, tables, max_q):
    """Attention of requests [B] with up to ``max_q`` tokens each, padded: outputs [B, max_q, H, D] in 32 bits."""
    B, W = tables.shape
    H, KVH, D, page = s.H, s.KVH, s.D, s.page
    K = W * page
    ids = tables.long()
    k = (s.k[ids].float() * s.ks[ids][..., None, None]).transpose(2, 3).reshape(B, K, KVH, D)
    v = (s.v[ids].float() * s.vs[ids][..., None, None]).transpose(2, 3).reshape(B, K, KVH, D)
    n = (q_start[1:] - q_start[:-1]).long()
    i = torch.arange(max_q, device=q.device)
    row = (q_start[:-1].long()[:, None] + i).clamp(max=q.shape[0] - 1)
    qs = q.float().view(-1, KVH, H // KVH, D)[row]                                      # [B, max_q, KVH, G, D]
    pos = (seq_lens.long() - n)[:, None] + i                                            # [B, max_q]
    j = torch.arange(K, device=q.device)
    seen = j <= pos[..., None]
    if s.window:
        seen = seen & (j > pos[..., None] - s.window)
    scores = torch.matmul(qs.permute(0, 2, 3, 1, 4) * s.scale, k.permute(0, 2, 3, 1)[:, :, None])           # [B, KVH, G, max_q, K]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    out = torch.matmul(p, v.permute(0, 2, 1, 3)[:, :, None]) / p.sum(-1, keepdim=True)
    return out.permute(0, 3, 1, 2, 4).reshape(B, max_q, H * D), row, i < n[:, None]


def _plain_attend(s):
    nd = s.singles
    if nd:
        out, _, _ = _plain_rows(s, s.q, s.q_start[:nd + 1], s.seq_lens[:nd], s.tables[:nd], 1)
        s.out[:nd] = out[:, 0]
    if nd < s.B:
        out, row, real = _plain_rows(s, s.q, s.q_start[nd:], s.seq_lens[nd:], s.tables[nd:], s.step.max_q_len)
        s.out[row[real]] = out[real].to(BF16)
    return {"out": s.out}


def _plain_maps(s):
    g, r, i, p = s.updates.long().unbind(1)
    s.tables[g, r, i] = p.to(I32)
    row, start, n = s.requests.long().unbind(0)
    ends = n.cumsum(0)
    s.q_start[0] = 0
    s.q_start[1:] = ends
    s.seq_lens.copy_(start + n)
    t = torch.arange(s.T, device=row.device)
    of = torch.repeat_interleave(torch.arange(s.B, device=row.device), n, output_size=s.T)
    s.token_request.copy_(of)
    pos = start[of] + t - (ends - n)[of]
    s.positions.copy_(pos)
    live = torch.arange(s.tables.shape[2], device=row.device) < ((start + n + s.page - 1) // s.page)[:, None]
    s.block_tables.copy_(torch.where(live, s.tables[:, row], 0))
    s.slots.copy_(s.block_tables[:, of, pos // s.page] * s.page + pos % s.page)
    return _maps_of(s)


# -- what a pass cannot do without -------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    c = case
    q, ctx = _lens(c)
    T, B = sum(q), len(q)
    if c["op"] == "maps":
        G, W = c["groups"], c["width"]
        live = sum(-(-x // c["page"]) for x in ctx)
        return {"bytes": 4.0 * (3 * B + 2 * B + 1 + 2 * T + G * (T + live + B * W)), "flops": 0.0}
    H, KVH, D = HEADS[c["size"]]
    if c["op"] == "write":
        new = T * KVH * D
        blocks = sum(-(-m // c["page"]) - (m - n) // c["page"] for n, m in zip(q, ctx))
        return {"bytes": 2.0 * T * (H + 2 * KVH) * D + 2.0 * T * H * D + 2.0 * new + 16.0 * blocks * KVH + 4.0 * T * (D + 2),
                "flops": 6.0 * T * (H + KVH) * D / 2}
    w = c["window"]
    keys = sum(min(s, n + w - 1) if w else s for n, s in zip(q, ctx))
    return {"bytes": 4.0 * T * H * D + 2.0 * keys * KVH * D + 8.0 * KVH * (keys // c["page"]) + 4.0 * (keys // c["page"] + 2 * B),
            "flops": 4.0 * _seen(c, q, ctx) * H * D}


# -- in 64 bits --------------------------------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    if case["op"] == "maps":
        return None                       # whole numbers: they are equal or they are wrong
    s = prepare(case, seed)
    return _exact_write(s) if s.op == "write" else _exact_attend(s)


def _e4m3(x):
    """The nearest value with three bits behind the leading one, the least exponent -6, ties to even: in 64 bits."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_write(s):
    T, H, KVH, D, page = s.T, s.H, s.KVH, s.D, s.page
    x = s.qkv.double().reshape(T, -1, D)
    half = D // 2
    c = s.cos.to(BF16).double().index_select(0, s.positions.long()).unsqueeze(1).expand(T, H + KVH, half)
    n = s.sin.to(BF16).double().index_select(0, s.positions.long()).unsqueeze(1).expand(T, H + KVH, half)
    z = torch.complex(x[:, :H + KVH, :half], x[:, :H + KVH, half:]) * torch.complex(c, n)
    turned = torch.cat([z.real, z.imag], dim=2)
    got = {"q": turned[:, :H].reshape(T, H * D)}
    slots = s.slots.tolist()
    for name, scales, cache, rows in (("k", s.ks, s.k, turned[:, H:]), ("v", s.vs, s.v, x[:, H + KVH:])):
        sc, vals = scales.double(), cache.double()
        t = 0
        while t < T:
            u, pg = t, slots[t] // page
            while u < T and slots[u] // page == pg:
                u += 1
            lo = slots[t] % page
            top = rows[t:u].abs().amax(dim=(0, 2))
            need = torch.tensor([2.0 ** max(-50, math.ceil(math.log2(a / TOP))) if a > 0 else 2.0 ** -50 for a in top.tolist()],
                                dtype=torch.float64, device=top.device)
            new = need if lo == 0 else torch.maximum(need, sc[pg])
            if lo:
                vals[pg] = _e4m3(vals[pg] * (sc[pg] / new)[:, None, None])
            vals[pg, :, lo:lo + u - t] = _e4m3(rows[t:u] / new[:, None]).transpose(0, 1)
            sc[pg] = new
            t = u
        got[name], got[name + "_scale"] = vals, sc
    return got


def _exact_attend(s):
    H, KVH, D, page = s.H, s.KVH, s.D, s.page
    out = torch.empty((s.T, H, D), dtype=torch.float64, device=DEV)
    t = 0
    for b, (n, length) in enumerate(zip(s.q_lens, s.ctx)):
        ids = s.tables[b, :-(-length // page)].long()
        for h in range(KVH):
            k = (s.k[ids, h].double() * s.ks[ids, h].double()[:, None, None]).reshape(-1, D)[:length]
            v = (s.v[ids, h].double() * s.vs[ids, h].double()[:, None, None]).reshape(-1, D)[:length]
            pos = torch.arange(length - n, length, device=DEV)
            j = torch.arange(length, device=DEV)
            hidden = j[None] > pos[:, None]
            if s.window:
                hidden |= j[None] <= pos[:, None] - s.window
            for g in range(h * (H // KVH), (h + 1) * (H // KVH)):
                w = torch.einsum("td,jd->tj", s.q[t:t + n, g * D:(g + 1) * D].double(), k) * s.scale
                w = torch.softmax(w.masked_fill(hidden, -math.inf), dim=-1)
                out[t:t + n, g] = torch.einsum("tj,jd->td", w, v)
        t += n
    return {"out": out.reshape(s.T, H * D)}
