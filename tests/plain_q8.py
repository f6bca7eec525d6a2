"""The 8-bit cache in plain torch and 64 bits: what the writes leave in the pages, what attention over them gives.

Also the twin of its three operators (``Q8Twin``), for tests of host logic without a GPU."""

from __future__ import annotations

import math

import torch

TOP = 448.0
LIMIT = TOP * 2.0 ** 50


def e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value (ties to even) of finite float64 values within the range."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def scale_for(top: float) -> float:
    """The least power of two, 2^-50 at least, under which ``top`` fits; NaN beyond the range."""
    if not top <= LIMIT:
        return math.nan
    if top == 0:
        return 2.0 ** -50
    m, e = math.frexp(top)
    return 2.0 ** max(-50, e - 9 + (m > 0.875))


def write_rows(cache: torch.Tensor, scale: torch.Tensor, rows: torch.Tensor, slots: list[int]) -> None:
    """cache [pages, KVH, page, D] (float64: the values in units of the scale), scale [pages, KVH]; rows [T, KVH, D] float64."""
    page = cache.shape[2]
    live = [t for t, s in enumerate(slots) if s >= 0]
    rows, slots = rows[live], [slots[t] for t in live]
    T, t = len(slots), 0
    while t < T:
        pg, u = slots[t] // page, t
        while u < T and slots[u] // page == pg:
            u += 1
        at = [s % page for s in slots[t:u]]
        for h in range(cache.shape[1]):
            x = rows[t:u, h]
            held, need = float(scale[pg, h]), scale_for(float(x.abs().max()) if bool(torch.isfinite(x).all()) else math.inf)
            now = need if 0 in at else (math.nan if held != held or need != need else max(held, need))
            if 0 not in at and now > held:
                others = [r for r in range(page) if r not in at]
                cache[pg, h, others] = e4m3(cache[pg, h, others] * (held / now))
            cache[pg, h, at] = 0.0 if now != now else e4m3(x / now)
            scale[pg, h] = now
        t = u


def rotate(x: torch.Tensor, positions: torch.Tensor, cos, sin, rot: int, dtype) -> torch.Tensor:
    """x [T, heads, D] float64, rotated by halves over the first ``rot`` dims with table rows in ``dtype``."""
    if rot == 0:
        return x
    c = cos[positions.long()].to(dtype).double()[:, None]
    s = sin[positions.long()].to(dtype).double()[:, None]
    a, b = x[..., : rot // 2], x[..., rot // 2: rot]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)


def attend(q, k, v, ks, vs, tables, q_lens, lens, page, scale, window):
    """(outputs [T, H, D], mean of |v| under the weights, largest sum of |q k| * scale of a row's keys [T, H, 1], keys seen), float64.
    ``k``, ``v``: the pages' values in units of their scales, any type."""
    T, H, D = q.shape
    KVH = ks.shape[1]
    per = H // KVH
    outs, size, mags = (torch.zeros((T, H, n), dtype=torch.float64, device=q.device) for n in (D, D, 1))
    t = 0
    for b, (n, length) in enumerate(zip(q_lens, lens)):
        if length == 0:
            t += n
            continue
        ids = tables[b, : -(-length // page)].long()
        rows = lambda x, s: (x[ids].double() * s[ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :length]  # noqa: E731
        K, V = (rows(x, s).repeat_interleave(per, 0) for x, s in ((k, ks), (v, vs)))
        Q = q[t:t + n].double().transpose(0, 1)
        pos, j = torch.arange(length - n, length, device=q.device)[:, None], torch.arange(length, device=q.device)[None]
        seen = j <= pos
        if window:
            seen = seen & (j > pos - window)
        # (a hidden key's weight is zero whatever it holds; a key that is seen and holds a NaN makes its row one)
        bad = torch.isnan(K).any(-1) | torch.isnan(V).any(-1)
        K, V = (torch.where(bad[..., None], torch.zeros_like(x), x) for x in (K, V))
        s = (Q @ K.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        w = torch.where((bad[:, None] & seen[None]).any(-1, keepdim=True), torch.full_like(w, math.nan), w)
        outs[t:t + n] = (w @ V).transpose(0, 1)
        size[t:t + n] = (w @ V.abs()).transpose(0, 1)
        mags[t:t + n] = (Q.abs() @ K.abs().transpose(1, 2) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True).transpose(0, 1)
        t += n
    return outs, size, mags


def maps(requests, updates, tables, page, T, W):
    """(q_start, seq_lens, token_request, positions, slots, block_tables, tables) of a step, as lists and tensors on the CPU."""
    tables = tables.clone().cpu()
    G = tables.shape[0]
    for g, r, i, p in updates.tolist():
        tables[g, r, i] = p
    row, start, n = requests.tolist()
    B = len(row)
    q_start, seq, of, pos = [0], [], [], []
    slots = [[] for _ in range(G)]
    bt = torch.zeros((G, B, W), dtype=torch.int32)
    for b in range(B):
        q_start.append(q_start[-1] + n[b])
        seq.append(start[b] + n[b] if row[b] >= 0 else 0)
        live = -(-seq[b] // page)
        of += [b] * n[b]
        pos += range(start[b], start[b] + n[b])
        for g in range(G):
            slots[g] += [int(tables[g, row[b], p // page]) * page + p % page if row[b] >= 0 else -1
                         for p in range(start[b], start[b] + n[b])]
            if row[b] >= 0:
                m = min(live, W, tables.shape[2])
                bt[g, b, :m] = tables[g, row[b], :m]
    return q_start, seq, of, pos, slots, bt, tables
