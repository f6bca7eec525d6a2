"""The flat token batch of one step, on the device.

Same content as the reference's ``ModelInput`` / ``AttentionMetadata``
(turingserve/runner/attention_metadata.py:10-27, built in turingserve/runner/input_builder.py:105-150):
ids, positions, per-token cache slots, cumulative query starts, context lengths after the step,
padded block tables, rows whose logits are wanted.  Differences: everything is int32; there is one
slot mapping and one block table per cache GROUP; each request also brings its state slot; and the
whole step travels in ONE pinned buffer and ONE host-to-device copy.

Requests with a single token (decodes) are placed first (input_builder.py:41-48), whatever order
the caller gave; ``sample_rows`` keeps the caller's order.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np
import torch

from turingserve_b200 import kernels
from turingserve_b200.cache.manager import CacheManager, RequestCache


@dataclass
class StepEntry:
    """One request's share of a step: its next ``tokens`` and the places among them (``want``)
    whose logits are asked for."""

    cache: RequestCache
    tokens: list[int]
    want: list[int] = field(default_factory=list)
    # When set, the (single) token is not known to the host yet: its id is row ``feedback`` of the
    # previous step's sampler output and is put in place on the device (``tokens`` holds a stand-in).
    feedback: int | None = None


@dataclass
class GroupInputs:
    block_tables: torch.Tensor      # [B, W] int32, padded with the null page 0
    slot_mapping: torch.Tensor      # [T] int32, -1 = do not write
    table_width: int


@dataclass
class StepInputs:
    num_tokens: int
    num_requests: int
    num_decode: int                 # leading requests with exactly one token
    input_ids: torch.Tensor         # [T] int32
    positions: torch.Tensor         # [T] int32
    token_request: torch.Tensor     # [T] int32: index of the request a token belongs to
    q_start: torch.Tensor           # [B+1] int32
    seq_lens: torch.Tensor          # [B] int32: context length after this step
    state_slots: torch.Tensor       # [B] int32
    sample_rows: torch.Tensor       # [S] int32 rows of the flat batch
    groups: list[GroupInputs]
    feedback_rows: torch.Tensor     # [F] int32 rows of the flat batch whose id comes from the device
    feedback_src: torch.Tensor      # [F] int32 rows of the previous sampler output
    # host copies, for launch geometry and for parts written in plain torch
    q_lens: list[int]
    starts: list[int]
    max_q_len: int
    max_seq_len: int
    # The single-token requests together read this many keys or more: their attention should be the
    # kernel built for streaming, not the one built for the shortest chain.  Set from the real
    # lengths; a captured step keeps one graph for each value.
    streaming_decode: bool = False
    # every row of the batch is wanted, in batch order (a captured decode step)
    all_rows_sampled: bool = False
    # the step's token ids on the host, where it knows them all (None: some are fed back on the device)
    host_ids: np.ndarray | None = None
    # Whoever runs the step vouches that its arrays and the cache rows of earlier steps are in place before its first
    # kernel starts (a copy from the host stands between them and the step): attention may read them while the
    # step's kernels before it still run.  A step that is built ahead, behind others that still run, is not settled.
    settled: bool = False


# From about this many keys under the decode rows of a step (requests x longest context), or a third of them in one
# request, the kernel that cuts a request's keys over as many blocks as the chip has takes the decode attention, below
# the one whose blocks of a (request, kv head) are one cluster (12 heads over 2 kv heads of 128, us a launch: 1 x 16,000
# keys 15.7 / 12.4, 1 x 32,000 19.3 / 20.8, 1 x 64,000 24.6 / 38.1, 8 x 32,000 50.5 / 53.0; where clusters are switched off, the
# third costs nothing against the older kernel: 1 x 32,000 18.9 / 18.8, heads of 64 14.5 / 18.4).  The kernels' front adds its
# own rules for many requests and for caches that the streaming kernel does not take.
STREAMING_DECODE_KEYS = 98304


def streaming_decode(num_decode: int, longest_context: int) -> bool:
    return max(num_decode, min(num_decode, 1) * 3) * longest_context >= STREAMING_DECODE_KEYS


def _align(n: int, a: int = 4) -> int:
    return (n + a - 1) // a * a


class StepInputBuilder:
    """Fills a pinned host arena and copies it to a persistent device arena.

    On a GPU the page tables of all live requests stay there (a row per state slot), and what the arena brings of the maps is each
    request's row, its length and its new tokens' number, with the pages that were added or given back since the request's
    last step: positions, slots and block tables are made from that by one kernel (``ops().step_maps``).  Without a GPU,
    or without a cache, for a step of fewer rows than ``device_map_rows``, and for one whose block tables are wider than
    ``max_pages_per_request``, the host lays them out (a captured step is bound to the layout of its rows' number and its tables' fixed width, so
    the rule goes by nothing else)."""

    # ms a decode step through ``LLMEngine.step``, maps from the host / from the GPU (medians of eight runs of 50 steps in turn on one engine, contexts of
    # 2,048, 12 heads over 2, 28 layers, where the GPU bounds the step and most of the host's work is hidden): pages of 16, 2 requests 1.043 /
    # 1.047, 3 1.057 / 1.061, 4 1.080 / 1.081, 6 1.110 / 1.105 (the GPU's less in 8 pairs of 8), 8 1.150 / 1.146 (8 of 8), 12 1.295 / 1.292, 16 to 64
    # within the runs' spread, 128 4.11 / 3.96; pages of 64, 4 1.072 / 1.074 (2 of 8), 6 1.104 / 1.101 (7 of 8), 8 1.148 / 1.143 (8 of 8), 128 3.96 /
    # 3.95.  Of 8 layers, where the host bounds it: 1 0.303 / 0.306, 4 in pages of 64 0.324 / 0.324, 8 0.389 / 0.375 (pages of 16 0.427 / 0.379), 64 in
    # pages of 16 1.81 / 1.22, 128 of 4,000 tokens 5.87 / 3.92.
    device_map_rows = 6

    def __init__(self, cache: CacheManager, max_tokens: int, max_requests: int,
                 max_pages_per_request: int, device) -> None:
        self.cache = cache
        self.max_tokens, self.max_requests = max_tokens, max_requests
        self.max_pages = max_pages_per_request
        self.device = device
        g = len(cache.groups)
        cap = (_align(max_tokens) * (3 + g) + _align(max_requests + 1) + 4 * _align(max_requests)
               + _align(max_tokens) + g * _align(max_requests * max_pages_per_request) + 64)
        pin = device is not None and torch.device(device).type == "cuda"
        self.tables = self._sent = None
        if pin and g:
            rows = cache.max_requests
            self.tables = torch.zeros((g, rows, max_pages_per_request), dtype=torch.int32, device=device)
            # per state slot: the admission it was last seen with, and per group how many pages, and from which on, the GPU knows
            self._sent = [(0, [0] * g, [0] * g) for _ in range(rows)]
            # pages that a step adds or gives back, in all groups (more of them: a copy of their own)
            self.max_updates = 2 * g * (max_tokens // cache.page_size + 2 * max_requests)
            cap += 3 * _align(max_requests) + 4 * self.max_updates
        self.capacity = cap
        self._host = [torch.empty(cap, dtype=torch.int32, pin_memory=pin) for _ in range(2)]
        self._events = [None, None]
        self._turn = 0
        self._dev = torch.empty(cap, dtype=torch.int32, device=device)

    def order(self, entries: list[StepEntry]) -> list[int]:
        """Indices of ``entries`` in batch order: single-token requests first, stable."""
        dec = [i for i, e in enumerate(entries) if len(e.tokens) == 1]
        rest = [i for i, e in enumerate(entries) if len(e.tokens) != 1]
        return dec + rest

    def build(self, entries: list[StepEntry], *, fixed_width: int | None = None,
              pad_requests: int = 0, arena: torch.Tensor | None = None) -> StepInputs:
        """Lay out the step.  ``pad_requests`` puts that many empty decode rows (context 0, slot -1,
        null pages) behind the single-token requests: used to fill a captured batch size.  ``fixed_width`` forces the
        block-table width; ``arena`` is an alternative device buffer (static addresses)."""
        order = self.order(entries)
        n_dec = sum(1 for e in entries if len(e.tokens) == 1)
        # batch order: single-token requests, the padding rows, then the rest
        order = order[:n_dec] + [None] * pad_requests + order[n_dec:]
        rows_e = [None if i is None else entries[i] for i in order]
        ents = [e for e in rows_e if e is not None]
        B = len(rows_e)
        q_lens = [1 if e is None else len(e.tokens) for e in rows_e]
        T = sum(q_lens)
        if B > self.max_requests:
            raise ValueError(f"step has {B} requests, the engine was sized for {self.max_requests}")
        if T > self.max_tokens:
            raise ValueError(f"step has {T} tokens, the engine was sized for {self.max_tokens}")
        if T == 0:
            raise ValueError("empty step")
        starts = [0 if e is None else e.cache.num_tokens for e in rows_e]
        num_decode = n_dec + pad_requests
        ps = self.cache.page_size
        widths = []
        for gi in range(len(self.cache.groups)):
            w = max([len(e.cache.tables[gi]) for e in ents] + [1])
            if fixed_width is not None:
                if w > fixed_width:
                    raise ValueError("block table wider than the fixed width")
                w = fixed_width
            widths.append(w)

        # caller-order sample rows
        row_of = {}
        off = 0
        for i, n in zip(order, q_lens):
            if i is not None:
                row_of[i] = off
            off += n
        sample = []
        for i, e in enumerate(entries):
            for w_ in e.want:
                if not 0 <= w_ < len(e.tokens):
                    raise ValueError(f"request {e.cache.request_id!r}: wanted place {w_} outside its {len(e.tokens)} tokens")
                sample.append(row_of[i] + w_)
        S = len(sample)

        # (a request of more pages than the GPU's tables have columns: from the host, if its arena holds the step)
        if self.tables is not None and B >= self.device_map_rows and max(widths) <= self.max_pages:
            return self._build_on_device(rows_e, q_lens, starts, num_decode, max(widths), sample, arena)
        host_t = self._host[self._turn]
        ev = self._events[self._turn]
        if ev is not None:
            ev.synchronize()
        host = host_t.numpy()
        cursor = 0

        def take(n: int):
            nonlocal cursor
            a = cursor
            cursor += _align(n)
            return a

        # With a caller-owned arena (a captured graph reads it at fixed addresses) the layout may depend
        # only on T, B and the table widths, never on how many rows are wanted or fed back.
        static = arena is not None
        o_ids, o_pos, o_req = take(T), take(T), take(T)
        o_qs, o_sl, o_ss, o_sr = take(B + 1), take(B), take(B), take(T if static else max(S, 1))
        fb = [(b, e.feedback) for b, e in enumerate(rows_e) if e is not None and e.feedback is not None]
        F = len(fb)
        o_fr, o_fs = take(B if static else max(F, 1)), take(B if static else max(F, 1))
        o_slot = [take(T) for _ in widths]
        o_bt = [take(B * w) for w in widths]
        used = cursor
        if used > self.capacity:
            raise ValueError("step does not fit the input arena")

        ids = host[o_ids:o_ids + T]
        pos = host[o_pos:o_pos + T]
        req = host[o_req:o_req + T]
        qs = host[o_qs:o_qs + B + 1]
        sl = host[o_sl:o_sl + B]
        ss = host[o_ss:o_ss + B]
        qs[0] = 0
        t = 0
        for b, e in enumerate(rows_e):
            if e is None:                           # a padding row: no context, nothing written
                ids[t] = 0
                pos[t] = 0
                req[t] = b
                t += 1
                qs[b + 1] = t
                sl[b] = 0
                ss[b] = self.cache.null_slot
                continue
            n = len(e.tokens)
            ids[t:t + n] = e.tokens
            pos[t:t + n] = np.arange(starts[b], starts[b] + n, dtype=np.int32)
            req[t:t + n] = b
            t += n
            qs[b + 1] = t
            sl[b] = starts[b] + n
            ss[b] = e.cache.slot
        host[o_sr:o_sr + S] = sample
        for i, (b, src) in enumerate(fb):
            if q_lens[b] != 1:
                raise ValueError("a token fed back on the device must be a request's only token in the step")
            host[o_fr + i] = qs[b]
            host[o_fs + i] = src
            ids[qs[b]] = 0
        for gi, w in enumerate(widths):
            bt = host[o_bt[gi]:o_bt[gi] + B * w].reshape(B, w)
            bt[:] = 0
            sm = host[o_slot[gi]:o_slot[gi] + T]
            t = 0
            for b, e in enumerate(rows_e):
                if e is None:
                    sm[t] = -1
                    t += 1
                    continue
                table = e.cache.tables[gi]
                bt[b, :len(table)] = table
                n = len(e.tokens)
                p = pos[t:t + n]
                tab = np.asarray(table, dtype=np.int32)
                sm[t:t + n] = tab[p // ps] * ps + p % ps
                t += n

        dev = self._dev if arena is None else arena
        dev[:used].copy_(host_t[:used], non_blocking=True)
        if torch.device(self.device).type == "cuda":
            e_ = torch.cuda.Event()
            e_.record()
            self._events[self._turn] = e_
        self._turn ^= 1

        def d(o, n):
            return dev[o:o + n]

        groups = [GroupInputs(d(o_bt[gi], B * w).view(B, w), d(o_slot[gi], T), w)
                  for gi, w in enumerate(widths)]
        return StepInputs(
            num_tokens=T, num_requests=B, num_decode=num_decode, input_ids=d(o_ids, T),
            positions=d(o_pos, T), token_request=d(o_req, T), q_start=d(o_qs, B + 1),
            seq_lens=d(o_sl, B), state_slots=d(o_ss, B), sample_rows=d(o_sr, S), groups=groups,
            feedback_rows=d(o_fr, F), feedback_src=d(o_fs, F),
            q_lens=q_lens, starts=starts, max_q_len=max(q_lens), max_seq_len=int(sl.max()) if B else 0,
            streaming_decode=streaming_decode(num_decode, int(sl[:num_decode].max()) if num_decode else 0),
            host_ids=ids.copy() if F == 0 else None)

    def _page_updates(self, ents) -> tuple[list[int], list]:
        """([group, row, index, page, ...] that the GPU's tables lack for these requests, what to remember once they are sent)."""
        ups, seen = [], []
        for e in ents:
            rc = e.cache
            admission, held, live = self._sent[rc.slot]
            if admission != rc.admission:
                held = live = [0] * len(rc.tables)
            now_held = [len(t) for t in rc.tables]
            if admission == rc.admission and now_held == held and rc.first_live_page == live:
                continue
            for gi, table in enumerate(rc.tables):
                for i in range(live[gi], min(rc.first_live_page[gi], held[gi])):
                    if table[i] == 0:
                        ups += (gi, rc.slot, i, 0)
                for i in range(held[gi], len(table)):
                    ups += (gi, rc.slot, i, table[i])
            seen.append((rc.slot, (rc.admission, now_held, list(rc.first_live_page))))
        return ups, seen

    def _build_on_device(self, rows_e: list, q_lens: list[int], starts: list[int], num_decode: int, width: int, sample: list[int],
                         arena: torch.Tensor | None) -> StepInputs:
        """The same step with its maps made on the GPU out of lengths."""
        B, T, S, G = len(rows_e), sum(q_lens), len(sample), len(self.cache.groups)
        static = arena is not None                  # (its layout may depend on T, B and the width only)
        dev = self._dev if arena is None else arena
        fb = [(b, e.feedback) for b, e in enumerate(rows_e) if e is not None and e.feedback is not None]
        if any(q_lens[b] != 1 for b, _ in fb):
            raise ValueError("a token fed back on the device must be a request's only token in the step")
        F = len(fb)
        ups, seen = self._page_updates([e for e in rows_e if e is not None])
        U = len(ups) // 4
        cursor = 0

        def take(n: int):
            nonlocal cursor
            a = cursor
            cursor += _align(n)
            return a

        # the second copy's part, what the kernel writes, and the first copy's part, whose updates are of any number
        o_ids, o_ss, o_sr = take(T), take(B), take(T if static else max(S, 1))
        o_fr, o_fs = take(B if static else max(F, 1)), take(B if static else max(F, 1))
        second = cursor
        o_pos, o_req, o_qs, o_sl = take(T), take(T), take(B + 1), take(B)
        o_slot = cursor
        cursor += G * _align(T)
        o_bt = cursor
        cursor += G * _align(B * width)
        o_rq = take(3 * B)
        o_up = cursor
        few = U <= self.max_updates
        used = cursor + (4 * U if few else 0)
        if used > self.capacity:
            raise ValueError("step does not fit the input arena")

        host_t, ev = self._host[self._turn], self._events[self._turn]
        if ev is not None:
            ev.synchronize()
        host = host_t.numpy()
        host[o_rq:o_rq + 3 * B] = [-1 if e is None else e.cache.slot for e in rows_e] + starts + q_lens
        if few:
            host[o_up:o_up + 4 * U] = ups
        ids = host[o_ids:o_ids + T]
        ids[:num_decode] = [0 if e is None else e.tokens[0] for e in rows_e[:num_decode]]
        t, firsts = num_decode, list(range(num_decode))
        for b in range(num_decode, B):
            ids[t:t + q_lens[b]] = rows_e[b].tokens
            firsts.append(t)
            t += q_lens[b]
        host[o_ss:o_ss + B] = [self.cache.null_slot if e is None else e.cache.slot for e in rows_e]
        host[o_sr:o_sr + S] = sample
        for i, (b, src) in enumerate(fb):
            host[o_fr + i] = firsts[b]
            host[o_fs + i] = src
            ids[firsts[b]] = 0

        def d(o, *shape):
            n = 1
            for x in shape:
                n *= x
            return dev[o:o + n].view(shape)

        dev[o_rq:used].copy_(host_t[o_rq:used], non_blocking=True)
        updates = d(o_up, U, 4) if few else torch.tensor(ups, dtype=torch.int32).view(U, 4).to(dev.device)
        q_start, seq_lens, request, positions = d(o_qs, B + 1), d(o_sl, B), d(o_req, T), d(o_pos, T)
        slots = dev[o_slot:o_slot + G * _align(T)].view(G, -1)[:, :T]
        tables = dev[o_bt:o_bt + G * _align(B * width)].view(G, -1)[:, :B * width].unflatten(1, (B, width))
        kernels.ops().step_maps(d(o_rq, 3, B), updates, self.tables, self.cache.page_size, q_start, seq_lens, request, positions, slots, tables)
        for slot, what in seen:
            self._sent[slot] = what
        # This copy stands between the maps and the step: attention reads them before it waits for the kernels before it.
        dev[:second].copy_(host_t[:second], non_blocking=True)
        e_ = torch.cuda.Event()
        e_.record()
        self._events[self._turn] = e_
        self._turn ^= 1
        ends = [0 if e is None else s + n for e, s, n in zip(rows_e, starts, q_lens)]
        return StepInputs(
            num_tokens=T, num_requests=B, num_decode=num_decode, input_ids=d(o_ids, T), positions=positions, token_request=request,
            q_start=q_start, seq_lens=seq_lens, state_slots=d(o_ss, B), sample_rows=d(o_sr, S),
            groups=[GroupInputs(tables[gi], slots[gi], width) for gi in range(G)],
            feedback_rows=d(o_fr, F), feedback_src=d(o_fs, F), q_lens=q_lens, starts=starts, max_q_len=max(q_lens),
            max_seq_len=max(ends), streaming_decode=streaming_decode(num_decode, max(ends[:num_decode], default=0)),
            host_ids=ids.copy() if F == 0 else None)
