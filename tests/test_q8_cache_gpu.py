"""The 8-bit cache on the GPU against 64 bits: the write (scales, values, pages that grow), attention over it, and both in a run.

Bounds.  A value on its way to 8 bits is off by half a step, 2^-4 of it, or by half the least step, 2^-10 of its page's scale; a rotated
key by 2^-22 of the products' sizes before that (three roundings of 2^-24 each on sums of two products).  An attention output is rounded
to its type (bfloat16: 2^-8 of it).  Before that, with M the mean of |v| under the weights and A the largest scale * sum |q k| of the row's
keys: scores summed in 32 bits in any order are off by at most (D + 4) 2^-24 A, which moves each weight by twice that at most (numerator
and denominator); the kernels that take the queries as half floats add 2^-25 of the largest |q| an element, below 2^-24 (D + 4) A wherever A is
not tiny; a base-2 exponential and its argument's rounding (scores up to 64 in these tests: 2^-24 * 64) add 2^-17; weights as half floats
2^-11 each and 2^-25 of the largest (weight * scale) for the smallest, over n keys; sums of n terms in 32 bits 2^-24 n at most."""

from types import SimpleNamespace

import math

import pytest
import torch

from tests import plain_q8 as plain
from turingserve_b200.kernels import KernelError

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from turingserve_b200 import kernels
    kernels.use(None)
    return kernels.ops()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def pages_of(total, KVH, page, D, g, spread=3):
    exps = torch.randint(-8, -8 + spread, (total, KVH), generator=g, device=DEV)
    x = (torch.randn((total, KVH, page, D), generator=g, device=DEV) * 100).clamp(-448, 448).to(F8)
    return x, torch.ldexp(torch.ones((total, KVH), device=DEV), exps)


def rope_tables(n, rot):
    f = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, max(rot, 2), 2, device=DEV).double() / max(rot, 2))
    return f.cos().float(), f.sin().float()


def tables_for(lens, page, g, spare=2):
    need = [max(1, -(-n // page)) for n in lens]
    total = sum(need) + 1 + spare
    ids = (torch.randperm(total - 1, generator=g, device=DEV) + 1)[: sum(need)].split(need)
    t = torch.zeros((len(lens), max(need) + 1), dtype=torch.int32, device=DEV)
    for b, x in enumerate(ids):
        t[b, : need[b]] = x
    return t, total


# ---------------------------------------------------------------------------------------------------------------- write

WRITES = [
    # (q_lens, tokens before, H, KVH, D, rot, page, type)
    ([1], [516], 12, 2, 128, 128, 64, BF16),
    ([1], [64], 14, 2, 64, 64, 64, BF16),                    # the page's first row
    ([1] * 33, [7 * i for i in range(33)], 28, 4, 128, 128, 16, BF16),
    ([300], [0], 12, 2, 128, 128, 64, BF16),
    ([301, 65], [37, 200], 14, 2, 64, 64, 16, BF16),
    ([1, 1, 1, 130, 2], [99, 64, 0, 63, 15], 28, 4, 128, 128, 16, BF16),
    ([257], [11], 3, 1, 128, 128, 256, BF16),                # a page of more rows than a block takes in one turn
    ([40, 9], [5, 0], 6, 3, 80, 80, 7, BF16),                # sizes that no fast variant takes
    ([40, 9], [5, 0], 4, 2, 128, 64, 16, BF16),              # rotated over half of the head
    ([19], [3], 4, 4, 64, 0, 16, BF16),                      # no rotation: the values are exact
    ([1, 21], [30, 3], 6, 2, 128, 128, 16, torch.float32),
    ([700], [100], 40, 8, 128, 128, 64, BF16),
    ([1, 1, 1100, 190], [64, 300, 37, 1], 6, 2, 64, 64, 48, BF16),       # wider spans
    ([1300], [7], 7, 1, 128, 128, 256, BF16),
    ([1, 2500, 1650], [5, 61, 0], 4, 1, 128, 128, 16, BF16),             # and smaller blocks
]


class Write:
    def __init__(self, q_lens, before, H, KVH, D, rot, page, dtype, seed=0, magnitude=2.0):
        g = gen(seed + sum(q_lens) + D + page)
        self.H, self.KVH, self.D, self.rot, self.page, self.dtype = H, KVH, D, rot, page, dtype
        self.lens = [a + b for a, b in zip(q_lens, before)]
        T = sum(q_lens)
        self.x = torch.randn((T, (H + 2 * KVH) * D), generator=g, device=DEV)
        self.x = (self.x * magnitude ** torch.randn((T, 1), generator=g, device=DEV)).to(dtype)
        self.cos, self.sin = rope_tables(max(self.lens), rot)
        self.positions = torch.cat([torch.arange(b, b + n, device=DEV) for n, b in zip(q_lens, before)]).int()
        self.tables, total = tables_for(self.lens, page, g)
        self.slots = torch.cat([(self.tables[b][(p := torch.arange(s - n, s, device=DEV)) // page] * page + p % page)
                                for b, (n, s) in enumerate(zip(q_lens, self.lens))]).int()
        self.k, self.ks = pages_of(total, KVH, page, D, g)
        self.v, self.vs = pages_of(total, KVH, page, D, g)
        self.q = torch.zeros((T, H * D), dtype=dtype, device=DEV)

    def run(self, ops):
        before = self.x.clone()
        self.k0, self.v0, self.ks0, self.vs0 = (t.clone() for t in (self.k, self.v, self.ks, self.vs))
        ops.rope_kv_write_q8(self.q, self.x, self.positions, self.cos, self.sin, self.H, self.KVH, self.D, self.rot, self.k, self.v,
                             self.ks, self.vs, self.slots, self.page)
        assert torch.equal(before.view(torch.uint8), self.x.view(torch.uint8))

    def check(self):
        T, H, KVH, D = self.x.shape[0], self.H, self.KVH, self.D
        x = self.x.double().view(T, -1, D)
        turned = plain.rotate(x[:, : H + KVH], self.positions, self.cos, self.sin, self.rot, self.dtype)
        # the products' sizes: |a c| + |b s| and |b c| + |a s| (with the sine's sign turned the first half of a rotation is that sum,
        # the second a difference; the second half's sum is the first half's of the halves swapped)
        h = self.rot // 2
        swapped = torch.cat([x[..., h:2 * h], x[..., :h], x[..., 2 * h:]], -1)
        sums = [plain.rotate(y[:, : H + KVH].abs(), self.positions, self.cos.abs(), -self.sin.abs(), self.rot, self.dtype)
                for y in (x, swapped)]
        size = torch.cat([sums[0][..., :h], sums[1][..., :h], sums[0][..., 2 * h:].abs()], -1)
        half_step = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24
        off = (self.q.double().view(T, H, D) - turned[:, :H]).abs()
        fits = bool((off <= half_step * turned[:, :H].abs() + 2.0 ** -22 * size[:, :H]).all())
        assert fits
        written = torch.zeros(self.k.shape[:1] + self.k.shape[2:3], dtype=torch.bool, device=DEV)
        live = self.slots[self.slots >= 0].long()
        written[live // self.page, live % self.page] = True
        touched = written.any(1)
        for got, sc, was, sc_was, rows, sizes in ((self.k, self.ks, self.k0, self.ks0, turned[:, H:], size[:, H:]),
                                                  (self.v, self.vs, self.v0, self.vs0, x[:, H + KVH:], None)):
            want, sc_want = was.double(), sc_was.double()
            plain.write_rows(want, sc_want, rows, self.slots.tolist())
            assert torch.equal(sc.double(), sc_want)
            # pages that no token goes to keep their bytes
            assert torch.equal(got.view(torch.uint8)[~touched], was.view(torch.uint8)[~touched])
            have = got.double()
            if sizes is None or self.rot == 0:
                assert torch.equal(have, want)
                continue
            # other rows of the pages: exact; rows of this call: by the bound
            rest = (~written)[:, None, :, None].expand_as(have)
            assert torch.equal(have[rest], want[rest])
            p, a = live // self.page, live % self.page
            s = sc.double()[p][..., None]
            keep = self.slots >= 0
            off = (have[p, :, a] * s - rows[keep]).abs()
            fits = bool((off <= 2.0 ** -4 * rows[keep].abs() + 2.0 ** -10 * s + 2.0 ** -21 * sizes[keep]).all())
            assert fits
            # and nearly all of them are the very values of 64 bits (a rounding's border is hit by one in 2^-22 / 2^-4)
            assert float((have != want).double().mean()) < 1e-3


@pytest.mark.parametrize("case", WRITES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-r{c[5]}-p{c[6]}")
def test_write(ops, case):
    w = Write(*case)
    w.run(ops)
    w.check()


def test_write_twice_is_the_same(ops):
    w = Write(*WRITES[5])
    w.run(ops)
    first = [t.clone() for t in (w.q, w.k.view(torch.uint8), w.v.view(torch.uint8), w.ks, w.vs)]
    w.run(ops)
    assert all(torch.equal(a, b) for a, b in zip(first, (w.q, w.k.view(torch.uint8), w.v.view(torch.uint8), w.ks, w.vs)))


def test_a_page_grows_row_by_row(ops):
    """Rows of growing size one call at a time: what stands in the page after each, old rows among it."""
    H, KVH, D, page = 2, 2, 64, 16
    g = gen(5)
    k, ks = pages_of(3, KVH, page, D, g)
    v, vs = pages_of(3, KVH, page, D, g)
    wants = [[t.double(), s.double()] for t, s in ((k, ks), (v, vs))]
    cos, sin = rope_tables(64, 0)
    for i, mag in enumerate([1.0, 0.5, 3.0, 2.0 ** -20, 1e6, 0.0, 7.0, 2.0 ** 30, 1.0]):
        x = torch.randn((1, (H + 2 * KVH) * D), generator=g, device=DEV).mul(mag).to(BF16)
        slots = i32([2 * page + i])
        ops.rope_kv_write_q8(torch.empty((1, H * D), dtype=BF16, device=DEV), x, i32([i]), cos, sin, H, KVH, D, 0, k, v, ks, vs, slots, page)
        rows = x.double().view(1, -1, D)
        for (want, s), got, gs, r in zip(wants, (k, v), (ks, vs), (rows[:, H:H + KVH], rows[:, H + KVH:])):
            plain.write_rows(want, s, r, slots.tolist())
            assert torch.equal(gs.double(), s)
            assert torch.equal(got.double()[2, :, : i + 1], want[2, :, : i + 1])
            assert torch.equal(got.double()[:2], want[:2])


def test_what_is_not_finite_makes_its_page_nan_until_it_is_begun_anew(ops):
    H, KVH, D, page = 2, 2, 128, 16
    g = gen(6)
    cos, sin = rope_tables(64, D)
    for bad in (math.inf, -math.inf, math.nan, 3e18):
        k, ks = pages_of(3, KVH, page, D, g)
        v, vs = pages_of(3, KVH, page, D, g)

        def put(first, n, value=None):
            x = torch.randn((n, (H + 2 * KVH) * D), generator=g, device=DEV).to(BF16)
            if value is not None:
                x.view(n, -1, D)[0, H] = value                    # the first kv head's key
                x.view(n, -1, D)[0, H + KVH + 1, 5] = value       # the second kv head's value
            pos = torch.arange(first, first + n, device=DEV).int()
            ops.rope_kv_write_q8(torch.empty((n, H * D), dtype=BF16, device=DEV), x, pos, cos, sin, H, KVH, D, D, k, v, ks, vs,
                                 page + pos, page)
        put(0, 5)
        put(5, 3, bad)
        assert ks[1].isnan().tolist() == [True, False] and vs[1].isnan().tolist() == [False, True]
        put(8, 10)                                                # goes on into the next page
        assert ks[1].isnan().tolist() == [True, False] and vs[1].isnan().tolist() == [False, True]
        assert not ks[2].isnan().any() and not vs[2].isnan().any()
        assert not k.double().isnan().any() and not v.double().isnan().any()      # the values never hold one
        put(0, 3)
        assert not ks.isnan().any() and not vs.isnan().any()


def test_rows_without_a_slot_are_not_written(ops):
    w = Write([1, 1, 20, 1], [3, 16, 40, 9], 4, 2, 64, 64, 16, BF16)
    w.slots[1] = -1
    w.slots[5:9] = -1
    w.run(ops)
    w.check()


def test_queries_alone_and_queries_as_columns_of_a_wider_tensor(ops):
    w = Write([30], [3], 4, 2, 128, 128, 16, BF16)
    wide = torch.zeros((30, 3 * 512), dtype=BF16, device=DEV)
    w.q = wide[:, 512:1024]
    w.run(ops)
    w.check()
    assert not wide[:, :512].any() and not wide[:, 1024:].any()
    alone = torch.zeros((30, 512), dtype=BF16, device=DEV)
    ops.rope_kv_write_q8(alone, w.x, w.positions, w.cos, w.sin, 4, 2, 128, 128, None, None, None, None, w.slots, 16)
    assert torch.equal(alone, w.q)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_queries_within_the_rows_they_come_from_are_refused(ops, dtype):
    w = Write([5], [3], 4, 2, 64, 64, 16, dtype)
    before, held = w.x.clone(), w.k.clone()
    w.q = w.x[:, :256]
    with pytest.raises(KernelError, match="lie in qkv"):
        w.run(ops)
    assert torch.equal(w.x, before) and torch.equal(w.k.view(torch.uint8), held.view(torch.uint8))


# ------------------------------------------------------------------------------------------------------------ attention

class Attend:
    def __init__(self, q_lens, lens, H, KVH, D, page, window=0, dtype=BF16, seed=0, limit=0, std=1.0):
        g = gen(seed + sum(lens) + D + H)
        self.q_lens, self.lens, self.page, self.window, self.KVH = q_lens, lens, page, window, KVH
        self.tables, total = tables_for(lens, page, g)
        self.k, self.ks = pages_of(total, KVH, page, D, g)
        self.v, self.vs = pages_of(total, KVH, page, D, g, spread=6)
        T = sum(q_lens)
        self.q = (torch.randn((T, H, D), generator=g, device=DEV) * std).to(dtype)
        self.out = torch.full((T, H * D), 7.0, dtype=dtype, device=DEV)
        self.scale = D ** -0.5
        nd = 0
        while nd < len(q_lens) and q_lens[nd] == 1:
            nd += 1
        starts = [sum(q_lens[:b]) for b in range(len(q_lens) + 1)]
        self.step = SimpleNamespace(num_requests=len(q_lens), num_decode=nd, q_start=i32(starts), seq_lens=i32(lens),
                                    max_q_len=max(q_lens), max_seq_len=limit or max(lens), settled=True)

    def run(self, ops):
        ops.attention_q8(self.out, self.q, self.k, self.v, self.ks, self.vs, self.tables, self.step, self.KVH, self.page, self.scale,
                         self.window)
        return self.out

    def check(self):
        T, H, D = self.q.shape
        want, size, mags = plain.attend(self.q, self.k, self.v, self.ks, self.vs, self.tables, self.q_lens, self.lens, self.page,
                                        self.scale, self.window)
        got = self.out.double().view(T, H, D)
        n = min(max(self.lens), self.window or max(self.lens))
        half_step = 2.0 ** -8 if self.out.dtype == BF16 else 2.0 ** -24
        # the largest value of any page seen bounds what the smallest weights lose
        top = float((self.vs[~self.vs.isnan()].max() if (~self.vs.isnan()).any() else 0.0)) * 448.0
        bound = (half_step * want.abs() + (2 * (D + 4) * 2.0 ** -24 * mags + 2.0 ** -17 + n * 2.0 ** -24) * size)
        if self.out.dtype == BF16:
            bound = bound + 2.0 ** -11 * size + n * 2.0 ** -25 * top
        bad = want.isnan()
        assert torch.equal(bad, got.isnan())
        off = (got - want).abs()
        ok = (off <= bound) | bad
        assert bool(ok.all()), (float((off / bound)[~bad].max()), ok.logical_not().nonzero()[:4].tolist())


ATTENDS = [
    # (tokens brought, contexts, H, KVH, D, page, window)
    ([1], [1], 12, 2, 128, 64, 0),
    ([1], [57], 12, 2, 128, 64, 0),
    ([1] * 5, [1, 31, 32, 33, 65], 12, 2, 128, 16, 0),
    ([1] * 8, [2048 - 37 * i for i in range(8)], 12, 2, 128, 64, 0),
    ([1] * 3, [500, 0, 17], 14, 2, 64, 16, 0),                 # a row that pads the batch: zeros
    ([1] * 40, [100 + 90 * i for i in range(40)], 28, 4, 128, 16, 0),
    ([1] * 2, [6001, 13], 40, 8, 128, 64, 0),
    ([1], [30011], 12, 2, 128, 64, 0),
    ([1] * 6, [40, 700, 300, 301, 1024, 5], 12, 2, 128, 16, 300),
    ([1] * 2, [1000, 64], 16, 1, 64, 32, 0),                   # 16 heads over one
    ([1] * 2, [1000, 64], 9, 1, 128, 16, 37),
    ([1] * 2, [333, 64], 3, 3, 128, 16, 0),                    # a head each
    ([1] * 2, [333, 64], 34, 2, 128, 16, 0),                   # 17 heads over one: no fast variant
    ([1] * 3, [333, 64, 8], 6, 2, 80, 7, 50),                  # sizes that no fast variant takes
    ([1] * 2, [200, 9], 4, 2, 128, 5, 0),                      # pages of 5
    ([1] * 130, [20 + i for i in range(130)], 14, 2, 64, 16, 0),
    ([2], [2], 12, 2, 128, 64, 0),
    ([300], [300], 12, 2, 128, 64, 0),
    ([129], [1130], 28, 4, 128, 16, 0),
    ([65, 200, 3], [65, 777, 1003], 14, 2, 64, 16, 0),
    ([200, 64], [500, 64], 12, 2, 128, 64, 100),               # a window shorter than the portion
    ([90], [1500], 14, 2, 64, 32, 70),
    ([50, 7], [60, 9], 6, 2, 80, 7, 11),
    ([40], [141], 8, 1, 256, 16, 0),
    ([1, 1, 1, 130, 2], [99, 640, 1, 463, 150], 28, 4, 128, 16, 0),
    ([1, 1, 77], [99, 640, 463], 5, 5, 128, 64, 128),
    ([500], [2500], 40, 8, 128, 64, 0),
]
ids = [f"{len(c[0])}x{max(c[0])}of{max(c[1])}-{c[2]}-{c[3]}-{c[4]}-p{c[5]}-w{c[6]}" for c in ATTENDS]


@pytest.mark.parametrize("case", ATTENDS, ids=ids)
def test_attention(ops, case):
    a = Attend(*case)
    a.run(ops)
    a.check()


@pytest.mark.parametrize("case", [ATTENDS[2], ATTENDS[8], ATTENDS[19], ATTENDS[24]], ids=lambda c: f"{len(c[0])}x{max(c[0])}")
def test_attention_float32(ops, case):
    a = Attend(*case, dtype=torch.float32)
    a.run(ops)
    a.check()


@pytest.mark.parametrize("case", [ATTENDS[3], ATTENDS[6], ATTENDS[18], ATTENDS[24]], ids=lambda c: f"{len(c[0])}x{max(c[0])}")
def test_scores_far_apart(ops, case):
    """Queries eight times larger: weights from 1 down to nothing."""
    a = Attend(*case, std=4.0, seed=3)
    a.run(ops)
    a.check()


@pytest.mark.parametrize("case", [ATTENDS[3], ATTENDS[5], ATTENDS[24], ATTENDS[20]], ids=lambda c: f"{len(c[0])}x{max(c[0])}")
def test_rows_that_were_never_written_are_not_seen(ops, case):
    """Behind a request's last row, in the null page and in pages that nobody holds: any bytes, scales of NaN."""
    a = Attend(*case)
    used = torch.zeros(a.k.shape[0], dtype=torch.bool, device=DEV)
    for b, n in enumerate(a.lens):
        held = -(-n // a.page)
        used[a.tables[b, :held].long()] = True
        if n % a.page:
            for c in (a.k, a.v):
                c.view(torch.uint8)[a.tables[b, held - 1].long(), :, n % a.page:] = 0x7f
    for s in (a.ks, a.vs):
        s[~used] = math.nan
    for c in (a.k, a.v):
        c.view(torch.uint8)[~used] = 0xff
    a.run(ops)
    a.check()


@pytest.mark.parametrize("case", [ATTENDS[3], ATTENDS[8], ATTENDS[18], ATTENDS[20], ATTENDS[24], ATTENDS[22]],
                         ids=lambda c: f"{len(c[0])}x{max(c[0])}w{c[6]}")
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_page_of_nan_reaches_the_rows_that_see_it_alone(ops, case, which):
    a = Attend(*case)
    b = len(a.lens) - 1
    for lp in {0, a.lens[b] // (2 * a.page)}:
        (a.ks if which == "k" else a.vs)[a.tables[b, lp].long(), 0] = math.nan
    a.run(ops)
    a.check()


def test_a_query_that_is_not_finite_is_its_own_row_alone(ops):
    for case in (ATTENDS[3], ATTENDS[24], ATTENDS[17]):
        a = Attend(*case)
        rows = ((0, 1, math.nan), (2, 0, math.inf), (4, 2, -math.inf))
        for t, h, x in rows:
            a.q[t, h, 5] = x
        clean = a.q.clone()
        for t, h, _ in rows:
            clean[t, h] = 0
        a.run(ops)
        got = a.out.view(a.q.shape).clone()
        for t, h, _ in rows:
            assert got[t, h].isnan().all()
        a.q = clean
        a.run(ops)
        for t, h, _ in rows:
            got[t, h] = a.out.view(a.q.shape)[t, h]
        assert torch.equal(got, a.out.view(a.q.shape))


@pytest.mark.parametrize("case", [ATTENDS[3], ATTENDS[18]], ids=["singles", "portion"])
def test_scales_over_the_whole_range(ops, case):
    """Pages whose values are 2^-50, 1 and 2^50 of each other's size: nothing is lost against the largest contribution."""
    a = Attend(*case)
    for s in (a.vs,):
        pick = torch.randint(0, 3, s.shape, generator=gen(9), device=DEV)
        s.copy_(torch.tensor([2.0 ** -50, 1.0, 2.0 ** 50], device=DEV)[pick])
    a.run(ops)
    want, size, mags = plain.attend(a.q, a.k, a.v, a.ks, a.vs, a.tables, a.q_lens, a.lens, a.page, a.scale, a.window)
    T, H, D = a.q.shape
    n = max(a.lens)
    # (a half float's weight is off by 2^-25 of the largest weight * scale, times 448 at most, over n keys; the largest is at most
    # the sum of all, size / 2^-3 where its values are not all small)
    bound = 2.0 ** -8 * want.abs() + (2 * (D + 4) * 2.0 ** -24 * mags + 2.0 ** -17 + n * 2.0 ** -24 + 2.0 ** -11) * size
    bound = bound + n * 2.0 ** -25 * 448 * size.amax(-1, keepdim=True)
    fits = bool(((a.out.double().view(T, H, D) - want).abs() <= bound).all())
    assert fits


@pytest.fixture
def forced(ops):
    """Sets the instance of the portions' kernel and the splits of the single tokens'; the rules hold again afterwards."""
    def force(row_tiles=0, splits=0, clusters=True, portion_splits=0):
        ops.lib.ts_set_q8_prefill(row_tiles)
        ops.lib.ts_set_q8_prefill_splits(portion_splits)
        ops.q8_splits, ops.q8_clusters = splits, clusters
    yield force
    force()


@pytest.mark.parametrize("row_tiles", [1, 2])
@pytest.mark.parametrize("case", [c for c in ATTENDS if max(c[0]) > 1] + [([513, 2, 700], [1025, 2, 5000], 12, 2, 128, 16, 0),
                                                                            ([400], [400], 34, 2, 64, 48, 0)],
                         ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}-{c[4]}-w{c[6]}")
def test_one_and_two_row_tiles(ops, forced, case, row_tiles):
    forced(row_tiles=row_tiles, portion_splits=1)
    for std in (1.0, 4.0):
        a = Attend(*case, std=std)
        a.run(ops)
        a.check()


@pytest.mark.parametrize("splits", [2, 4, 8])
@pytest.mark.parametrize("case", [c for c in ATTENDS if max(c[0]) > 1] + [([513, 2, 700], [1025, 2, 5000], 12, 2, 128, 16, 0),
                                                                            ([400], [400], 34, 2, 64, 48, 0), ([3, 2, 9], [3000, 2, 1100], 4, 1, 128, 64, 700)],
                         ids=lambda c: f"{len(c[0])}x{max(c[0])}of{max(c[1])}-{c[4]}-w{c[6]}")
def test_portions_cut_over_blocks(ops, forced, case, splits):
    forced(row_tiles=1, portion_splits=splits)
    for std in (1.0, 4.0):
        a = Attend(*case, std=std)
        a.run(ops)
        a.check()


@pytest.mark.parametrize("splits", [2, 8])
def test_a_portion_cut_over_blocks_sees_nan_where_it_does(ops, forced, splits):
    """Shares whose keys are all NaN, none, or some, against one block for all of them: NaN in the same rows, the same values elsewhere.
    (Either is off by 2^-8 of the output, and by weights of 2^-11 and sums in 32 bits, below 2^-10 of the largest value together.)"""
    for poisoned in ([0], [7], list(range(3, 12)), list(range(25))):
        outs = []
        for n in (1, splits):
            forced(row_tiles=1, portion_splits=n)
            a = Attend([700], [1600], 6, 2, 128, 64, 500)
            a.ks[a.tables[0][poisoned].long()] = math.nan
            a.run(ops)
            outs.append(a.out.float())
        assert torch.equal(outs[0].isnan(), outs[1].isnan())
        off = (outs[0] - outs[1]).nan_to_num().abs()
        top = float((a.v.float() * a.vs[..., None, None]).abs().max())
        assert float(off.max()) <= 2 * (2.0 ** -8 * float(outs[0].nan_to_num().abs().max()) + 2.0 ** -10 * top)


@pytest.mark.parametrize("splits,clusters", [(1, False), (2, True), (3, False), (5, True), (8, True), (8, False), (29, False), (128, False)])
@pytest.mark.parametrize("case", [ATTENDS[2], ATTENDS[3], ATTENDS[4], ATTENDS[6], ATTENDS[8], ATTENDS[9], ATTENDS[10], ATTENDS[14]],
                         ids=lambda c: f"{len(c[0])}of{max(c[1])}-{c[2]}-{c[4]}-p{c[5]}-w{c[6]}")
def test_single_tokens_cut_over_blocks(ops, forced, case, splits, clusters):
    """More blocks than tiles among them: blocks and warps without a key."""
    forced(splits=splits, clusters=clusters)
    a = Attend(*case)
    if len(a.lens) > 2:
        a.vs[a.tables[0, 0].long(), 0] = math.nan                  # (a part that is all NaN, beside parts without keys)
    a.run(ops)
    a.check()


def test_a_cache_of_more_than_2_32_bytes(ops):
    """Its last pages: written, and read by single tokens and by a portion."""
    H, KVH, D, page = 8, 8, 128, 64
    total = (1 << 32) // (KVH * page * D) + 2000
    k, v = (torch.empty((total, KVH, page, D), dtype=F8, device=DEV) for _ in range(2))
    ks, vs = torch.ones((total, KVH), device=DEV), torch.ones((total, KVH), device=DEV)
    assert k.numel() > 1 << 32
    a = Attend([1, 1, 150], [700, 65, 333], H, KVH, D, page)
    moved = a.tables + (total - 1 - a.k.shape[0])
    for b, n in enumerate(a.lens):
        held = -(-n // page)
        for big, small in ((k, a.k), (v, a.v), (ks, a.ks), (vs, a.vs)):
            big[moved[b, :held].long()] = small[a.tables[b, :held].long()]
    want = a.run(ops).clone()
    a.k, a.v, a.ks, a.vs, a.tables = k, v, ks, vs, moved.contiguous()
    assert torch.equal(a.run(ops), want)
    w = Write([70, 1], [10, 40], H, KVH, D, D, page, BF16)
    w.run(ops)
    w_slots, shift = w.slots, (total - 10) * page
    outs = [t.clone() for t in (w.k, w.v, w.ks, w.vs)]
    for big, small in ((k, w.k0), (v, w.v0), (ks, w.ks0), (vs, w.vs0)):
        big[total - 10:total - 10 + small.shape[0]] = small
    w.slots = w_slots + shift
    ops.rope_kv_write_q8(w.q, w.x, w.positions, w.cos, w.sin, H, KVH, D, D, k, v, ks, vs, w.slots, page)
    for big, small in zip((k, v, ks, vs), outs):
        got = big[total - 10:total - 10 + small.shape[0]]
        assert torch.equal(got.reshape(-1).view(torch.uint8), small.reshape(-1).view(torch.uint8))


def test_a_negative_scale_and_none(ops):
    for scale in (-0.09, 0.0):
        for case in (ATTENDS[3], ATTENDS[24], ATTENDS[22]):
            a = Attend(*case)
            a.scale = scale
            a.run(ops)
            plus = Attend(*case)
            plus.scale, plus.q = abs(scale), -plus.q if scale < 0 else plus.q
            want, size, mags = plain.attend(plus.q, a.k, a.v, a.ks, a.vs, a.tables, a.q_lens, a.lens, a.page, abs(scale), a.window)
            bound = 2.0 ** -8 * want.abs() + (2 * 132 * 2.0 ** -24 * mags + 2.0 ** -17 + 2100 * 2.0 ** -24 + 2.0 ** -11) * size
            fits = bool(((a.out.double().view(a.q.shape) - want).abs() <= bound + 2100 * 2.0 ** -25 * float(a.vs.max()) * 448).all())
            assert fits


def test_portions_with_caches_in_any_order_in_memory(ops):
    """Values before keys, keys and values far apart."""
    for case in (ATTENDS[3], ATTENDS[24]):
        a = Attend(*case)
        want = a.run(ops).clone()
        both = torch.empty((2, *a.k.shape), dtype=F8, device=DEV)
        both[0], both[1] = a.v, a.k
        a.v, a.k = both[0], both[1]
        assert torch.equal(a.run(ops), want)


def test_strides(ops):
    """Queries and outputs as columns of wider tensors."""
    for case in (ATTENDS[3], ATTENDS[24]):
        a = Attend(*case)
        T, H, D = a.q.shape
        plain_out = a.run(ops).clone()
        wide_q = torch.randn((T, 3 * H * D), device=DEV).to(BF16)
        wide_q[:, H * D:2 * H * D] = a.q.reshape(T, -1)
        wide_o = torch.zeros((T, 2 * H * D + 8), dtype=BF16, device=DEV)
        a.q = wide_q[:, H * D:2 * H * D].view(T, H, D)
        a.out = wide_o[:, 8:H * D + 8]
        a.run(ops)
        assert torch.equal(a.out, plain_out)
        assert not wide_o[:, :8].any() and not wide_o[:, H * D + 8:].any()


def test_the_same_bits_whatever_the_longest_context(ops):
    """A captured step is launched for the longest context that the engine allows."""
    for case in (ATTENDS[3], ATTENDS[24]):
        a, b = Attend(*case), Attend(*case, limit=40000)
        b.tables = torch.cat([b.tables, torch.zeros((b.tables.shape[0], 600), dtype=torch.int32, device=DEV)], 1).contiguous()
        b.run(ops)
        b.check()
        a.run(ops)
        a.check()


def test_captured_and_replayed_beside_eager_calls(ops):
    """Two captured calls and eager ones between them: each has its own answer, replay after replay."""
    a, b = Attend(*ATTENDS[6], limit=8000), Attend(*ATTENDS[24])
    want_a, want_b = a.run(ops).clone(), b.run(ops).clone()
    graphs = []
    for x in (a, b):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            x.run(ops)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.run(ops)
        graphs.append(g)
    other = Attend([1] * 20, [3000] * 20, 28, 4, 128, 16)
    want_other = other.run(ops).clone()
    for _ in range(3):
        for x in (a, b, other):
            x.out.fill_(3.0)
        graphs[0].replay()
        other.run(ops)
        graphs[1].replay()
        assert torch.equal(a.out, want_a) and torch.equal(b.out, want_b) and torch.equal(other.out, want_other)


def test_another_stream(ops):
    a = Attend(*ATTENDS[6])
    want = a.run(ops).clone()
    side = torch.cuda.Stream()
    a.out.fill_(3.0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.run(ops)
    side.synchronize()
    assert torch.equal(a.out, want)


# ---------------------------------------------------------------------------------------------------- both, as they run

@pytest.mark.parametrize("H,KVH,D,page,window", [(12, 2, 128, 64, 0), (14, 2, 64, 16, 100), (28, 4, 128, 16, 0)])
def test_portions_then_single_tokens(ops, H, KVH, D, page, window):
    """A prompt in portions and then token by token: after every step the pages are what 64 bits say, and so are the outputs."""
    g = gen(11)
    lens, total = [0, 0], 40
    cuts = [[150, 31], [77, 0], [1, 1], [1, 1], [1, 1]]
    ids = (torch.randperm(total - 1, generator=g, device=DEV) + 1).int()
    tables = ids[:38].view(2, 19).contiguous()
    k, ks = torch.zeros((total, KVH, page, D), dtype=F8, device=DEV), torch.ones((total, KVH), device=DEV)
    v, vs = k.clone(), ks.clone()
    cos, sin = rope_tables(400, D)
    for cut in cuts:
        who = [b for b in range(2) if cut[b]]
        q_lens = [cut[b] for b in who]
        T = sum(q_lens)
        x = torch.randn((T, (H + 2 * KVH) * D), generator=g, device=DEV).to(BF16)
        pos = torch.cat([torch.arange(lens[b], lens[b] + cut[b], device=DEV) for b in who]).int()
        slots = torch.cat([tables[b][(p := torch.arange(lens[b], lens[b] + cut[b], device=DEV)) // page] * page + p % page
                           for b in who]).int()
        q = torch.empty((T, H * D), dtype=BF16, device=DEV)
        was = [t.double() for t in (k, ks, v, vs)]
        ops.rope_kv_write_q8(q, x, pos, cos, sin, H, KVH, D, D, k, v, ks, vs, slots, page)
        rows = x.double().view(T, -1, D)
        plain.write_rows(was[2], was[3], rows[:, H + KVH:], slots.tolist())
        assert torch.equal(v.double(), was[2]) and torch.equal(vs.double(), was[3])
        for b in who:
            lens[b] += cut[b]
        a = Attend.__new__(Attend)
        a.q_lens, a.lens, a.page, a.window, a.KVH = q_lens, [lens[b] for b in who], page, window, KVH
        a.k, a.v, a.ks, a.vs, a.q, a.scale = k, v, ks, vs, q.view(T, H, D), D ** -0.5
        a.tables = tables[who].contiguous()
        a.out = torch.empty((T, H * D), dtype=BF16, device=DEV)
        starts = [sum(q_lens[:i]) for i in range(len(who) + 1)]
        a.step = SimpleNamespace(num_requests=len(who), num_decode=sum(n == 1 for n in q_lens), q_start=i32(starts),
                                 seq_lens=i32(a.lens), max_q_len=max(q_lens), max_seq_len=max(a.lens), settled=False)
        a.run(ops)
        a.check()
