"""The kernels around a cache that is held in 8 bits, against plain forms in float64.

Bounds. A rounding is off by half a step: 2^-8 of the number in bfloat16, 2^-11 and 2^-24 in fp16 and float32, 2^-4 in e4m3.

store: a number that is not rotated is stored by two exact operations (a product with a power of two, one rounding), so codes and
scales are those of the oracle. A rotated one is x1 cos - x2 sin in float32: cosine and sine within 2 units (2^-22), two products
and a sum, off by at most 2^-21 (|x1| + |x2|); then rounded, to the queries' type or to e4m3 (in steps of 2^-9 scale at least).

attention, float32 arithmetic: a score is off by e_s <= (D + 4) 2^-24 times sum |q k| scale, a weight by a factor of
1 +- 2 e_s + (n + 8) 2^-23 (exp, the sums of n terms), which is at most that share of sum w |v|.
attention, matrix cores: products of bfloat16 numbers are exact and their sums float32, so scores are as above; a weight is rounded to
bfloat16 in numerator and denominator, 2 * 2^-8 of sum w |v|; the result is rounded, 2^-8 of itself and at most
2^-8 of what it is off.
"""
import math
import random

import pytest
import torch

import plain_f8
from plain_f8 import F8

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu_device):
    from pytriton_llama_amd import ops
    return ops


# ---- store ---------------------------------------------------------------------------------------
def empty_cache(pages, Hkv, P, D):
    """Codes that an earlier owner has left (also NaNs) and scales that are no longer anybody's."""
    g = torch.Generator().manual_seed(3)
    codes = torch.randint(0, 256, (2, pages, Hkv, P, D), generator=g, dtype=torch.uint8).view(F8)
    return codes.cuda(), torch.full((2, pages, Hkv), 2.0 ** 100, device="cuda")


STORES = [  # dtype, Hq, Hkv, D, page size
    (torch.bfloat16, 8, 2, 64, 16), (torch.bfloat16, 4, 4, 128, 16), (torch.float32, 6, 3, 64, 16),
    (torch.bfloat16, 4, 1, 96, 32), (torch.bfloat16, 10, 5, 128, 64), (torch.float32, 2, 1, 30, 5), (torch.bfloat16, 3, 3, 34, 7),
    (torch.float32, 2, 2, 2, 1), (torch.bfloat16, 16, 8, 256, 16), (torch.bfloat16, 2, 2, 640, 3), (torch.float32, 4, 2, 128, 128),
]


def steps_of(P, pages):
    """Steps of a few sequences, as (sequence, tokens) lists: portions that begin and end inside pages, and single tokens."""
    return [[(0, 1), (1, 2 * P + 3)], [(0, 1), (1, 1), (2, P)], [(2, 1), (0, 1), (1, max(1, P - 1))], [(0, 1), (1, 1), (2, 1)],
            [(3, 1)], [(3, 3 * P), (0, 2)]]


@pytest.mark.parametrize("rotated", [False, True], ids=["as they are", "rotated"])
@pytest.mark.parametrize("dtype,Hq,Hkv,D,P", STORES)
def test_store(ops, dtype, Hq, Hkv, D, P, rotated):
    g = torch.Generator().manual_seed(D * P + Hq)
    pages = 40
    (kc, vc), (ks, vs) = empty_cache(pages, Hkv, P, D)
    plain = [plain_f8.Blocks(kc.cpu(), ks.cpu()), plain_f8.Blocks(vc.cpu(), vs.cpu())]
    rng = random.Random(1)
    free = list(range(pages))
    rng.shuffle(free)
    table, length = {}, {}
    inv_freq = 10000.0 ** (-torch.arange(0, D, 2).float() / D) if rotated else None
    used = set()
    for step in steps_of(P, pages):
        positions, slots = [], []
        for s, n in step:
            start = length.get(s, 0)
            for p in range(start, start + n):
                if p % P == 0:
                    table.setdefault(s, []).append(free.pop())
                slots.append(table[s][p // P] * P + p % P)
                positions.append(p + 5000 * s)
            length[s] = start + n
        slots += [-1, pages * P, -1]                 # tokens that are not stored
        positions += [0, 7, 100000]
        T = len(slots)
        # one row stride of a fused projection; sizes from tiny to large, so that scales grow
        x = torch.randn(T, (Hq + 2 * Hkv) * D + 16, generator=g) * torch.exp(3 * torch.randn(T, 1, generator=g))
        x = x.to(dtype)
        q, k, v = (x[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
        pos = torch.tensor(positions, dtype=torch.int32)
        xd = x.cuda()
        qd, kd, vd = (xd[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
        sd = torch.tensor(slots, dtype=torch.int32, device="cuda")
        for again in range(2):                       # the same once more changes nothing
            got_q = ops.rope_store_f8(qd, kd, vd, pos.cuda(), None if inv_freq is None else inv_freq.cuda(), sd, kc, vc, ks, vs)
        assert torch.equal(xd.cpu(), x)              # what is read stays as it was
        want_q = plain_f8.rotate(q, pos, inv_freq)
        half = D // 2
        both = q.double().abs()[..., :half] + q.double().abs()[..., half:]
        slack = 2.0 ** -21 * torch.cat([both, both], -1) if rotated else 0
        step_q = 2.0 ** (-8 if dtype == torch.bfloat16 else -24)
        assert ((got_q.cpu().double() - want_q).abs() <= slack * (1 + step_q) + step_q * want_q.abs()).all()
        new = [plain_f8.rotate(k, pos, inv_freq), v.double()]
        for blocks, x_new in zip(plain, new):
            blocks.store(x_new, slots)
        used |= {s // P for s in slots if 0 <= s < pages * P}
        at = sorted(used)
        for blocks, codes, scale, turned in zip(plain, (kc, vc), (ks, vs), (rotated, False)):
            held = codes.cpu().float().double()[at] * scale.cpu().double()[at][:, :, None, None]
            want = blocks.held[at]
            if not turned:
                assert torch.equal(scale.cpu().double()[at], blocks.scale[at])
                assert torch.equal(held, want)
            else:
                # (a number at the edge of two scales may have taken the other one)
                ratio = scale.cpu().double()[at] / blocks.scale[at]
                assert ((ratio == 1) | (ratio == 2) | (ratio == 0.5)).all() and (ratio != 1).double().mean() <= 0.01
                s = torch.maximum(scale.cpu().double()[at], blocks.scale[at])[:, :, None, None]
                # the oracle's number is within half a step of what was stored, and so is the kernel's; both may have been rounded
                # anew as often as the scale grew, where numbers are steps of 2^-9 scale
                assert ((held - want).abs() <= 2 * 2.0 ** -4 * want.abs() + 2.0 ** -9 * s).all()
                assert ((held - want).abs() > 2.0 ** -9 * s).double().mean() <= 1e-3
        # (so that what one step left of a tie does not go on to the next)
        for blocks, codes, scale in zip(plain, (kc, vc), (ks, vs)):
            blocks.scale[at] = scale.cpu().double()[at]
            blocks.held[at] = codes.cpu().float().double()[at] * blocks.scale[at][:, :, None, None]
    others = [p for p in range(pages) if p not in used]
    (kc0, vc0), (ks0, vs0) = empty_cache(pages, Hkv, P, D)
    assert torch.equal(kc.view(torch.uint8)[others], kc0.view(torch.uint8)[others])
    assert torch.equal(vc.view(torch.uint8)[others], vc0.view(torch.uint8)[others])
    assert torch.equal(ks[others], ks0[others]) and torch.equal(vs[others], vs0[others])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_store_at_the_edges_of_numbers(ops, dtype):
    """Zeros, the smallest and largest numbers, edges of scales, ties, infinities and NaN."""
    P, D = 16, 32
    rows = torch.zeros(P, 1, D)
    rows[0, 0, :8] = torch.tensor([448.0, -448.0, 2.0 ** -6, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).tiny
    firsts = [448.0, 450.0, 1.75, 1.7578125, 2.0 ** -140 if dtype == torch.float32 else tiny, tiny, 0.0, big, 2.0 ** 127, 1.0]
    (kc, vc), (ks, vs) = empty_cache(len(firsts), 1, P, D)
    for page, f in enumerate(firsts):
        x = rows.clone()
        x[0, 0, 8] = f
        if page == 9:
            x[1, 0, 0], x[1, 0, 1], x[2, 0, 2] = math.inf, -math.inf, math.nan
        x = x.to(dtype)
        slots = torch.arange(page * P, page * P + P, dtype=torch.int32, device="cuda")
        xd = x.cuda()
        ops.rope_store_f8(xd, xd, xd, slots, None, slots, kc, vc, ks, vs)
        want = plain_f8.Blocks(torch.zeros(len(firsts), 1, P, D).to(F8), torch.ones(len(firsts), 1))
        want.store(x.double(), slots.tolist())
        got = kc[page].cpu().float().double() * ks[page].cpu().double()[:, None, None]
        assert torch.equal(ks[page].cpu().double(), want.scale[page])
        assert torch.equal(got.nan_to_num(-7.0), want.held[page].nan_to_num(-7.0))
        assert torch.equal(torch.isnan(got), torch.isnan(want.held[page]))
    assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8))


@pytest.mark.parametrize("T,rotated", [(1, True), (5, True), (16, True), (16, False)])
@pytest.mark.parametrize("D", [64, 34])
def test_store_of_rows_that_lack_their_norms_factor(ops, T, rotated, D):
    """The factor of a row is rsqrt(mean square + eps), off by at most 2^-20 here (a float32 sum of 80 numbers and the root); it
    comes in before the rotation, so the numbers stored are those of rows that have it, but for that and a tie."""
    Hq, Hkv, P = 6, 3, 16
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).bfloat16()
    partials = torch.rand(T, 80, generator=g) * 50
    f = torch.rsqrt(partials.double().sum(-1) / 512 + 1e-5)
    pos = torch.arange(7, 7 + T, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(0, D, 2).float() / D) if rotated else None
    slots = torch.arange(7, 7 + T, dtype=torch.int32)
    cut = lambda y: [y[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv))]   # noqa: E731
    codes, scales = torch.zeros(2, 3, Hkv, P, D).to(F8).cuda(), torch.full((2, 3, Hkv), 2.0 ** -126, device="cuda")
    got = ops.rope_store_f8(*cut(x.cuda()), pos.cuda(), None if inv is None else inv.cuda(), slots.cuda(), codes[0], codes[1], scales[0],
                            scales[1], ops.RowScale(partials.cuda(), 512, 1e-5))
    q, k, v = cut(x.double() * f[:, None])
    want = plain_f8.rotate(q, pos, inv)
    size = torch.cat([q.abs()[..., :D // 2] + q.abs()[..., D // 2:]] * 2, -1)
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -19 * size + 2.0 ** -8 * want.abs() * (1 + 2.0 ** -10)).all()
    for i, new in enumerate((plain_f8.rotate(k, pos, inv), v)):
        plain = plain_f8.Blocks(torch.zeros(3, Hkv, P, D).to(F8), torch.full((3, Hkv), 2.0 ** -126))
        plain.store(new, slots.tolist())
        held = codes[i].cpu().float().double() * scales[i].cpu().double()[:, :, None, None]
        s = plain.scale[:, :, None, None]
        assert ((held - plain.held).abs() <= 2 * 2.0 ** -4 * plain.held.abs() + 2.0 ** -9 * s).all()
        assert ((held - plain.held).abs() > 2.0 ** -9 * s).double().mean() <= 2e-3
    with pytest.raises(ops.KernelError):
        y = torch.zeros(17, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")
        c = [y[:, a * D:b * D].view(17, b - a, D) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv))]
        ops.rope_store_f8(*c, torch.zeros(17, dtype=torch.int32, device="cuda"), None, None, codes[0], codes[1], scales[0], scales[1],
                          ops.RowScale(torch.ones(17, 4, device="cuda"), 4, 0.0))


def test_store_of_nothing(ops):
    (kc, vc), (ks, vs) = empty_cache(3, 2, 16, 64)
    before = kc.view(torch.uint8).clone(), ks.clone()
    x = torch.randn(5, 6, 64, device="cuda").bfloat16()
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    f = torch.ones(32, device="cuda")
    out = ops.rope_store_f8(x[:, :2], x[:, 2:4], x[:, 4:], pos, f, None, kc, vc, ks, vs)
    assert torch.equal(kc.view(torch.uint8), before[0]) and torch.equal(ks, before[1]) and out.shape == (5, 2, 64)
    none = ops.rope_store_f8(x[:0, :2], x[:0, 2:4], x[:0, 4:], pos[:0], f, pos[:0], kc, vc, ks, vs)
    assert none.shape == (0, 2, 64)


# ---- attention -------------------------------------------------------------------------------------
class Step:
    """A step over an 8-bit cache: ``seqs`` (rows, context), queries as columns of a wider matrix."""

    def __init__(self, dtype, Hq, Hkv, D, P, seqs, window=0, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.args = Hq, Hkv, D, P
        self.window, self.scale = window, D ** -0.5
        self.q_start = [0]
        for r, _ in seqs:
            self.q_start.append(self.q_start[-1] + r)
        self.ctx = [c for _, c in seqs]
        held = [-(-c // P) for c in self.ctx]
        pages = sum(held) + 3
        order = torch.randperm(pages, generator=g).tolist()
        width = max(held + [1])
        self.table = [[-1] * width for _ in seqs]
        at = 0
        for i, n in enumerate(held):
            self.table[i][:n] = order[at:at + n]
            at += n
        x = [torch.randn(pages, Hkv, P, D, generator=g) * torch.exp(0.7 * torch.randn(pages, Hkv, 1, 1, generator=g)) for _ in range(2)]
        (self.kc, self.ks), (self.vc, self.vs) = (plain_f8.quantised(y) for y in x)
        self.k = self.kc.float().double() * self.ks.double()[:, :, None, None]
        self.v = self.vc.float().double() * self.vs.double()[:, :, None, None]
        # what lies behind a sequence's last key, in its own page and in pages of nobody, is NaN
        nan = torch.tensor(0x7f, dtype=torch.uint8)
        for codes in (self.kc, self.vc):
            raw = codes.view(torch.uint8)
            raw[order[at:]] = nan
            for i, c in enumerate(self.ctx):
                if c % P:
                    raw[self.table[i][c // P], :, c % P:] = nan
        # pages left of every window are gone
        if window:
            for i, (r, c) in enumerate(seqs):
                first = max(0, c - r - window + 1)
                for p in range(min(first // P, width)):
                    self.table[i][p] = -1
        T = self.q_start[-1]
        self.rows = T + 2                                     # (two rows behind the last sequence)
        self.wide = (spread * torch.randn(self.rows, Hq * D + 24, generator=g)).to(dtype)
        self.q = self.wide[:, 8:8 + Hq * D].view(self.rows, Hq, D)
        self.seqs = seqs

    def device(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
        Hq, _, D, _ = self.args
        self.qd = self.wide.cuda()[:, 8:8 + Hq * D].view(self.rows, Hq, D)
        self.out = torch.full((self.rows, Hq, D), 77.0, device="cuda", dtype=self.q.dtype)
        self.cache = [t.cuda() for t in (self.kc, self.vc, self.ks, self.vs)]
        self.tables = i32(self.q_start), i32(self.ctx), i32(self.table)
        return self

    def blocks(self, rows, first=0):
        items = [(i, o) for i, (r, _) in enumerate(self.seqs) if i >= first for o in range(0, r, rows)] + [(0, 1 << 20)]
        return (torch.tensor([i for i, _ in items], dtype=torch.int32, device="cuda"),
                torch.tensor([o for _, o in items], dtype=torch.int32, device="cuda"))

    def check(self, sink=None, first=0, last=None, matrix_cores=False):
        last = len(self.seqs) if last is None else last
        want, size, score = plain_f8.attention(self.q[:self.q_start[-1]], self.k, self.v, self.q_start, self.ctx, self.table, self.scale,
                                               self.window, None if sink is None else sink.cpu())
        a, b = self.q_start[first], self.q_start[last]
        got = self.out.cpu().double()
        assert (got[b:] == 77).all() and (got[:a] == 77).all()
        D, n = self.args[2], max(self.ctx)
        weights = 2 * (D + 4) * 2.0 ** -24 * score + (n + 8) * 2.0 ** -23 + (2 * 2.0 ** -8 if matrix_cores else 0)
        step = 2.0 ** (-8 if self.q.dtype == torch.bfloat16 else -24)
        bound = size * weights * (1 + step) + step * want.abs() + 1e-30
        off = (got[a:b] - want[a:b]).abs()
        assert not torch.isnan(off).any()
        worst = (off / bound[a:b]).max().item() if b > a else 0.0
        assert worst <= 1.0, f"off by {worst:.3f} of the bound"


SEQS = [(1, 1), (1, 2), (1, 16), (1, 17), (1, 0), (1, 127), (1, 128), (1, 129), (1, 300), (5, 5), (3, 40), (70, 203), (16, 16), (17, 33)]
GENERIC = [  # dtype, Hq, Hkv, D, page size, window
    (torch.float32, 8, 2, 64, 16, 0), (torch.bfloat16, 6, 2, 128, 16, 0), (torch.float32, 4, 4, 30, 5, 0), (torch.bfloat16, 3, 1, 33, 7, 9),
    (torch.float32, 2, 1, 256, 24, 50), (torch.bfloat16, 2, 2, 640, 3, 0), (torch.float32, 40, 2, 4, 1, 17), (torch.bfloat16, 2, 2, 96, 16, 1),
]


@pytest.mark.parametrize("dtype,Hq,Hkv,D,P,window", GENERIC)
def test_generic(ops, dtype, Hq, Hkv, D, P, window):
    s = Step(dtype, Hq, Hkv, D, P, SEQS, window, seed=D).device()
    ops.attention_generic_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(16), s.scale, window)
    s.check()


def test_generic_with_a_sink(ops):
    s = Step(torch.float32, 4, 2, 64, 16, SEQS, 0, seed=2).device()
    sink = torch.tensor([-3.0, 0.0, 2.5, 40.0], device="cuda")
    ops.attention_generic_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(16), s.scale, 0, sink)
    s.check(sink)


DECODE_SEQS = [(1, c) for c in (1, 2, 15, 16, 17, 0, 31, 32, 33, 127, 128, 129, 255, 500, 1027)]
DECODES = [  # Hq, Hkv, D, page size, window
    (32, 8, 64, 16, 0), (32, 8, 128, 16, 0), (6, 2, 96, 32, 0), (5, 1, 32, 64, 0), (16, 1, 64, 16, 0), (20, 1, 128, 16, 0),
    (66, 2, 64, 16, 0), (4, 4, 128, 128, 0), (8, 2, 64, 16, 100), (8, 2, 128, 16, 1), (8, 2, 96, 16, 33), (2, 2, 64, 1024, 130),
]


@pytest.mark.parametrize("Hq,Hkv,D,P,window", DECODES)
def test_decode(ops, Hq, Hkv, D, P, window):
    assert ops.attention_f8_fits(torch.bfloat16, Hq, Hkv, D, P)
    s = Step(torch.bfloat16, Hq, Hkv, D, P, DECODE_SEQS, window, seed=Hq + D, spread=1.5).device()
    tickets = torch.zeros(4 * len(s.seqs) * Hkv * -(-(Hq // Hkv) // 16), dtype=torch.int32, device="cuda")
    for _ in range(2):
        s.out.fill_(77.0)
        ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, len(s.seqs), s.scale, window, tickets=tickets)
        s.check(matrix_cores=True)
        assert not tickets.any()


@pytest.mark.parametrize("D", [64, 128])
def test_decode_of_the_first_sequences_with_a_sink(ops, D):
    s = Step(torch.bfloat16, 8, 4, D, 16, DECODE_SEQS + [(9, 30)], 0, seed=7).device()
    sink = torch.tensor([-3.0, 0.0, 2.5, 40.0, 1.0, -60.0, 5.0, 3.0], device="cuda")
    n = 13
    ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, n, s.scale, 0, sink)
    s.check(sink, last=n, matrix_cores=True)


@pytest.mark.parametrize("contexts", [[20011], [9000, 3], [4100] * 9, list(range(0, 1500, 21)), [7] * 300])
def test_decode_cut_into_parts(ops, contexts):
    """Long contexts and many sequences: parts of a pair that are merged, all kinds of places for a part's beginning and end."""
    s = Step(torch.bfloat16, 4, 2, 64, 16, [(1, c) for c in contexts], 0, seed=len(contexts), spread=2.0).device()
    ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, len(s.seqs), s.scale)
    s.check(matrix_cores=True)


def test_decode_of_scores_that_are_no_numbers(ops):
    """A key that is not finite gives NaNs to the rows that see it and to no other."""
    s = Step(torch.bfloat16, 4, 2, 64, 16, [(1, 40), (1, 300), (1, 33)], 0, seed=1)
    s.kc.view(torch.uint8)[s.table[1][2], 1, 5, 7] = 0xff
    s.device()
    ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, 3, s.scale)
    got = torch.isnan(s.out[:3]).view(3, 2, 2 * 64)
    assert got[1, 1].all() and not got[1, 0].any() and not got[0].any() and not got[2].any()


PREFILLS = [  # Hq, Hkv, D, page size, window
    (8, 2, 64, 16, 0), (8, 2, 128, 16, 0), (6, 2, 96, 32, 0), (5, 1, 32, 64, 0), (4, 4, 128, 128, 0), (8, 2, 64, 16, 100),
    (8, 2, 128, 16, 1), (6, 2, 96, 16, 33), (2, 2, 64, 1024, 130),
]
PREFILL_SEQS = [(1, 1), (1, 90), (1, 0), (2, 2), (5, 5), (64, 64), (65, 65), (3, 128), (70, 203), (128, 128), (17, 33), (200, 431)]


@pytest.mark.parametrize("rows,groups", [(64, 0), (64, 3), (128, 0), (128, 2)])
@pytest.mark.parametrize("Hq,Hkv,D,P,window", PREFILLS)
def test_prefill(ops, Hq, Hkv, D, P, window, rows, groups):
    s = Step(torch.bfloat16, Hq, Hkv, D, P, PREFILL_SEQS, window, seed=Hq + D, spread=1.5).device()
    ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(rows), s.scale, window, rows, groups)
    s.check(matrix_cores=True)


@pytest.mark.parametrize("rows,groups", [(64, 0), (64, 2), (128, 0), (128, 2)])
@pytest.mark.parametrize("Hq,Hkv,D,P,window", [(8, 2, 64, 16, 0), (4, 2, 128, 32, 0), (3, 1, 96, 16, 40), (4, 4, 32, 64, 0), (4, 2, 128, 16, 70)])
def test_prefill_of_numbers_that_are_none(ops, Hq, Hkv, D, P, window, rows, groups):
    """A value that is a NaN is one in its column for the rows that see its key, a key that is one in all columns; other rows of the
    block, before it or with a window that has passed it, are what they are without it."""
    s = Step(torch.bfloat16, Hq, Hkv, D, P, [(70, 203), (1, 40), (200, 431), (64, 64), (5, 1500)], window, seed=D, spread=1.5)
    last = Hkv - 1
    for seq, key, head, d in [(0, 150, 0, 0), (0, 202, last, D - 1), (2, 231, last, 17), (2, 300, 0, 31), (2, 430, 0, 3), (3, 1, last, 5),
                              (3, 40, 0, 16), (4, 1497, last, 30)]:
        s.vc.view(torch.uint8)[s.table[seq][key // P], head, key % P, d] = 0xff if d % 2 else 0x7f
        s.v[s.table[seq][key // P], head, key % P, d] = math.nan
    s.kc.view(torch.uint8)[s.table[3][50 // P], last, 50 % P, 9] = 0x7f
    s.k[s.table[3][50 // P], last, 50 % P, 9] = math.nan
    s.device()
    ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(rows), s.scale, window, rows, groups)
    want = plain_f8.attention(s.q[:s.q_start[-1]], s.k, s.v, s.q_start, s.ctx, s.table, s.scale, window)[0]
    nan, got = torch.isnan(want), s.out[:s.q_start[-1]].cpu()
    assert nan.any() and not nan.all() and torch.equal(torch.isnan(got), nan)
    # (the other numbers: against the same without the NaNs, whose rows and columns are left out)
    for x in (s.k, s.v):
        x.nan_to_num_(0.0)
    s.out[:s.q_start[-1]] = torch.where(nan, plain_f8.attention(s.q[:s.q_start[-1]], s.k, s.v, s.q_start, s.ctx, s.table, s.scale,
                                                                 window)[0].to(got.dtype), got).cuda()
    s.check(matrix_cores=True)


@pytest.mark.parametrize("rows", [64, 128])
def test_prefill_behind_decoding_sequences_with_a_sink(ops, rows):
    s = Step(torch.bfloat16, 8, 4, 64, 16, [(1, 40), (1, 700), (33, 90), (150, 150)], 0, seed=7).device()
    sink = torch.tensor([-3.0, 0.0, 2.5, 40.0, 1.0, -60.0, 5.0, 3.0], device="cuda")
    ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(rows, 2), s.scale, 0, rows, 0, sink)
    s.out[0, :] = s.out[1, :] = 77.0             # (the list's empty item names the first sequence)
    s.check(sink, first=2, matrix_cores=True)


@pytest.mark.parametrize("dtype,Hkv,D,P", [(torch.float32, 1, 10, 3), (torch.bfloat16, 3, 34, 1), (torch.float32, 1, 12, 5), (torch.bfloat16, 1, 2, 1),
                                           (torch.float32, 1, 20, 7)])
def test_layers_of_a_pool_of_odd_pages(ops, dtype, Hkv, D, P):
    """Layers that begin at a multiple of 2 or 4 bytes: stored, grown and read as in a cache of their own."""
    layers, pages, n = 3, 7, 5 * P + 1
    g = torch.Generator().manual_seed(D)
    codes = torch.zeros(2, layers, pages, Hkv, P, D, device="cuda", dtype=torch.uint8).view(F8)
    scales = torch.zeros(2, layers, pages, Hkv, device="cuda")
    table = torch.randperm(pages, generator=g).tolist()
    slots = torch.tensor([table[i // P] * P + i % P for i in range(n)], dtype=torch.int32)
    pos = torch.arange(n, dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    for layer in range(layers):
        alone = [torch.zeros(pages, Hkv, P, D, device="cuda", dtype=torch.uint8).view(F8) for _ in range(2)] + [
            torch.zeros(pages, Hkv, device="cuda") for _ in range(2)]
        pooled = [codes[0, layer], codes[1, layer], scales[0, layer], scales[1, layer]]
        x = (torch.randn(n, 4 * Hkv, D, generator=g) * torch.exp(2 * torch.randn(n, 1, 1, generator=g))).to(dtype).cuda()
        outs = []
        for cache in (alone, pooled):
            for a, b in ((0, 2 * P + 1), (2 * P + 1, n)):              # (the second call begins inside of a page)
                q = ops.rope_store_f8(x[a:b, :2 * Hkv], x[a:b, 2 * Hkv:3 * Hkv], x[a:b, 3 * Hkv:], pos[a:b].cuda(), None,
                                      slots[a:b].cuda(), *cache)
            out = torch.empty_like(q)
            ops.attention_generic_f8(out, q, *cache, i32([0, b - a]), i32([n]), i32([table]), i32([0] * -(-(b - a) // 16)),
                                     i32(list(range(0, b - a, 16))), D ** -0.5)
            outs.append(out)
        assert torch.equal(outs[0], outs[1]) and not torch.isnan(outs[0]).any()
        for a, b in zip(alone, pooled):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---- copies ----------------------------------------------------------------------------------------
POOLS = [[(3, 20, (2, 16, 64), torch.bfloat16)], [(2, 9, (3, 5, 7), torch.float32), (2, 9, (3,), torch.float32)],
         [(4, 600, (2, 16, 32), F8), (4, 600, (2, 16, 32), F8), (4, 600, (2,), torch.float32), (4, 600, (2,), torch.float32)],
         [(1, 2, (1,), torch.uint8)], [(5, 700, (13,), torch.uint8), (1, 700, (8, 16, 128), torch.bfloat16)]]


@pytest.mark.parametrize("pools", POOLS, ids=range(len(POOLS)))
@pytest.mark.parametrize("n", [0, 1, 5, 256, 300])
def test_copies(ops, pools, n):
    g = torch.Generator().manual_seed(n)
    pages = pools[0][1]
    n = min(n, pages // 2)
    made = [torch.randint(0, 256, (layers, p) + shape + (torch.empty((), dtype=dt).element_size(),), generator=g, dtype=torch.uint8)
            for layers, p, shape, dt in pools]
    order = torch.randperm(pages, generator=g).tolist()
    dst, src = order[:n], [order[n + i // 2] for i in range(n)]
    raw = [m.cuda() for m in made]
    ops.copy_pages([r.view(dt).view(r.shape[:-1]) for r, (_, _, _, dt) in zip(raw, pools)], src, dst)
    for r, m in zip(raw, made):
        m[:, dst] = m[:, src]
        assert torch.equal(r.cpu(), m)
