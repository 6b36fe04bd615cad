"""The operators of the 8-bit cache as programs use them: one behind the other, recorded and replayed, on other streams, over caches whose
offsets pass 32 bits; and what they refuse."""
import pytest
import torch

import plain_f8
from test_cache_f8_gpu import F8, Step

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from pytriton_llama_amd import ops
    return ops


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def empty_cache(layers, pages, Hkv, P, D):
    shape = (layers, pages, Hkv, P, D)
    return [torch.zeros(shape, device="cuda", dtype=torch.uint8).view(F8) for _ in range(2)] + [
        torch.zeros(shape[:3], device="cuda") for _ in range(2)]


class Decoding:
    """Two layers' decode steps of a batch whose inputs change from step to step in place."""

    def __init__(self, ops, n=3, Hq=8, Hkv=2, D=64, P=16, width=40):
        self.ops, self.n, self.D, self.Hkv, self.P, self.width = ops, n, D, Hkv, P, width
        g = torch.Generator().manual_seed(3)
        self.pools = empty_cache(2, n * width + 1, Hkv, P, D)
        self.table = i32(torch.randperm(n * width, generator=g).view(n, width).tolist())
        self.x = torch.zeros((n, (Hq + 2 * Hkv) * D), device="cuda", dtype=torch.bfloat16)
        q, k, v = self.x.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        self.qkv = q.view(n, Hq, D), k.view(n, Hkv, D), v.view(n, Hkv, D)
        self.positions, self.slots, self.ctx = i32([0] * n), i32([-1] * n), i32([0] * n)
        self.q_start = i32(range(n + 1))
        self.inv_freq = (10000.0 ** (-torch.arange(0, D, 2) / D)).cuda()
        self.out = torch.zeros((2, n, Hq, D), device="cuda", dtype=torch.bfloat16)
        self.tickets = torch.zeros(4 * n * Hkv, dtype=torch.int32, device="cuda")

    def feed(self, contexts, seed):
        """The next step: sequence i has contexts[i] tokens with its new one (0: a place of the batch that is not used)."""
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.x.shape, generator=g).to(self.x.dtype))
        table = self.table.cpu()
        self.positions.copy_(i32([max(c - 1, 0) for c in contexts]))
        self.slots.copy_(i32([int(table[i, (c - 1) // self.P]) * self.P + (c - 1) % self.P if c else -1 for i, c in enumerate(contexts)]))
        self.ctx.copy_(i32(contexts))

    def step(self):
        for layer in range(2):
            cache = [p[layer] for p in self.pools]
            q = self.ops.rope_store_f8(*self.qkv, self.positions, self.inv_freq, self.slots, *cache)
            self.ops.attention_decode_f8(self.out[layer], q, *cache, self.q_start, self.ctx, self.table, self.n, self.D ** -0.5,
                                         tickets=self.tickets)


def bits(tensors):
    return [t.view(torch.uint8).clone() if t.dtype == F8 else t.clone() for t in tensors]


def test_recorded_steps_of_two_graphs_that_share_tickets(ops):
    """Steps by two recorded graphs in turn, eager work of the same tickets between them, against the same steps one by one. Contexts go
    from lengths that are not cut to lengths that are, places of the batch are left and taken again."""
    eager, replayed = Decoding(ops), Decoding(ops)
    for d in (eager, replayed):
        d.feed([0, 0, 0], 0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            d.step()
        torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            replayed.step()
        graphs.append(g)
    for turn, contexts in enumerate([[1, 1, 1], [2, 17, 16], [0, 18, 640], [3, 0, 601], [4, 530, 602], [639, 531, 0], [640, 532, 1], [1, 1, 1]]):
        for d in (eager, replayed):
            d.feed(contexts, turn)
        eager.step()
        if turn == 5:
            replayed.step()
        graphs[turn % 2].replay()
        if turn % 3 == 0:
            graphs[turn % 2].replay()                        # (the same once more changes nothing)
        torch.cuda.synchronize()
        assert torch.equal(eager.out, replayed.out)
        for a, b in zip(bits(eager.pools), bits(replayed.pools)):
            assert torch.equal(a, b)
        assert not replayed.tickets.any()


@pytest.mark.parametrize("rows", [64, 128])
def test_recorded_prompt_portions(ops, rows):
    """A recorded call over tables that change: the blocks are cut by the contexts that it is replayed with."""
    steps = [Step(torch.bfloat16, 4, 2, 64, 16, [(90, c), (30, 2100 - c)], 0, seed=c) for c in (90, 600, 1500, 2070)]
    width = max(len(s.table[0]) for s in steps)
    for s in steps:
        s.table = [t + [-1] * (width - len(t)) for t in s.table]
        s.device()
        s.work = s.blocks(rows)
    pages = max(s.kc.shape[0] for s in steps)
    q, out = torch.empty_like(steps[0].qd), torch.empty_like(steps[0].out)
    cache = [torch.zeros((pages, *t.shape[1:]), device="cuda", dtype=torch.uint8 if t.dtype == F8 else t.dtype) for t in steps[0].cache]
    cache = [t.view(F8) if t.dtype == torch.uint8 else t for t in cache]
    tables, work = [torch.empty_like(t) for t in steps[0].tables], steps[0].work

    def feed(s):
        q.copy_(s.qd)
        out.fill_(77.0)
        for to, t in zip(cache, s.cache):
            if t.dtype == F8:
                to.view(torch.uint8)[:t.shape[0]].copy_(t.view(torch.uint8))
            else:
                to[:t.shape[0]].copy_(t)
        for to, t in zip(tables, s.tables):
            to.copy_(t)

    def call(tickets=None):
        ops.attention_prefill_f8(out, q, *cache, *tables, *work, steps[0].scale, 0, rows, 0, tickets=tickets)

    tickets = torch.zeros(4 * work[0].numel() * 4, dtype=torch.int32, device="cuda")
    feed(steps[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        call(tickets)
    with torch.cuda.graph(graphs[1]):
        call()                                               # (tickets of its own, made in the graph)
    for turn, s in enumerate(steps + steps[::-1]):
        for graph in graphs:
            feed(s)
            graph.replay()
            s.out = out
            s.check(matrix_cores=True)
        assert not tickets.any()
        feed(s)
        call(tickets)
        s.out = out
        s.check(matrix_cores=True)


@pytest.mark.parametrize("Hq,Hkv,D,window", [(16, 8, 64, 0), (16, 8, 128, 0), (16, 8, 96, 100), (16, 8, 32, 0)])
@pytest.mark.parametrize("n", [31, 33, 64, 66])
def test_decode_with_workgroups_of_four_and_of_eight_waves(ops, Hq, Hkv, D, window, n):
    """Around the numbers of pairs where the launch changes from one to the other (256 and 512 on a GPU of 256 compute units), with
    contexts around the ends of both's turns and one that is cut."""
    contexts = [(0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 257, 511, 513)[i % 13] for i in range(n - 1)] + [1500]
    s = Step(torch.bfloat16, Hq, Hkv, D, 16, [(1, c) for c in contexts], window, seed=n + D, spread=2.0).device()
    tickets = torch.zeros(4 * n * Hkv, dtype=torch.int32, device="cuda")
    for _ in range(2):
        s.out.fill_(77.0)
        ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, n, s.scale, window, tickets=tickets)
        s.check(matrix_cores=True)
        assert not tickets.any()


def test_recorded_copies_keep_their_pages(ops):
    """What a recorded copy copies was said when it was recorded; a recorded store of many rows takes its slots from where they are."""
    g = torch.Generator().manual_seed(0)
    pools = [torch.randint(0, 256, (2, 600, 3, 5), generator=g, dtype=torch.uint8).cuda(), torch.randn(2, 600, 16, generator=g).cuda()]
    src, dst = list(range(300)), list(range(599, 299, -1))
    q = torch.randn(200, 6, 64, generator=g).to(torch.bfloat16).cuda()
    cache = [p[0] for p in empty_cache(1, 40, 2, 16, 64)]
    slots, positions, inv_freq = i32(range(200)), i32(range(200)), torch.ones(32, device="cuda") / 7
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.copy_pages(pools, src[:1], dst[:1])
        ops.rope_store_f8(q[:, :2], q[:, 2:4], q[:, 4:], positions, inv_freq, slots, *cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.copy_pages(pools, src, dst)
        turned = ops.rope_store_f8(q[:, :2], q[:, 2:4], q[:, 4:], positions, inv_freq, slots, *cache)
    src[:], dst[:] = [5] * 300, [7] * 300
    for turn in range(4):
        for p in pools:
            p[:, :300].copy_(torch.randint(0, 256, p[:, :300].shape, generator=g).to(p.dtype))
        q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
        slots.copy_(i32([16 * turn + i + turn for i in range(200)]))
        want = [p.clone() for p in pools]
        for w in want:
            w[:, list(range(599, 299, -1))] = w[:, :300]
        own = [t.view(torch.uint8).clone().view(F8) if t.dtype == F8 else t.clone() for t in cache]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(pools, want))
        assert torch.equal(ops.rope_store_f8(q[:, :2], q[:, 2:4], q[:, 4:], positions, inv_freq, slots, *own), turned)
        assert all(torch.equal(a, b) for a, b in zip(bits(cache), bits(own)))


CUTS = [[(64, 5000)], [(1, 3000), (63, 2999), (65, 1100)], [(200, 3000)], [(64, 64), (64, 900), (17, 1500), (3, 385), (5, 384)]]


@pytest.mark.parametrize("D,P,window", [(64, 16, 0), (128, 32, 0), (96, 16, 700), (32, 16, 0)])
@pytest.mark.parametrize("seqs", CUTS, ids=range(len(CUTS)))
def test_few_blocks_are_cut_along_their_keys(ops, seqs, D, P, window):
    s = Step(torch.bfloat16, 4, 2, D, P, seqs, window, seed=len(seqs) + D, spread=2.0).device()
    work = s.blocks(64)
    tickets = torch.zeros(4 * work[0].numel() * 4, dtype=torch.int32, device="cuda")
    for _ in range(2):
        s.out.fill_(77.0)
        ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *work, s.scale, window, tickets=tickets)
        s.check(matrix_cores=True)
        assert not tickets.any()


@pytest.mark.parametrize("D,window", [(64, 0), (128, 0), (96, 900), (32, 0)])
@pytest.mark.parametrize("seqs", CUTS + [[(300, 2000), (129, 1400), (1, 3), (2, 2)]], ids=range(len(CUTS) + 1))
def test_few_blocks_of_128_rows_are_cut_along_their_keys(ops, seqs, D, window):
    s = Step(torch.bfloat16, 4, 2, D, 16, seqs, window, seed=len(seqs) + D, spread=2.0).device()
    work = s.blocks(128)
    tickets = torch.zeros(4 * work[0].numel() * 4, dtype=torch.int32, device="cuda")
    for _ in range(2):
        s.out.fill_(77.0)
        ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *work, s.scale, window, 128, tickets=tickets)
        s.check(matrix_cores=True)
        assert not tickets.any()


@pytest.mark.parametrize("rows", [64, 128])
@pytest.mark.parametrize("heads", [16, 32])
def test_blocks_share_few_workgroups(ops, heads, rows):
    """So many heads that the workgroups of one are few: each has ends of blocks and several blocks, short ones and one without
    keys among them."""
    seqs = [(30, 900), (200, 1000), (1, 0), (1, 1300), (65, 65), (1, 1)]
    s = Step(torch.bfloat16, heads, 1, 32, 16, seqs, 0, seed=heads, spread=2.0).device()
    work = s.blocks(rows)
    assert 2 * work[0].numel() <= ops.compute_units(s.qd.device) * 3 // heads
    ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *work, s.scale, 0, rows)
    s.check(matrix_cores=True)


def test_rows_without_keys_and_without_a_sink_of_their_own(ops):
    """A sink of -inf is no sink: rows without keys are zeros, the others what they are without."""
    s = Step(torch.bfloat16, 4, 2, 64, 16, [(1, 0), (1, 40), (1, 0)], 0, seed=3).device()
    sink = torch.full((4,), float("-inf"), device="cuda")
    for call in ("decode", "prefill", "generic"):
        s.out.fill_(77.0)
        if call == "decode":
            ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, 3, s.scale, 0, sink)
        elif call == "prefill":
            ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(64), s.scale, 0, 64, 0, sink)
        else:
            ops.attention_generic_f8(s.out, s.qd, *s.cache, *s.tables, *s.blocks(16), s.scale, 0, sink)
        s.check(matrix_cores=True)


def test_calls_on_two_streams_at_once(ops):
    """Each with tickets of its own."""
    seqs = [(1, c) for c in (3000, 1, 700, 129)]
    steps = [Step(torch.bfloat16, 8, 2, 64, 16, seqs, 0, seed=i).device() for i in range(2)]
    long = [Step(torch.bfloat16, 8, 2, 64, 16, [(100, 2000)], 0, seed=i).device() for i in range(2)]
    blocks = [s.blocks(64) for s in long]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, l, b, stream in zip(steps, long, blocks, streams):
            with torch.cuda.stream(stream):
                ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, len(seqs), s.scale)
                ops.attention_prefill_f8(l.out, l.qd, *l.cache, *l.tables, *b, l.scale)
    torch.cuda.synchronize()
    for s in steps + long:
        s.check(matrix_cores=True)


def test_pages_that_sequences_share(ops):
    """Two sequences read the pages of the first one's beginning; what each stores behind it goes to a page of its own, of which one is a
    copy."""
    Hq, Hkv, D, P = 4, 2, 64, 16
    pools = empty_cache(1, 8, Hkv, P, D)
    cache = [p[0] for p in pools]
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(40 + 2, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()

    def parts(x):
        q, k, v = x.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        return q.view(-1, Hq, D), k.view(-1, Hkv, D), v.view(-1, Hkv, D)

    ops.rope_store_f8(*parts(rows[:40]), i32(range(40)), None, i32([5 * P + i for i in range(16)] + [2 * P + i for i in range(16)]
                                                              + [7 * P + i for i in range(8)]), *cache)
    ops.copy_pages(pools, [7], [1])
    assert all(torch.equal(p[0, 7].view(torch.uint8), p[0, 1].view(torch.uint8)) if p.dtype == F8 else torch.equal(p[0, 7], p[0, 1])
               for p in pools)
    q = ops.rope_store_f8(*parts(rows[40:]), i32([40, 40]), None, i32([7 * P + 8, P + 8]), *cache)
    out = torch.empty_like(q)
    ops.attention_decode_f8(out, q, *cache, i32([0, 1, 2]), i32([41, 41]), i32([[5, 2, 7], [5, 2, 1]]), 2, D ** -0.5)
    for i in range(2):
        alone = empty_cache(1, 3, Hkv, P, D)
        alone = [p[0] for p in alone]
        ops.rope_store_f8(*parts(rows[:40]), i32(range(40)), None, i32(range(40)), *alone)
        qi = ops.rope_store_f8(*parts(rows[40 + i:41 + i]), i32([40]), None, i32([40]), *alone)
        oi = torch.empty_like(qi)
        ops.attention_decode_f8(oi, qi, *alone, i32([0, 1]), i32([41]), i32([[0, 1, 2]]), 1, D ** -0.5)
        assert torch.equal(out[i], oi[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D,P", [(4, 2, 64, 16), (8, 8, 128, 16), (3, 3, 64, 16), (2, 1, 96, 16), (4, 2, 34, 7), (6, 2, 128, 32), (2, 1, 64, 64)])
@pytest.mark.parametrize("lengths", [[129], [1, 1, 200, 1], [700, 1, 1, 1598], [1] * 150 + [2000]], ids=["129", "203", "2300", "2150"])
def test_a_call_of_many_rows_stores_what_calls_of_a_page_store(ops, dtype, Hq, Hkv, D, P, lengths):
    """Sequences that begin inside of pages, some rows that are not stored among them: one call, and a call for every page."""
    g = torch.Generator().manual_seed(D + len(lengths))
    slots, pages, pieces = [], 0, []
    order = torch.randperm(sum(n // P + 2 for n in lengths), generator=g).tolist()
    for i, n in enumerate(lengths):
        off = (5 * i) % P if n > 1 else 3 % P                # (what lies before: an earlier step's)
        at = 0
        while at < n:
            take = min(P - off, n - at)
            pieces.append((len(slots), take))
            slots += [order[pages] * P + off + j for j in range(take)]
            pages, at, off = pages + 1, at + take, 0
        slots += [-1] * (i % 3)
    T, total = len(slots), len(order)
    x = (torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * torch.exp(2 * torch.randn(T, 1, generator=g))).to(dtype).cuda()
    q, k, v = (x[:, a * D:b * D].view(T, b - a, D) for a, b in ((0, Hq), (Hq, Hq + Hkv), (Hq + Hkv, Hq + 2 * Hkv)))
    positions, sd = i32([(7 * t) % 4001 for t in range(T)]), i32(slots)
    inv_freq = (500000.0 ** (-torch.arange(0, D, 2) / D)).cuda()
    codes = torch.randint(0, 127, (2, total, Hkv, P, D), generator=g, dtype=torch.uint8)
    scales = 2.0 ** torch.randint(-9, 3, (2, total, Hkv), generator=g)
    caches = [[codes[0].cuda().view(F8), codes[1].cuda().view(F8), scales[0].cuda(), scales[1].cuda()] for _ in range(2)]
    for _ in range(2):
        got = ops.rope_store_f8(q, k, v, positions, inv_freq, sd, *caches[0])
    want = torch.empty_like(got)
    for first, n in pieces:
        s = slice(first, first + n)
        want[s] = ops.rope_store_f8(q[s], k[s], v[s], positions[s], inv_freq, sd[s], *caches[1])
    stored = (sd >= 0).cpu()
    assert torch.equal(got.cpu()[stored], want.cpu()[stored])
    for a, b in zip(bits(caches[0]), bits(caches[1])):
        assert torch.equal(a, b)


def test_offsets_that_pass_32_bits(ops):
    """Pools of 4.5 GiB, of which the last pages are used."""
    Hq, Hkv, D, P = 8, 8, 128, 16
    pages = 9 * 2 ** 29 // (Hkv * P * D)
    s = Step(torch.bfloat16, Hq, Hkv, D, P, [(1, 100), (1, 333), (40, 90)], 0, seed=4)
    used = s.kc.shape[0]
    first = pages - used
    far = [torch.zeros((1, pages, Hkv, P, D), device="cuda", dtype=torch.uint8) for _ in range(2)] + [
        torch.zeros((1, pages, Hkv), device="cuda") for _ in range(2)]
    for to, t in zip(far, (s.kc, s.vc, s.ks, s.vs)):
        to[0, first:].copy_((t.view(torch.uint8) if t.dtype == F8 else t).cuda())
    far = [t.view(F8) if t.dtype == torch.uint8 else t for t in far]
    s.table = [[p + first if p >= 0 else p for p in row] for row in s.table]
    s.device()
    s.table = [[p - first if p >= 0 else p for p in row] for row in s.table]       # (the plain form reads the used pages by themselves)
    cache = [t[0] for t in far]
    for call in ("decode", "prefill 64", "prefill 128", "generic"):
        s.out.fill_(77.0)
        if call == "decode":
            ops.attention_decode_f8(s.out, s.qd, *cache, *s.tables, 2, s.scale)
            s.check(last=2, matrix_cores=True)
            continue
        if call == "generic":
            ops.attention_generic_f8(s.out, s.qd, *cache, *s.tables, *s.blocks(16), s.scale)
        else:
            rows = int(call.split()[1])
            ops.attention_prefill_f8(s.out, s.qd, *cache, *s.tables, *s.blocks(rows), s.scale, 0, rows)
        s.check(matrix_cores=True)
    # a store into the last page, and a copy of it
    g = torch.Generator().manual_seed(9)
    x = torch.randn(P, Hkv, D, generator=g).to(torch.bfloat16)
    last = pages - 1
    ops.rope_store_f8(x.cuda(), x.cuda(), x.cuda(), i32(range(P)), None, i32([last * P + i for i in range(P)]), *cache)
    codes, scales = plain_f8.quantised(x.float().transpose(0, 1)[None])
    assert torch.equal(cache[0][last].cpu().view(torch.uint8), codes[0].view(torch.uint8))
    assert torch.equal(cache[3][last].cpu(), scales[0])
    ops.copy_pages(far, [last, last], [last - 1, 0])
    for p in (last - 1, 0):
        assert torch.equal(cache[1][p].cpu().view(torch.uint8), codes[0].view(torch.uint8))
        assert torch.equal(cache[2][p].cpu(), scales[0])


def test_what_the_operators_refuse(ops):
    from pytriton_llama_amd.ops import KernelError
    s = Step(torch.bfloat16, 4, 2, 64, 16, [(1, 20), (3, 40)], 0, seed=0).device()
    k, v, ks, vs = s.cache
    q_start, ctx, table = s.tables
    work = s.blocks(64)
    before = s.out.clone()

    def attention(which, *more, out=s.out, q=s.qd, cache=s.cache, tables=s.tables, **named):
        first = {"decode": (1,), "prefill": work, "generic": work}[which]
        getattr(ops, f"attention_{which}_f8")(out, q, *cache, *tables, *first, s.scale, *more, **named)

    float_cache = [k.view(torch.uint8), v, ks, vs]
    for which in ("decode", "prefill", "generic"):
        wrong = [
            dict(cache=float_cache), dict(cache=[k[:, :1], v, ks, vs]), dict(cache=[k, v[1:], ks, vs]), dict(cache=[k, v, ks[:, :1], vs]),
            dict(cache=[k, v, ks.double(), vs]), dict(cache=[k.transpose(0, 1), v.transpose(0, 1), ks, vs]),
            dict(cache=[k, v.cpu(), ks, vs]), dict(tables=(q_start, ctx, table.long())), dict(tables=(q_start, ctx.cpu(), table)),
            dict(tables=(q_start[:-1], ctx, table)), dict(tables=(q_start, ctx, table[:1])), dict(tables=(q_start, ctx, table[0])),
            dict(q=s.qd[:, :3]), dict(q=s.qd.float()), dict(out=s.out.half()), dict(q=s.qd.transpose(0, 1)), dict(window=-1),
            dict(sink=torch.zeros(3, device="cuda")), dict(sink=torch.zeros(4, device="cuda", dtype=torch.bfloat16)),
        ]
        for named in wrong:
            with pytest.raises(KernelError):
                attention(which, **named)
    odd = Step(torch.bfloat16, 4, 2, 64, 24, [(1, 20)], 0, seed=0).device()      # (pages of 24 rows: not for the matrix cores)
    assert not ops.attention_f8_fits(torch.bfloat16, 4, 2, 64, 24)
    with pytest.raises(KernelError):
        ops.attention_decode_f8(odd.out, odd.qd, *odd.cache, *odd.tables, 1, odd.scale)
    with pytest.raises(KernelError):
        ops.attention_prefill_f8(odd.out, odd.qd, *odd.cache, *odd.tables, *odd.blocks(64), odd.scale)
    with pytest.raises(KernelError):                          # more sequences than the tables have
        ops.attention_decode_f8(s.out, s.qd, *s.cache, *s.tables, 3, s.scale)
    with pytest.raises(KernelError):                          # more sequences than queries
        ops.attention_decode_f8(s.out[:1], s.qd[:1], *s.cache, *s.tables, 2, s.scale)
    with pytest.raises(KernelError):
        attention("decode", tickets=torch.zeros(64, device="cuda"))
    with pytest.raises(KernelError):
        attention("prefill", block_rows=32)
    with pytest.raises(KernelError):
        ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, *work, 0.0)
    with pytest.raises(KernelError):
        ops.attention_prefill_f8(s.out, s.qd, *s.cache, *s.tables, work[0], work[1][:1], s.scale)
    assert torch.equal(s.out, before)

    x = torch.zeros((3, 8 * 64), device="cuda", dtype=torch.bfloat16)
    q, kk, vv = x.split([256, 128, 128], dim=1)
    q, kk, vv = q.view(3, 4, 64), kk.view(3, 2, 64), vv.view(3, 2, 64)
    inv, slots, positions = torch.ones(32, device="cuda"), i32([0, 1, 2]), i32([0, 1, 2])
    held = bits(s.cache)
    for args in [(q, kk, vv[:2], positions, inv, slots), (q, kk, vv.float(), positions, inv, slots), (q, kk.contiguous(), vv, positions, inv, slots),
                 (q, kk, vv, positions[:2], inv, slots), (q, kk, vv, positions.long(), inv, slots), (q, kk, vv, positions, inv[:3], slots),
                 (q, kk, vv, positions, inv.double(), slots), (q, kk, vv, positions, inv, slots[:1]), (q, kk, vv, positions, inv, slots.cpu()),
                 (q.half(), kk.half(), vv.half(), positions, inv, slots), (q[..., ::2], kk[..., ::2], vv[..., ::2], positions, inv, slots)]:
        with pytest.raises(KernelError):
            ops.rope_store_f8(*args, *s.cache)
    many = torch.zeros((17, 8, 64), device="cuda", dtype=torch.bfloat16)
    lacking = ops.RowScale(torch.ones((17, 4), device="cuda"), 256, 1e-5)
    with pytest.raises(KernelError):
        ops.rope_store_f8(many[:, :4], many[:, 4:6], many[:, 6:], i32(range(17)), inv, None, *s.cache, row_scale=lacking)
    with pytest.raises(KernelError):                          # the factor of other rows
        ops.rope_store_f8(q, kk, vv, positions, inv, slots, *s.cache, row_scale=lacking)
    for a, b in zip(held, bits(s.cache)):
        assert torch.equal(a, b)

    pool = torch.arange(24, device="cuda").view(1, 6, 4)
    for pools, src, dst in [([pool], [0, 1], [2]), ([pool], [0], [6]), ([pool], [-1], [0]), ([pool], [0, 1], [2, 2]), ([pool], [0, 1], [1, 2]),
                            ([pool], [3], [3]), ([pool.transpose(1, 2)], [0], [1]), ([pool.cpu()], [0], [1]), ([pool] * 17, [0], [1])]:
        with pytest.raises(KernelError):
            ops.copy_pages(pools, src, dst)
    assert torch.equal(pool.flatten().cpu(), torch.arange(24))
