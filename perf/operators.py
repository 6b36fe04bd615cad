"""The operators of the cache that is held in 8 bits, and of its pages, as cases that can be timed and compared.

A page holds ``page`` tokens of every kv head. A block is the part of a page that belongs to one kv head; the keys of a block
share one scale, a power of two, and so do its values: what is held is e4m3(x / scale). Four kinds of case:

store    the new tokens of a step: rotation of queries and keys, keys and values into their pages.
decode   attention of requests that bring one token each.
prefill  attention of portions of prompts, each behind what its request has in the cache.
copy     copies of pages, all layers, as when requests branch.

Sizes are those of the repository's own benchmark (Llama-3.2-1B: 32 heads of 64 on 8; Llama-3.1-8B: 32 heads of 128 on 8) at
its batches and contexts. Where ``own`` is false the operators are computed by elementary torch operations.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
E4M3_MAX = 448.0
LEAST_EXPONENT = -126          # scales stay normal float32 numbers


# ---- the cases ---------------------------------------------------------------------------------
def listed():
    small = {"heads": 32, "kv_heads": 8, "dim": 64, "page": 16, "dtype": "bfloat16"}
    large = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bfloat16"}
    return [
        # the headline batch takes a step: eight tokens, each into a page that is partly filled
        {"name": "store_decode_b8", "kind": "store", **small, "batch": 8, "shortest": 2048, "longest": 2090, "portion": 0, "prefix": 0},
        # continuous batching on the large model, a step of 2,048 tokens: a portion that begins and ends inside pages beside
        # twenty requests that decode
        {"name": "store_mixed_8b", "kind": "store", **large, "batch": 20, "shortest": 130, "longest": 2900, "portion": 2028, "prefix": 1021},
        # one user's chat: few keys, where the launch counts
        {"name": "decode_chat", "kind": "decode", **small, "batch": 1, "shortest": 45, "longest": 45, "window": 0},
        # the headline: eight requests behind 2,048-token prompts
        {"name": "decode_b8", "kind": "decode", **small, "batch": 8, "shortest": 2048, "longest": 2090, "window": 0},
        # a full server: 64 requests at all stages of their generations
        {"name": "decode_b64_ragged", "kind": "decode", **small, "batch": 64, "shortest": 61, "longest": 2610, "window": 0},
        # long documents on the large model
        {"name": "decode_8b_long", "kind": "decode", **large, "batch": 8, "shortest": 5000, "longest": 7000, "window": 0},
        # two requests at the end of the large model's positions: the cache that 8 bits make room for
        {"name": "decode_8b_128k", "kind": "decode", **large, "batch": 2, "shortest": 120001, "longest": 131000, "window": 0},
        # a batch of short prompts, as the reference's own benchmark sends it
        {"name": "prefill_8_short", "kind": "prefill", **small, "batch": 8, "shortest": 10, "longest": 60, "prefix": 0, "window": 0},
        # the headline's prompt
        {"name": "prefill_2048", "kind": "prefill", **small, "batch": 1, "shortest": 2048, "longest": 2048, "prefix": 0, "window": 0},
        # a portion of a long prompt on the large model, behind the portions before it
        {"name": "prefill_8b_portion", "kind": "prefill", **large, "batch": 1, "shortest": 1531, "longest": 1531, "prefix": 6145, "window": 0},
        # sixteen requests of the large model branch into five each: the last page of each, four times, in 32 layers (in the
        # engine's type; the pages of a cache in 8 bits are half as large)
        {"name": "copy_8b_fork", "kind": "copy", **large, "layers": 32, "pages": 64, "pool": 256},
        # (one request in two: a page a layer)
        {"name": "copy_1b_fork", "kind": "copy", **small, "layers": 16, "pages": 1, "pool": 64},
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of these ranges: 1 to 16 kv heads with 1 to 8 heads each, head sizes of 64 and 128 and now and then 96, pages
    of 16 to 64 tokens; now and then float32."""
    kind = rng.choice(["store", "decode", "decode", "prefill", "copy"])
    dim = rng.choice([64, 64, 128, 128, 96])
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    case = {"kind": kind, "kv_heads": kv, "heads": kv * rng.choice([1, 2, 4, 4, 5, 8]), "dim": dim,
            "page": rng.choice([16, 16, 32, 64]), "dtype": "float32" if rng.random() < 0.15 else "bfloat16"}
    if kind == "store":
        batch = rng.choice([0, rng.randint(1, 64)])
        portion = 0 if batch and rng.random() < 0.4 else _log_between(rng, 2, 2048)
        longest = _log_between(rng, 1, 8000)
        return {**case, "batch": batch, "shortest": _log_between(rng, 1, longest), "longest": longest, "portion": portion,
                "prefix": rng.choice([0, rng.randint(1, 6000)])}
    if kind == "decode":
        batch = _log_between(rng, 1, 64)
        # (keys in all: at most half a million with 8 kv heads of 64, four times that for one request)
        longest = _log_between(rng, 1, max(16, min(100000, 4000000 // (batch * kv * dim // 64))))
        if case["dtype"] == "float32":
            longest = min(longest, 4000)
        return {**case, "batch": batch, "shortest": _log_between(rng, 1, longest), "longest": longest,
                "window": _log_between(rng, 1, longest) if rng.random() < 0.15 else 0}
    if kind == "prefill":
        batch = rng.choice([1, 1, rng.randint(2, 8)])
        if case["dtype"] == "float32":
            longest, prefix = _log_between(rng, 2, 200), rng.choice([0, rng.randint(1, 700)])
        else:
            longest, prefix = _log_between(rng, 2, 1600 if batch == 1 else 400), rng.choice([0, rng.randint(1, 4000 // batch)])
        while longest > 2 and 4.0 * case["heads"] * dim * batch * longest * (prefix + longest / 2) > 1.6e11:
            longest, prefix = longest // 2, prefix // 2
        return {**case, "batch": batch, "shortest": rng.randint(1, longest), "longest": longest, "prefix": prefix,
                "window": _log_between(rng, 1, longest + prefix) if rng.random() < 0.15 else 0}
    layers = rng.randint(1, 32)
    pages = _log_between(rng, 1, max(1, min(400, (1 << 29) // (layers * kv * case["page"] * dim * 4))))
    return {**case, "layers": layers, "pages": pages, "pool": 2 * pages + rng.randint(1, 50)}


def _lengths(case):
    """``batch`` lengths from the shortest to the longest, evenly spread, in an order that is neither rising nor falling."""
    n, a, b = case["batch"], case["shortest"], case["longest"]
    spread = [a + (b - a) * i // max(1, n - 1) for i in range(n)]
    return sorted(spread, key=lambda x: (x * 2654435761) % 4294967291)


def _sequences(case):
    """(rows, keys) of every sequence of a step: those that bring one token first."""
    if case["kind"] == "store":
        return [(1, n) for n in _lengths(case)] + ([(case["portion"], case["prefix"] + case["portion"])] if case["portion"] else [])
    if case["kind"] == "decode":
        return [(1, n) for n in _lengths(case)]
    return sorted(((n, case["prefix"] + n) for n in _lengths(case)), key=lambda s: s[0] != 1)


def _seen(rows, keys, window):
    """Pairs of a row and a key that it sees."""
    firsts = range(keys - rows + 1, keys + 1)
    return sum(min(k, window) if window else k for k in firsts)


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    Hq, Hkv, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "copy":
        return {"bytes": 2.0 * 2 * case["layers"] * case["pages"] * Hkv * P * D * size, "flops": 0.0}
    seqs = _sequences(case)
    T = sum(r for r, _ in seqs)
    if case["kind"] == "store":
        # queries read and written, keys and values read in the engine's type and written in 8 bits, the blocks' scales
        blocks = sum((k - 1) // P - (k - r) // P + 1 for r, k in seqs) * Hkv * 2
        return {"bytes": T * (2 * Hq * D * size + 2 * Hkv * D * (size + 1)) + 8.0 * blocks + 8 * T, "flops": 4.0 * T * (Hq + 2 * Hkv) * D}
    w = case["window"]
    keys = sum(min(k, r + w - 1) if w else k for r, k in seqs)
    pairs = sum(_seen(r, k, w) for r, k in seqs)
    return {"bytes": 2.0 * T * Hq * D * size + keys * Hkv * (2.0 * D + 8.0 / P) + 4.0 * keys / P, "flops": 4.0 * pairs * Hq * D}


# ---- what a program has in hand ------------------------------------------------------------------
class _State:
    pass


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _power_of_two_scale(largest):
    """The smallest 2^e, e >= -126, with largest <= 448 * 2^e."""
    m, e = torch.frexp(largest)                            # largest = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=LEAST_EXPONENT)
    e = torch.where(largest > 0, e, torch.full_like(e, LEAST_EXPONENT))
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)       # (2^e by its bits: pow is not exact on every device)


def _cache(g, pages, case):
    """Pages of 8-bit numbers as keys or values leave them there, and their scales: normal, with channels of their own size."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn(shape, generator=g, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn(case["kv_heads"], 1, case["dim"], generator=g, device=DEVICE))
    scale = _power_of_two_scale(x.abs().amax((2, 3)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def _tables(s, case, g):
    """The tables of a step: where each sequence's rows and keys lie. Pages come in no order."""
    P = case["page"]
    s.seqs = _sequences(case)
    held = [-(-k // P) for _, k in s.seqs]
    s.n, s.T, s.pages = len(s.seqs), sum(r for r, _ in s.seqs), sum(held)
    order = torch.randperm(s.pages, generator=g, device=DEVICE).tolist()
    table, starts, at = [[0] * max(held) for _ in held], [0], 0
    for i, n in enumerate(held):
        table[i][:n] = order[at:at + n]
        at += n
        starts.append(starts[-1] + s.seqs[i][0])
    s.table_host = table
    s.q_start, s.ctx_len, s.block_table = _int32(starts), _int32([k for _, k in s.seqs]), _int32(table)
    s.longest_q, s.longest_k = max(r for r, _ in s.seqs), max(k for _, k in s.seqs)


def _blocks_of_rows(seqs, first, rows):
    """(sequence, first row) of every block of so many rows of the sequences from ``first`` on, the ones with most keys first."""
    items = [(-(k - r + min(o + rows, r)), i, o) for i, (r, k) in enumerate(seqs) if i >= first for o in range(0, r, rows)]
    items.sort(key=lambda x: x[0])
    return _int32([i for _, i, _ in items]), _int32([o for _, _, o in items])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    Hq, Hkv, D, P = case["heads"], case["kv_heads"], case["dim"], case["page"]
    s = _State()
    s.case, s.dtype = case, dtype
    if case["kind"] == "copy":
        shape = (case["layers"], case["pool"], Hkv, P, D)
        s.k = torch.randn(shape, generator=g, device=DEVICE).to(dtype)
        s.v = torch.randn(shape, generator=g, device=DEVICE).to(dtype)
        order = torch.randperm(case["pool"], generator=g, device=DEVICE).tolist()
        n = case["pages"]
        s.dst, s.src = order[:n], [order[n + i // 4] for i in range(n)]          # (a page is copied up to four times)
        s.dst_index, s.src_index = _int32(s.dst).long(), _int32(s.src).long()
        return s
    _tables(s, case, g)
    if case["kind"] == "store":
        qkv = torch.randn(s.T, (Hq + 2 * Hkv) * D, generator=g, device=DEVICE)
        qkv *= torch.exp(0.5 * torch.randn((Hq + 2 * Hkv) * D, generator=g, device=DEVICE))
        qkv = qkv.to(dtype)
        s.q = qkv[:, :Hq * D].view(s.T, Hq, D)
        s.k = qkv[:, Hq * D:(Hq + Hkv) * D].view(s.T, Hkv, D)
        s.v = qkv[:, (Hq + Hkv) * D:].view(s.T, Hkv, D)
        s.inv_freq = 500000.0 ** (-torch.arange(0, D, 2, device=DEVICE, dtype=torch.float32) / D)
        # the pool: the pages that the step writes (the earlier ones of its requests are not touched), in no order
        written = [(i, p) for i, (r, k) in enumerate(s.seqs) for p in range((k - r) // P, (k - 1) // P + 1)]
        order = torch.randperm(len(written), generator=g, device=DEVICE).tolist()
        place = dict(zip(written, order))
        positions = [p for r, k in s.seqs for p in range(k - r, k)]
        of_token = [place[i, p // P] for i, (r, k) in enumerate(s.seqs) for p in range(k - r, k)]
        s.positions, s.slots = _int32(positions), _int32([p * P + x % P for p, x in zip(of_token, positions)])
        s.page_of, s.row_of = _int32(of_token).long(), _int32([x % P for x in positions]).long()
        # pages that begin anew with this step: its first token for them is theirs
        begun = [False] * len(order)
        for (i, p), at in place.items():
            begun[at] = p * P >= s.seqs[i][1] - s.seqs[i][0]
        s.begun = torch.tensor(begun, device=DEVICE)
        both = [_cache(g, len(order), case) for _ in range(2)]
        # what the requests have in these pages: nothing behind their tokens
        filled = [0] * len(order)
        for (i, p), at in place.items():
            filled[at] = max(0, min(P, s.seqs[i][1] - s.seqs[i][0] - p * P))
        keep = torch.arange(P, device=DEVICE)[None, None, :, None] < _int32(filled)[:, None, None, None]
        s.codes = torch.stack([torch.where(keep, c.float(), 0.0).to(torch.float8_e4m3fn) for c, _ in both])
        s.scales = torch.stack([x for _, x in both])
        return s
    s.q = (1.5 * torch.randn(s.T, Hq, D, generator=g, device=DEVICE)).to(dtype)
    s.scale = D ** -0.5
    s.k, s.k_scale = _cache(g, s.pages, case)
    s.v, s.v_scale = _cache(g, s.pages, case)
    # which sequence, and which of its rows, every row of the step is; and the other way round
    s.seq_of = torch.tensor([i for i, (r, _) in enumerate(s.seqs) for _ in range(r)], device=DEVICE)
    s.place_of = torch.tensor([o for r, _ in s.seqs for o in range(r)], device=DEVICE)
    s.rows = (s.q_start[:-1, None].long() + torch.arange(s.longest_q, device=DEVICE)).clamp(max=s.T - 1)
    # the lists that a step brings for the kernels, and the counters that its launches share
    s.decodes = sum(r == 1 for r, _ in s.seqs) if case["kind"] == "decode" else 0
    s.blocks_16 = _blocks_of_rows(s.seqs, 0, 16)
    s.blocks_64, s.blocks_128 = _blocks_of_rows(s.seqs, s.decodes, 64), _blocks_of_rows(s.seqs, s.decodes, 128)
    s.tickets = torch.zeros(4 * s.n * Hkv, dtype=torch.int32, device=DEVICE)
    return s


# ---- one pass ------------------------------------------------------------------------------------
def _values(codes, scale):
    """The numbers that 8-bit blocks [..., kv heads, page, D] stand for."""
    return codes.float() * scale[..., None, None]


def _rotated(x, angles):
    """Pairs (j, j + D/2) of every head, float32."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, n = angles.cos().float()[:, None], angles.sin().float()[:, None]
    return torch.cat([a * c - b * n, b * c + a * n], -1)


def _store_plain(s):
    angles = (s.positions.float()[:, None] * s.inv_freq).double()      # (the framework's angle is this float32 product)
    q = _rotated(s.q, angles).to(s.dtype)
    new = torch.stack([_rotated(s.k, angles), s.v.float()])            # [2, T, Hkv, D]
    Hkv, D = new.shape[2:]
    pages = s.codes.shape[1]
    largest = torch.zeros(2, pages, Hkv, device=DEVICE).scatter_reduce(
        1, s.page_of[None, :, None].expand(2, -1, Hkv), new.abs().amax(-1), "amax")
    had = torch.where(s.begun[None, :, None], torch.zeros_like(s.scales), s.scales)
    scale = torch.maximum(_power_of_two_scale(largest), had)
    held = torch.where(s.begun[None, :, None, None, None], torch.zeros_like(s.codes, dtype=torch.float32), _values(s.codes, s.scales))
    held[:, s.page_of, :, s.row_of] = new.transpose(0, 1)
    s.codes.copy_((held / scale[..., None, None]).to(torch.float8_e4m3fn))
    s.scales.copy_(scale)
    return q


def _attention_plain(s):
    case = s.case
    Hq, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    table = s.block_table.long()
    gathered = [_values(c.view(torch.uint8)[table].view(torch.float8_e4m3fn), x[table]).transpose(2, 3).flatten(1, 2)
                for c, x in ((s.k, s.k_scale), (s.v, s.v_scale))]      # [n, keys, Hkv, D]
    k, v = (x.transpose(1, 2) for x in gathered)
    q = s.q[s.rows].float().view(s.n, s.longest_q, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).flatten(2, 3)    # [n, Hkv, G rows, D]
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    rows = (s.q_start[1:] - s.q_start[:-1])[:, None]
    at = (s.ctx_len[:, None] - rows + torch.arange(s.longest_q, device=DEVICE))[:, :, None]
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = (key <= at) & (key < s.ctx_len[:, None, None])
    seen &= key > at - (case["window"] or (1 << 30))
    scores = scores.view(s.n, Hkv, Hq // Hkv, s.longest_q, -1).masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p.flatten(2, 3), v.contiguous()).view(s.n, Hq, s.longest_q, D)
    return out[s.seq_of, :, s.place_of].to(s.dtype)


def _attention_own(s):
    from pytriton_llama_amd import ops
    case = s.case
    out = torch.empty_like(s.q)
    cache = (s.k, s.v, s.k_scale, s.v_scale)
    if not ops.attention_f8_fits(s.dtype, case["heads"], case["kv_heads"], case["dim"], case["page"]):
        ops.attention_generic_f8(out, s.q, *cache, s.q_start, s.ctx_len, s.block_table, *s.blocks_16, s.scale, case["window"])
    elif case["kind"] == "decode":
        ops.attention_decode_f8(out, s.q, *cache, s.q_start, s.ctx_len, s.block_table, s.n, s.scale, case["window"],
                                tickets=s.tickets)
    else:
        keys = min(s.longest_k, case["window"]) if case["window"] else s.longest_k
        rows, groups = ops.attention_prefill_f8_plan(s.q.device, case["heads"], case["dim"], s.blocks_64[0].numel(),
                                                     s.blocks_128[0].numel(), keys)
        ops.attention_prefill_f8(out, s.q, *cache, s.q_start, s.ctx_len, s.block_table,
                                 *(s.blocks_128 if rows == 128 else s.blocks_64), s.scale, case["window"], rows, groups)
    return out


def run(s):
    if s.case["kind"] == "copy":
        if own:
            from pytriton_llama_amd import ops
            ops.copy_pages((s.k, s.v), s.src, s.dst)
        else:
            s.k[:, s.dst_index] = s.k[:, s.src_index]
            s.v[:, s.dst_index] = s.v[:, s.src_index]
        return {"k": s.k, "v": s.v}
    if s.case["kind"] == "store":
        if own:
            from pytriton_llama_amd import ops
            q = ops.rope_store_f8(s.q, s.k, s.v, s.positions, s.inv_freq, s.slots, s.codes[0], s.codes[1], s.scales[0], s.scales[1])
        else:
            q = _store_plain(s)
        # what the pages now stand for (four significant bits and a power of two: bfloat16 holds it as it is)
        return {"q": q, "held": s.codes.to(torch.bfloat16) * s.scales.to(torch.bfloat16)[..., None, None]}
    return {"out": _attention_own(s) if own else _attention_plain(s)}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------
def _power_of_two(exponent):
    """2^exponent in float64, for whole exponents, by its bits."""
    return ((exponent.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exponent(x):
    """floor(log2 x) of positive normal float64 numbers."""
    return ((x.view(torch.int64) >> 52) & 2047) - 1023


def _to_e4m3(x):
    """The nearest e4m3 number (ties to the even one) of float64 numbers of at most 448."""
    step = _power_of_two(_exponent(x.abs().clamp(min=2.0 ** -6)) - 3)
    return torch.round(x / step) * step


def _exact_store(s):
    D, P = s.case["dim"], s.case["page"]
    half = D // 2
    angle = (s.positions.float()[:, None] * s.inv_freq[None]).double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
        return torch.cat([z.real, z.imag], -1)
    held = []
    for codes, scales, x in ((s.codes[0], s.scales[0], turned(s.k)), (s.codes[1], s.scales[1], s.v.double())):
        value, factor = codes.double(), scales.double()
        value[s.begun] = 0.0
        factor[s.begun] = 0.0
        # a block's largest new number, token by token of a page
        largest = torch.zeros_like(factor)
        for row in range(P):
            here = s.row_of == row
            largest[s.page_of[here]] = torch.maximum(largest[s.page_of[here]], x[here].abs().amax(-1))
        ratio = (largest / E4M3_MAX).clamp(min=2.0 ** LEAST_EXPONENT)
        need = _power_of_two(_exponent(ratio))
        need = torch.where(need < ratio, 2 * need, need)
        factor_new = torch.maximum(factor, need)
        value = _to_e4m3(value * (factor / factor_new)[..., None, None])
        value[s.page_of, :, s.row_of] = _to_e4m3(x / factor_new[s.page_of][..., None])
        held.append(value * factor_new[..., None, None])
    return {"q": turned(s.q), "held": torch.stack(held)}


def _exact_attention(s):
    Hkv, G, D, P, w = s.case["kv_heads"], s.case["heads"] // s.case["kv_heads"], s.case["dim"], s.case["page"], s.case["window"]
    outs, at = [], 0
    for i, (r, n) in enumerate(s.seqs):
        pages = s.block_table[i, :-(-n // P)].long()
        k, v = ((c.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double() * x[pages].double()[:, :, None, None])
                .permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :n] for c, x in ((s.k, s.k_scale), (s.v, s.v_scale)))
        position = torch.arange(n - r, n, device=DEVICE)[:, None]
        key = torch.arange(n, device=DEVICE)[None]
        hidden = (key > position) | ((position - key >= w) if w else False)
        heads = []
        for h in range(Hkv * G):
            score = s.q[at:at + r, h].double() @ k[h // G].T * s.scale
            weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            heads.append(weight @ v[h // G])
        outs.append(torch.stack(heads, 1))
        at += r
    return {"out": torch.cat(outs)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        k, v = s.k.double(), s.v.double()
        for pool in (k, v):
            for a, b in zip(s.src, s.dst):
                pool[:, b] = pool[:, a]
        return {"k": k, "v": v}
    return _exact_store(s) if case["kind"] == "store" else _exact_attention(s)
