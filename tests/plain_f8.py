"""Plain forms, in float64 on the CPU, of a cache that is held in 8 bits: the store into its pages and attention over them."""
import math

import torch

F8 = torch.float8_e4m3fn


def nearest(x):
    """The nearest e4m3 number of every float64 number of at most 448, ties to the even one."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(x), e - 4)
    return torch.round(x / step) * step


def scale_for(largest: float) -> float:
    e = -126
    while largest > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x, positions, inv_freq):
    """x [T, heads, D] by the angles positions * inv_freq, which are float32 products."""
    if inv_freq is None:
        return x.double()
    half = x.shape[-1] // 2
    angle = (positions.float()[:, None] * inv_freq.float()).double()[:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


class Blocks:
    """Keys or values: float64 numbers [pages, Hkv, page_size, D] and scales [pages, Hkv]."""

    def __init__(self, codes, scale):
        self.scale = scale.double().clone()
        self.held = codes.float().double() * self.scale[:, :, None, None]

    def store(self, x, slots):
        """x float64 [T, Hkv, D]; slots list."""
        P = self.held.shape[2]
        t = 0
        while t < len(slots):
            if slots[t] < 0 or slots[t] >= self.held.shape[0] * P:
                t += 1
                continue
            n = 1
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % P:
                n += 1
            page, off = divmod(slots[t], P)
            for h in range(x.shape[1]):
                new = x[t:t + n, h]
                fine = new[torch.isfinite(new)].abs()
                need = scale_for(float(fine.max()) if fine.numel() else 0.0)
                if off == 0:
                    self.held[page, h] = 0.0
                    self.scale[page, h] = need
                elif need > self.scale[page, h]:
                    self.scale[page, h] = need
                    self.held[page, h] = nearest(self.held[page, h] / need) * need
                s = float(self.scale[page, h])
                got = nearest(new.nan_to_num(0, 0, 0) / s) * s
                self.held[page, h, off:off + n] = torch.where(torch.isfinite(new), got, torch.full_like(got, math.nan))
            t += n


def quantised(x):
    """(codes, scales) of x float [pages, Hkv, page_size, D]."""
    largest = x.abs().amax((2, 3))
    scale = torch.tensor([[scale_for(float(v)) for v in row] for row in largest], dtype=torch.float32)
    return (x / scale[:, :, None, None]).to(F8), scale


def attention(q, k, v, q_start, ctx_len, table, scale, window=0, sink=None):
    """(result, sum of weight * |v|, bound of |sum of |q k|| * scale) for every row, float64. k, v: float64
    [pages, Hkv, page_size, D]; table: lists of page numbers."""
    T, Hq, D = q.shape
    Hkv, P = k.shape[1:3]
    G = Hq // Hkv
    out, size, score_size = torch.zeros(T, Hq, D).double(), torch.zeros(T, Hq, D).double(), torch.zeros(T, Hq, 1).double()
    for i, ctx in enumerate(ctx_len):
        rows = q_start[i + 1] - q_start[i]
        for r in range(rows):
            pos = ctx - rows + r
            lo = max(0, pos - window + 1) if window else 0
            if pos < lo or ctx == 0:
                continue
            keys = torch.arange(lo, pos + 1)
            pages = torch.tensor([table[i][j // P] for j in keys.tolist()])
            kk, vv = k[pages, :, keys % P], v[pages, :, keys % P]              # [n, Hkv, D]
            t = q_start[i] + r
            x = q[t].double().view(Hkv, G, D)
            s = torch.einsum("hgd,nhd->hgn", x, kk) * scale
            top = s.amax(-1, keepdim=True)
            if sink is not None:
                top = torch.maximum(top, sink.double().view(Hkv, G, 1))
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            if sink is not None:
                total = total + torch.exp(sink.double().view(Hkv, G, 1) - top)
            w = p / total
            out[t] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(Hq, D)
            size[t] = torch.einsum("hgn,nhd->hgd", w, vv.abs()).reshape(Hq, D)
            score_size[t] = (torch.einsum("hgd,nhd->hgn", x.abs(), kk.abs()) * scale).amax(-1).reshape(Hq, 1)
    return out, size, score_size
