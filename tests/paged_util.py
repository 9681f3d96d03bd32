"""A paged cache with random contents and the 64-bit definitions of the operators over portions of sequences (append, read, prompt attention, attention behind
a shared prefix), for their tests.  fp16 rounds by at most half a step: H = 2^-11 relative."""
import math

import torch

PAGE, D = 64, 128
H = 2.0 ** -11
F64, HALF = torch.float64, torch.float16
BASE = 500000.0


class Cache:
    """K and V pools of `pages` pages and the address table of sequences that hold `lens` positions.  The first `shared` pages of all sequences are the same.
    Every slot that no sequence holds has NaN for a scale and a zero, so a result that one of them reaches is no number."""

    def __init__(self, lens, hkv, bits, dev, shared=0, seed=0, extra_blocks=0):
        g = torch.Generator().manual_seed(seed)
        self.hkv, self.bits, self.lens, self.dev = hkv, bits, list(lens), dev
        B = len(lens)
        self.blocks = max(shared, max((-(-n // PAGE) for n in lens), default=1), 1) + extra_blocks
        n = shared + B * (self.blocks - shared)
        place = torch.randperm(n, generator=g)
        self.pages = torch.cat([place[:shared].expand(B, shared), place[shared:].view(B, self.blocks - shared)], 1).contiguous()
        self.cut = hkv * PAGE * D * bits // 8
        self.pools = []
        for _ in range(2):
            p = torch.randint(0, 256, (n, self.cut + hkv * PAGE * 4), dtype=torch.uint8, generator=g)
            top = 2 ** bits - 1
            meta = p[:, self.cut:].view(HALF).view(n, 2, hkv, PAGE)
            held = torch.zeros(n, PAGE, dtype=torch.bool)
            for b, length in enumerate(lens):
                for j in range(self.blocks):
                    held[self.pages[b, j], :max(0, min(PAGE, length - j * PAGE))] = True
            held[place[:shared]] = True
            meta[:, 0] = ((torch.rand(n, hkv, PAGE, generator=g) * 3 + 1) / top).half().masked_fill(~held[:, None], float("nan"))
            meta[:, 1] = ((torch.rand(n, hkv, PAGE, generator=g) * 0.4 + 0.3) * top).half().masked_fill(~held[:, None], float("nan"))
            self.pools.append(p.to(dev))
        self.pages = self.pages.to(dev)
        self.table = torch.stack([p.data_ptr() + self.pages * p.shape[1] for p in self.pools], 1).contiguous()
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.size = hkv * D * bits // 8
        self.args = (PAGE, self.size, bits == 4, True)

    def meta(self, which):
        return self.pools[which][:, self.cut:].view(HALF).view(-1, 2, self.hkv, PAGE)

    def codes(self, which):
        c = self.pools[which][:, :self.cut].view(-1, self.hkv, PAGE, D * self.bits // 8)
        return torch.stack([c & 15, c >> 4], -1).flatten(-2) if self.bits == 4 else c

    def values(self, which, b, n):
        """Positions 0 .. n - 1 of sequence b: [n, hkv, D] in 64 bits."""
        t = torch.arange(n, device=self.dev)
        page, slot = self.pages[b][t // PAGE], t % PAGE
        u = self.codes(which)[page, :, slot].to(F64)
        s, z = (self.meta(which)[page, i, :, slot].to(F64)[..., None] for i in (0, 1))
        return u * s + (-s * z).half().to(F64) if self.bits == 4 else s * (u - z)


def rotated(x, pos):
    """x [T, heads, D] at positions pos [T], in 64 bits."""
    angle = pos.to(F64)[:, None] * BASE ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=F64) / D)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.to(F64).chunk(2, -1)
    return torch.cat([c * a - s * b, c * b + s * a], -1)


def attention64(q, k, v, limit, scale):
    """q [n, hq, D], k / v [L, hkv, D], row i sees positions <= limit[i].  Returns the result, sum w |v| and sqrt(sum w^2 v^2) per number, and the largest
    sum |q k| of a row with a key that it sees."""
    n, hq, _ = q.shape
    if k.shape[0] == 0:
        zero = torch.zeros(n, hq, D, dtype=F64, device=q.device)
        return zero, zero, zero, zero[..., 0]
    k, v = (x.repeat_interleave(hq // x.shape[1], 1) for x in (k, v))
    seen = torch.arange(k.shape[0], device=q.device)[None] <= limit[:, None]
    s = torch.einsum("nhd,lhd->nhl", q.to(F64), k) * scale
    s = s.masked_fill(~seen[:, None], -math.inf)
    some = seen.any(1)[:, None, None]
    w = torch.where(some, torch.softmax(s, -1), 0.0)
    mass = torch.einsum("nhd,lhd->nhl", q.to(F64).abs(), k.abs()).masked_fill(~seen[:, None], 0.0).amax(-1)
    return (torch.einsum("nhl,lhd->nhd", w, v), torch.einsum("nhl,lhd->nhd", w, v.abs()), torch.einsum("nhl,lhd->nhd", w * w, v * v).sqrt(), mass)


def check_attention(out, want, scale):
    """Roundings to fp16 of the kernels' operands, each by at most H relative: every key (its score is off by at most d = H scale sum |q k|, its weight by 2 d with
    the denominator's), every weight (and the sum), every value (the weight times the scale, in the kernel that applies scales to weights; its product with codes
    up to three times the value's spread), the result.  A number is off by no more than all of them at their worst.  They are independent, so the rows
    together are off by about H / sqrt(3) of sqrt(sum w^2 v^2) for each of key, weight and value (the products with codes: 2.7 times), of the result, and of
    the results of the splits of a long axis (sqrt(sum of their squares) is that of w^2 v^2 again): 2 H in all, and no more than 4 H.  At their worst the splits add
    H sum w |v|, which is in the 6 H (2 for the weight and the sum, 1 for the value, 1 for a split; 3 in the tail kernel, which has no splits)."""
    o, absolute, spread, mass = want
    off = (out.to(F64) - o).abs()
    d = H * scale * mass[..., None]
    assert torch.isfinite(out).all()
    worst = H * o.abs() + absolute * (H * 6 + 2 * d * (1 + 2 * d)) + 2.0 ** -24
    assert (off <= worst).all(), float((off / worst).max())
    assert float(off.norm()) <= 4 * H * float((spread + o.abs()).norm()) + 1e-9 * off.numel() ** 0.5, float(off.norm() / (spread + o.abs()).norm()) / H
