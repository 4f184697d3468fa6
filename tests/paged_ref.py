"""A batch of sequences on the pages of a cache, and what the paged kernels make of it, in 64 bits on the CPU."""
import math

import torch

import block_ref as ref

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


class Batch:
    """Sequences of ``new`` new tokens and ``held`` tokens in all on pages dealt at random; ``rows`` >= sum(new) rows of tokens."""

    def __init__(self, new, held, page, seed=0, rows=None, spare=3, table_pages=None):
        self.new, self.held, self.page = list(new), list(held), page
        g = torch.Generator().manual_seed(seed)
        counts = [-(-max(h, 0) // page) for h in held]
        self.pages = sum(counts) + spare
        order = torch.randperm(self.pages, generator=g).int()
        self.table = torch.full((len(new), table_pages or max(1, max(counts))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.starts = torch.tensor([0] + list(torch.tensor(list(new)).cumsum(0)), dtype=torch.int32)
        self.lens = torch.tensor(self.held, dtype=torch.int32)
        self.rows = rows or max(1, sum(new))
        self.g = g

    def where(self, dev):
        return self.table.to(dev), self.starts.to(dev), self.lens.to(dev)

    def places(self):
        """(row, sequence, position, page or -1, row on the page) of every token"""
        out, first = [], 0
        for b, (n, h) in enumerate(zip(self.new, self.held)):
            for i in range(n):
                p = h - n + i
                page = int(self.table[b, p // self.page]) if 0 <= p < self.table.shape[1] * self.page else -1
                out.append((first + i, b, p, page if 0 <= page < self.pages else -1, p % self.page))
            first += n
        return out

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g) * std


def quantized(x):
    """16-bit rows -> (e4m3 bytes, e8m0 bytes): the rounding that the header defines, in 64 bits"""
    v = x.double().unflatten(-1, (-1, 32))
    most = v.abs().amax(-1)
    lost = ~torch.isfinite(v).all(-1)
    byte = torch.where(most == 0, 0, (torch.frexp(torch.where(lost, 1.0, most)).exponent - 1 - 8 + 127).clamp(0, 254))
    code = ref.nearest(v / torch.exp2(byte.double() - 127).unsqueeze(-1), ref.grid_of("mxfp8")) | (torch.signbit(v).long() << 7)
    code[lost] = 0
    byte[lost] = 255
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def values(data, scales):
    """the f64 values of mxfp8 bytes"""
    v = data.view(torch.float8_e4m3fn).double().unflatten(-1, (-1, 32))
    return (v * ref.scale_values(scales, "mxfp8").unsqueeze(-1)).flatten(-2)


def attention(batch, q, k, v, scale, window=0):
    """out, and what its error may be as a fraction of 2^-24: (out, weighted |v|, |v| summed, largest |score products|, keys) a row; k and v are f64 caches"""
    heads, group = k.shape[2], q.shape[1] // k.shape[2]
    out, near, far = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(3))
    reach = torch.zeros(q.shape[:2], dtype=torch.float64)
    first = 0
    for b, (n, h) in enumerate(zip(batch.new, batch.held)):
        seen = min(max(h, 0), batch.table.shape[1] * batch.page)
        p = torch.arange(seen)
        pages = batch.table[b].long()[p // batch.page] if seen else p
        there = (pages >= 0) & (pages < batch.pages)
        kb = k[pages.clamp(0, batch.pages - 1), p % batch.page] * there[:, None, None] if seen else k[:0, 0]
        vb = torch.where(there[:, None, None], v[pages.clamp(0, batch.pages - 1), p % batch.page], torch.zeros(())) if seen else v[:0, 0]
        for i in range(n):
            at = h - n + i
            lo, hi = max(0, at - window + 1) if window else 0, min(at + 1, seen)
            if hi <= lo:
                continue
            for g in range(heads):
                qq = q[first + i, g * group:(g + 1) * group].double()
                kk, vv = kb[lo:hi, g], vb[lo:hi, g]
                w = torch.softmax(qq @ kk.t() * scale, -1)
                rows = slice(g * group, (g + 1) * group)
                out[first + i, rows] = w @ vv
                near[first + i, rows] = w @ vv.abs()
                far[first + i, rows] = vv.abs().sum(0)
                reach[first + i, rows] = (qq.abs() @ kk.abs().t()).amax(-1) * abs(scale)
        first += n
    return out, near, far, reach


def bound(got_type, parts, d, keys):
    """How far an output may be off.  With u = half a step in the type (relative, 2^-11 f16, 2^-8 bf16): the output is rounded once, u |o|; the
    weights are rounded to the type, u of each; f32 scores of d products are off by (d + 2) 2^-24 of their magnitudes, which moves a weight by as much twice (its
    exponential and the sum), the exponential itself and the sums by 2^-22 + (keys / 16 + 64) 2^-24; an f16 weight below 2^-14 of the largest is off by 2^-25 of it."""
    out, near, far, reach = parts
    u = 2.0 ** -11 if got_type == torch.float16 else 2.0 ** -8
    slip = 2 * reach * (d + 2) * 2.0 ** -24 + 2.0 ** -21 + (keys / 16 + 64) * 2.0 ** -24
    tol = u * out.abs() + (u + slip).unsqueeze(-1) * near * (1 + u)
    return tol + (2.0 ** -25 * far + 2.0 ** -25 if got_type == torch.float16 else 1e-38)
