"""paged_attention over values that are no finite numbers: rows that do not see them have the result of 64 bits within the bound of any other, and so do columns beside
them in the same 16 bytes, whose own values are large: one that was lost with its neighbour would show."""
import pytest
import torch

import paged_ref as ref
from paged_ref import TYPES, Batch
from test_paged_cache import caches
from test_paged_tiles import LARGE, TILES, name, resolved
from test_paged_weights import bound

NAN, INF = float("nan"), float("inf")


class Poisoned:
    def __init__(self, dev, new, held, group, d, page, dtype, mx, window=0, heads=2):
        b = self.b = Batch(new, held, page, seed=sum(held) + d, rows=sum(new) + 2)
        self.dev, self.d, self.dtype, self.mx, self.window, self.group = dev, d, dtype, mx, window, group
        self.q = b.normal(b.rows, heads * group, d).to(TYPES[dtype])
        table = b.table.long()
        place = lambda s, p: (int(table[s, p // page]), p % page)
        kx, vx = b.normal(b.pages, page, heads, d), b.normal(b.pages, page, heads, d)
        # (sequence, position, column, width, kind) of what the last head's values hold
        self.events = []
        for s, (n, h) in enumerate(zip(new, held)):
            if n == 0:
                continue
            for i, kind in enumerate([NAN] if mx else [NAN, INF, -INF]):
                p = h - max(1, n // 3) + i
                if p < h:
                    self.events.append((s, p, 3, 1, kind))
            for p in range(max(0, h - n - (window or 0)), h, 29):      # all along what the rows see the ends of
                self.events.append((s, p, 11, 1, NAN if mx or p % 2 else INF))
            if mx:
                self.events.append((s, h - (n + 1) // 2, 32, 32, NAN))
        for s, p, col, width, _ in self.events:
            vx[place(s, p)][-1, col & ~7:(col & ~7) + 8] = 50.0
        self.k, self.v, self.scales = caches(b, heads, d, dtype, mx, dev)
        real = []
        for cache, scales, x in ((self.k, "k_scales", kx), (self.v, "v_scales", vx)):
            x = x.to(TYPES[dtype])
            if mx:
                data, byte = ref.quantized(x)
                cache.copy_(data)
                self.scales[scales].copy_(byte)
                real.append(ref.values(data, byte))
            else:
                cache.copy_(x)
                real.append(x.double())
        for s, p, col, width, kind in self.events:
            at, r = place(s, p)
            if width == 32:
                self.scales["v_scales"][at, r, -1, col // 32] = 255
            else:
                self.v[at, r, -1, col] = 0x7F if mx else kind
        for s, h in enumerate(held):                                    # behind the context, on its last page
            for r in range((h - 1) % page + 1, page) if h else ():
                at = int(table[s, (h - 1) // page])
                if mx:
                    self.scales["v_scales"][at, r], self.scales["k_scales"][at, r] = 255, 255
                else:
                    self.v[at, r], self.k[at, r] = NAN, INF
        self.parts = ref.attention(b, self.q, *real, float(torch.tensor(d ** -0.5, dtype=torch.float32)), window)
        self.tol = bound(self.q.dtype, self.parts, d, max(held))
        self.want = self.parts[0].clone()
        for row, s, p, _, _ in b.places():
            for s2, p2, col, width, kind in self.events:
                if s2 == s and p2 <= p and (not window or p2 > p - window):
                    self.want[row, -group:, col:col + width] += kind

    def check(self, ct, rows=None, **kw):
        q = self.q.to(self.dev)
        out = torch.full_like(q, 9.0)
        ct.paged_attention(q, self.k, self.v, *self.b.where(self.dev), ct.partition(out, [1, 1, self.d]), self.d ** -0.5, window=self.window, **self.scales,
                           variant=None if rows is None else name(self.dtype, self.mx, self.d, rows), **kw)
        assert rows is None or resolved(ct)[1] == rows
        n = sum(self.b.new)
        got, want = out.cpu().double()[:n], self.want[:n]
        same = torch.where(want.isfinite(), (got - want).abs() <= self.tol[:n], (got == want) | (got.isnan() & want.isnan()))
        assert bool(same.all()), (rows, int((~same).sum()), (~same).nonzero()[0].tolist(), got[~same][0].item(), want[~same][0].item())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("group,window", [(1, 0), (1, 1), (2, 60), (2, 333), (5, 0)])
def test_gpu_finite_values_beside_others_in_every_tile(ct, dev, dtype, d, mx, page, group, window):
    p = Poisoned(dev, [300, 0, 77, 3], [300, 50, 900, 400], group, d, page, dtype, mx, window)
    for rows in TILES[d]:
        p.check(ct, rows)
        p.check(ct, rows, max_new=300, max_context=900)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("new,held,group,window", [([1, 1, 1], [1, 300, 95], 4, 0), ([1, 1], [700, 40], 2, 33), ([8, 3, 0, 5], [8, 300, 20, 700], 4, 0), ([8, 3, 5], [90, 300, 700], 2, 20), ([30], [3000], 1, 700)])
def test_gpu_finite_values_beside_others_in_small_tiles(ct, dev, dtype, d, mx, new, held, group, window):
    p = Poisoned(dev, new, held, group, d, 16, dtype, mx, window)
    p.check(ct)
    p.check(ct, max_new=max(new), max_context=max(held))
