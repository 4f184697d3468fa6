"""paged_attention in tiles of every number of rows that its launcher chooses from, and what the launcher chooses."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import paged_ref as ref
from paged_ref import TYPES, Batch
from test_host_abi import _last
from test_paged_attention import attend, problem
from test_paged_cache import args
from test_paged_weights import bound, one_key_above_many

TILES = {64: (32, 64, 128, 256), 128: (32, 64, 128, 256), 256: (32, 64, 128)}
LARGE = [(d, mx) for d in TILES for mx in (False, True)]


def name(dtype, mx, d, rows=None):
    return f"{dtype}{'_mxfp8' if mx else ''}_d{d}" + ("" if rows is None else f"_rows{rows}")


def resolved(ct):
    """(variant, rows of a tile) of the last launch"""
    fn, info = C.c_char_p(), ct.KernelInfo()
    ct.check(ct.lib().cutile_last_resolved_kernel(C.byref(fn), C.byref(info)))
    assert fn.value == b"paged_attention"
    return info.variant.decode(), info.tile[0]


# ---- without a GPU --------------------------------------------------------------------------------------------------------
CHOICES = [  # (KV heads, group, D, sequences, new tokens of each, context): rows of a tile, workgroups to a tile
    ((8, 4, 128, 1, 8192, 8192), (256, 1)),
    ((8, 4, 128, 1, 512, 16896), (256, 4)),
    ((8, 4, 128, 1, 2048, 16896), (256, 1)),
    ((8, 4, 64, 1, 8192, 8192), (256, 1)),
    ((8, 4, 256, 1, 8192, 8192), (128, 1)),
    ((2, 2, 128, 1, 150, 6000), (32, 12)),
    ((8, 8, 128, 1, 84, 335), (32, 2)),
    ((1, 1, 64, 1, 300, 300), (32, 2)),
    ((8, 1, 128, 1, 512, 16960), (128, 8)),
    ((2, 4, 256, 3, 200, 900), (32, 2)),
    ((8, 4, 256, 1, 512, 16896), (128, 2)),
    ((8, 4, 128, 1, 2000, 2000), (128, 1)),
    ((8, 4, 64, 1, 1000, 1000), (64, 1)),
    ((8, 4, 256, 1, 1000, 1000), (64, 1)),
    ((8, 4, 128, 4, 300, 2000), (256, 2)),
]


@pytest.mark.parametrize("case,chosen", CHOICES)
def test_rows_that_the_launcher_chooses(fake_hip, case, chosen):
    ct, (heads, group, d, batch, new, context) = fake_hip, case
    t = args(d=d, heads=heads, pages=4)
    q = torch.empty((batch * new, heads * group, d), dtype=torch.half)   # (never touched)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)
    attend(ct, t, new=q, out=q, table=ints(batch, -(-context // 16)), starts=ints(batch + 1), lens=ints(batch), max_new=new, max_context=context)
    variant, rows = resolved(ct)
    tiles = batch * new * group // rows + batch
    assert (variant, rows, _last(ct)[0].grid[0] / (heads * tiles)) == (name("f16", False, d), *chosen)


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", TILES)
def test_rows_that_the_caller_fixes(fake_hip, d, mx):
    ct, t = fake_hip, args(d=d, rows=500, mx=mx)
    for rows in TILES[d]:
        attend(ct, t, variant=name("f16", mx, d, rows))
        assert resolved(ct) == (name("f16", mx, d, rows), rows)
        assert _last(ct)[0].symbol.decode() == f"paged_attention_entry__{name('f16', mx, d)}"
    few = args(d=d, rows=2, mx=mx)
    attend(ct, few, variant=name("f16", mx, d, TILES[d][-1]))        # no larger tiles: the name stands for types and D
    assert _last(ct)[0].symbol.decode() == f"paged_attention_entry__{name('f16', mx, d)}_few"
    n0 = ct.lib().cutile_testing_launch_count()
    for wrong in (name("bf16", mx, d, 32), name("f16", not mx, d, 32), name("f16", mx, d, 512), name("f16", mx, d) + "_rows", name("f16", mx, d) + "+few",
                  name("f16", mx, 64 if d == 256 else 256, 32), name("f16", mx, d, 16)):
        with pytest.raises(ct.CutileError, match="does not fit these arguments|no variant"):
            attend(ct, t, variant=wrong)
    if d == 256:
        with pytest.raises(ct.CutileError, match="does not fit these arguments"):
            attend(ct, t, variant=name("f16", mx, d, 256))
    assert ct.lib().cutile_testing_launch_count() == n0
    ct.check(ct.lib().cutile_kernel_set_preferred_variant(b"paged_attention", name("f16", mx, d, 64).encode()))
    try:
        attend(ct, t)
        assert resolved(ct) == (name("f16", mx, d, 64), 64)
        attend(ct, args(d=64 if d == 256 else 256, rows=500, mx=mx))     # a pin that does not fit is passed over
    finally:
        ct.check(ct.lib().cutile_kernel_set_preferred_variant(b"paged_attention", None))


@pytest.mark.parametrize("heads,d,batch,context,shares", [(8, 256, 16, 2000, 2), (1, 256, 20, 8192, 13), (2, 256, 45, 4000, 3), (8, 256, 9, 6000, 8), (8, 256, 25, 3000, 3), (8, 256, 40, 2000, 2), (8, 256, 1, 16000, 32),
                                                          (8, 128, 16, 2000, 4), (8, 64, 16, 4000, 4), (4, 128, 24, 6000, 6)])
def test_workgroups_that_share_the_keys_of_single_tokens(fake_hip, heads, d, batch, context, shares):
    """two to a compute unit, or one where one fits (D = 256) and the tiles come out even"""
    ct = fake_hip
    t = args(d=d, heads=heads, pages=4)
    q = torch.empty((batch, heads * 4, d), dtype=torch.half)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)
    attend(ct, t, new=q, out=q, table=ints(batch, -(-context // 16)), starts=ints(batch + 1), lens=ints(batch), max_new=1, max_context=context)
    assert _last(ct)[0].grid[0] == heads * batch * shares


@pytest.mark.parametrize("image", ["pagedcache", "pagedattention", "logits"])
def test_no_vector_register_is_spilled(image):
    notes = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--notes", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cutile-rs_amd", "lib", image + ".hsaco")],
                           stdout=subprocess.PIPE, text=True, check=True).stdout
    kernels = notes.split("- .agpr_count")[1:]
    assert kernels
    for kernel in kernels:
        symbol = re.search(r"\n    \.name: +(\S+)", kernel)[1]
        assert int(re.search(r"\.vgpr_spill_count: (\d+)", kernel)[1]) == 0 and int(re.search(r"\.private_segment_fixed_size: (\d+)", kernel)[1]) == 0, symbol


# ---- on a GPU ---------------------------------------------------------------------------------------------------------------
class Compared:
    """a batch's problem on the device and its outputs in 64 bits, for launches of different tiles"""

    def __init__(self, dev, b, heads, group, d, dtype, mx, window=0, layout="nhd"):
        self.b, self.d, self.dtype, self.mx, self.window, self.dev = b, d, dtype, mx, window, dev
        self.q, self.k, self.v, self.scales, self.real = problem(b, heads, group, d, dtype, mx, dev, layout)
        self.scale = d ** -0.5
        self.parts = ref.attention(b, self.q, *self.real, float(torch.tensor(self.scale, dtype=torch.float32)), window)
        self.tol = bound(self.q.dtype, self.parts, d, max(b.held))

    def launch(self, ct, rows, **kw):
        q = self.q.to(self.dev)
        out = torch.full_like(q, 9.0)
        ct.paged_attention(q, self.k, self.v, *self.b.where(self.dev), ct.partition(out, [1, 1, self.d]), self.scale, window=self.window, variant=name(self.dtype, self.mx, self.d, rows),
                           **self.scales, **kw)
        assert resolved(ct)[1] == rows
        return out

    def check(self, ct, rows, **kw):
        out = self.launch(ct, rows, **kw)
        n = sum(self.b.new)
        got = out.cpu().double()
        assert bool((got[n:] == 9.0).all()), "rows that are nobody's"
        bad = ~((got[:n] - self.parts[0][:n]).abs() <= self.tol[:n])
        assert not bad.any(), (rows, int(bad.sum()), bad.numel(), bad.nonzero()[0].tolist())
        return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("group,page,layout", [(1, 16, "nhd"), (1, 7, "hnd"), (3, 64, "both"), (3, 1, "nhd"), (40, 16, "hnd")])
def test_gpu_every_tile(ct, dev, dtype, d, mx, group, page, layout):
    """pages that a wavefront's rows of a load end with and others, sequences that end inside a tile, and short ones among them"""
    new, held = ([300, 5, 0, 77, 1], [300, 400, 0, 900, 60]) if group < 8 else ([8, 1], [300, 77])
    p = Compared(dev, Batch(new, held, page, seed=d + group, rows=sum(new) + 3), 2, group, d, dtype, mx, layout=layout)
    for rows in TILES[d]:
        p.check(ct, rows)
        p.check(ct, rows, max_new=max(new), max_context=max(held))


@pytest.mark.gpu
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("window", [1, 50, 333])
@pytest.mark.parametrize("page", [16, 7])
def test_gpu_windows_of_every_tile(ct, dev, d, mx, window, page):
    p = Compared(dev, Batch([200, 90, 1], [900, 90, 700], page, seed=window), 2, 2, d, "bf16" if page == 7 else "f16", mx, window)
    for rows in TILES[d]:
        p.check(ct, rows)


@pytest.mark.gpu
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("page", [32, 5])
def test_gpu_keys_of_every_tile_dealt_out(ct, dev, d, mx, page):
    """two, a few and many workgroups to a tile, whoever arrives last; the workspace is left as it was found"""
    p = Compared(dev, Batch([150, 35], [6000, 1500], page, seed=page, rows=187), 1, 2, d, "f16", mx)
    for rows in TILES[d]:
        for context in (500, 1000, 6000):
            ws = torch.zeros(ct.PAGED_ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=dev)
            out = p.check(ct, rows, max_new=150, max_context=context, workspace=ws)
            for _ in range(2):
                assert torch.equal(out, p.launch(ct, rows, max_new=150, max_context=context, workspace=ws))
            assert int(ws[:16384].count_nonzero()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("new", [[150, 1, 0], [0, 33, 150], [2, 1, 5], [0, 0, 0]])
def test_gpu_padded_batches(ct, dev, d, mx, new):
    """as many rows as if every sequence had max_new tokens, which a launch may take for a batch of nothing else"""
    most = max(*new, 1)
    b = Batch(new, [400, 700, 200], 16, seed=d, rows=3 * most)
    b.starts = b.starts + 2 if sum(new) + 2 <= b.rows else b.starts          # rows in front of the first that are nobody's, too
    q, k, v, scales, real = problem(b, 2, 2, d, "f16", mx, dev)
    first = int(b.starts[0])
    parts = ref.attention(b, q[first:], *real, float(torch.tensor(d ** -0.5, dtype=torch.float32)))
    tol = bound(q.dtype, parts, d, 700)
    for rows in (None, *TILES[d]):
        for ws in (None, torch.zeros(ct.PAGED_ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=dev)):
            out = torch.full_like(q, 9.0).to(dev)
            ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), d ** -0.5, max_new=most, max_context=700, workspace=ws, variant=rows and name("f16", mx, d, rows), **scales)
            got, n = out.cpu().double(), sum(new)
            assert bool((got[:first] == 9.0).all()) and bool((got[first + n:] == 9.0).all())
            assert bool(((got[first:first + n] - parts[0][:n]).abs() <= tol[:n]).all()), rows


@pytest.mark.gpu
@pytest.mark.parametrize("d,mx", LARGE)
def test_gpu_every_tile_captured(ct, dev, d, mx):
    """replays for other contents, with eager work between them, equal the eager launch"""
    b = Batch([150, 1], [2000, 700], 16, seed=d)
    q, k, v, scales, real = problem(b, 2, 2, d, "bf16", mx, dev)
    table, starts, lens = b.where(dev)
    qd, out, eager = q.to(dev), torch.zeros_like(q, device=dev), torch.zeros_like(q, device=dev)
    for rows in TILES[d]:
        ws = [torch.zeros(ct.PAGED_ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=dev) for _ in range(2)]
        launch = lambda o, w, **kw: ct.paged_attention(qd, k, v, table, starts, lens, ct.partition(o, [1, 2, d]), 0.09, max_new=150, max_context=2000, workspace=w, variant=name("bf16", mx, d, rows), **scales, **kw)
        launch(out, ws[0])
        torch.cuda.synchronize()
        g = ct.CapturedGraph().capture(lambda s: launch(out, ws[0], stream=s))
        for i in range(3):
            qd.copy_(b.normal(*q.shape))
            lens.copy_(torch.tensor([2000 - 37 * i, 700 - 300 * i]))
            out.fill_(5.0)
            torch.cuda.synchronize()
            g.launch()
            g.synchronize()
            launch(eager, ws[1])
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
        g.close()


@pytest.mark.gpu
@pytest.mark.parametrize("d,mx", LARGE)
@pytest.mark.parametrize("gap", [17.6, 24.5])
def test_gpu_one_key_above_many_others_in_every_tile(ct, dev, d, mx, gap):
    for rows in TILES[d]:
        one_key_above_many(ct, dev, "f16", mx, d, 300, 5000, 100, gap, max_new=300, max_context=5000, variant=name("f16", mx, d, rows))
