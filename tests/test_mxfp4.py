"""The MXFP4 product (scaled_flat.h, mxfp4_flat.hip), alone and behind the kernels that make its operands."""
import math

import pytest
import torch

import block_ref as ref

# rows, n, k: edges of the 16-row blocks, of 64- and 128-column strips, of 128- and 256-value steps of K and of the steps in flight; K shared
# by workgroups; K that ends inside a step
SIZES = [(1, 4, 128), (1, 64, 256), (16, 68, 384), (17, 60, 640), (33, 132, 1024), (64, 4, 2176), (70, 128, 8192), (1, 64, 8192), (129, 260, 1152), (300, 516, 896)]


def codes(rows, cols, seed, device, lo=0, hi=256):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return torch.randint(lo, hi, (rows, cols), dtype=torch.uint8, generator=g).to(device)


def operands(m, n, k, seed, device):
    return (codes(m, k // 2, seed, device), codes(n, k // 2, seed + 1, device), codes(m, k // 32, seed + 2, device, 122, 132),
            codes(n, k // 32, seed + 3, device, 118, 128))


def product(x, y, xs, ys, alpha=1.0):
    a, b = ref.values(x, xs, "mxfp4"), ref.values(y, ys, "mxfp4")
    return alpha * (a @ b.t()), abs(alpha) * (a.abs() @ b.abs().t())


def assert_product(z, want, size, k):
    """f32 sums: the matrix unit adds 128 products with all their bits but those far below the largest (2^-21 of the sum of magnitudes were
    measured), and K / 128 of them and up to 8 shares are added one after another; then z's rounding"""
    slack = 2.0 ** -20 + (k / 128 + 16) * 2.0 ** -24
    half = torch.finfo(z.dtype).eps / 2 if z.dtype != torch.float32 else 2.0 ** -24
    off = (z.double() - want).abs()
    assert bool((off <= slack * size + half * (want.abs() + slack * size) + 2.0 ** -149).all()), float((off / size).max())


def variants_of(ct, out):
    return [v.split(":")[1] for v in ct.kernel_list() if v.startswith("linear_tile_mxfp4:" + out) and "+" not in v]


def test_refusals(fake_hip):
    ct = fake_hip
    n0 = ct.lib().cutile_testing_launch_count()
    u8 = lambda r, c: torch.zeros(r, c, dtype=torch.uint8)
    x, y, xs, ys, z = u8(16, 128), u8(32, 128), u8(16, 8), u8(32, 8), torch.zeros(16, 32)
    run = lambda z=z, x=x, y=y, xs=xs, ys=ys, tile=(128, 128), **kw: ct.linear_tile_mxfp4(ct.partition(z, list(tile)), x, y, xs, ys, 1.0, **kw)
    big = torch.empty(256 * ((1 << 23) + (1 << 16)), dtype=torch.uint8).as_strided((256, 128), ((1 << 23) + (1 << 16), 1))
    cases = [
        (lambda: run(y=u8(32, 64)), "packed bytes"),
        (lambda: run(xs=u8(16, 4)), "scales must be"),
        (lambda: run(ys=u8(16, 8)), "scales must be"),
        (lambda: run(z=torch.zeros(16, 16)), "expected"),
        (lambda: run(z=torch.zeros(16, 32, dtype=torch.half)), "z must be f32 or bf16"),
        (lambda: run(x=u8(16, 96), y=u8(32, 96), xs=u8(16, 6), ys=u8(32, 6), generics=[128, 128, 64]), "K a multiple of 128"),
        (lambda: run(x=u8(16, 96), y=u8(32, 96), xs=u8(16, 6), ys=u8(32, 6)), "K = 192 is not a multiple of BK = 128"),
        (lambda: run(z=torch.zeros(16, 30), y=u8(30, 128), ys=u8(30, 8)), "aligned rows"),
        (lambda: run(x=u8(16, 136)[:, :128]), "aligned rows"),
        (lambda: run(x=u8(16, 144)[:, 8:136]), "aligned rows"),
        (lambda: run(xs=u8(16, 9)[:, :8]), "aligned rows"),
        (lambda: run(xs=u8(8, 16).t()), "unit inner strides"),
        (lambda: run(x=big, xs=u8(256, 8), z=torch.zeros(256, 32)), "below 2 GiB"),
        (lambda: run(z=torch.zeros(1, 32).expand(16, 32)), "elements of z overlap"),
        (lambda: run(generics=[64, 128]), "generic BM"),
        (lambda: run(generics=[128, 128, 96]), "not a multiple of BK"),
        (lambda: run(generics=[128, 128, 128, 32]), "BK_PACKED"),
        (lambda: run(variant="bf16_flat16x64"), "does not fit these arguments"),
        (lambda: run(grid=(2, 1, 1)), "does not match the inferred partition grid"),
    ]
    for fn, msg in cases:
        with pytest.raises(ct.CutileError, match=msg):
            fn()
    assert ct.lib().cutile_testing_launch_count() == n0


def test_null_arguments_of_the_c_entry(fake_hip):
    import ctypes as C

    ct = fake_hip
    u8 = lambda r, c: torch.zeros(r, c, dtype=torch.uint8)
    t = lambda v, d: C.pointer(ct.tensor_arg(v, d))
    args = [C.pointer(ct.partition(torch.zeros(16, 32), [128, 128]).arg()), t(u8(16, 128), ct.F4E2M1FNX2), t(u8(32, 128), ct.F4E2M1FNX2), t(u8(16, 8), ct.F8E8M0FNU),
            t(u8(32, 8), ct.F8E8M0FNU)]
    fn = ct.lib().cutile_launch_linear_tile_mxfp4
    assert fn(None, *args, C.c_float(1.0), None) == 0
    for i in range(len(args)):
        assert fn(None, *[None if i == j else a for j, a in enumerate(args)], C.c_float(1.0), None) == -2


def chosen(ct, m, n, k, tile=(128, 128), out=torch.bfloat16, **kw):
    """kernel and workgroups of a launch without a GPU (256 compute units)"""
    from test_host_abi import _last

    u8 = lambda r, c: torch.empty(r, c, dtype=torch.uint8)
    ct.linear_tile_mxfp4(ct.partition(torch.empty(m, n, dtype=out), list(tile), **({"prefix": True} if "grid" in kw else {})), u8(m, k // 2), u8(n, k // 2), u8(m, k // 32), u8(n, k // 32), **kw)
    rec, _ = _last(ct)
    return rec.symbol.decode().split("__")[1], rec.grid[0]


# rows, n, k, shares of K on 128 x 128 tiles
SHARED = [(100, 68, 1152, 1), (130, 260, 4736, 2), (200, 388, 9088, 3), (100, 68, 16256, 4), (100, 68, 37760, 6), (100, 68, 64640, 8)]


def test_rule(fake_hip):
    """what a launch is given to, by extents alone: any tile of z that covers it all may be computed by another one"""
    ct = fake_hip
    for tile in ((128, 128), (256, 256)):
        assert chosen(ct, 1, 14336, 4096, tile) == ("bf16_flat16x64", 224)
        assert chosen(ct, 64, 14336, 4096, tile) == ("bf16_flat64x64", 224)
        assert chosen(ct, 200, 14336, 4096, tile) == ("bf16_128x128x256_e2x2_lone", 224)
        assert chosen(ct, 512, 4096, 14336, tile) == ("bf16_128x128x256_e2x2_lone", 256)      # 128 tiles, K in two
        assert chosen(ct, 1700, 11000, 6784, tile)[0] in ("bf16_128x128x256_e2x2", "bf16_256x256x256_e4x2")
        assert chosen(ct, 4096, 4096, 4096, tile) == ("bf16_256x256x256_e4x2", 256)
    named = {"variant": "bf16_128x128x256_e2x2"}
    for m, n, k, shares in SHARED:
        assert chosen(ct, m, n, k, **named) == ("bf16_128x128x256_e2x2_lone", shares * -(-m // 128) * -(-n // 128)), (m, n, k)
    assert chosen(ct, 2100, 2052, 1024, **named) == ("bf16_128x128x256_e2x2", 17 * 17)
    assert chosen(ct, 128, 128, 384, **named) == ("bf16_128x128x256_e2x2", 1)                 # too short for two groups
    assert chosen(ct, 300, 512, 16384, grid=(2, 1, 1)) == ("bf16_128x128x256_e2x2_lone", 2)    # a part of z: its own tiles, whole K
    assert chosen(ct, 600, 512, 16384, (256, 256), grid=(2, 1, 1)) == ("bf16_256x256x256_e4x2", 2)


def test_registers_of_the_products(fake_hip):
    """only the 256 x 256 kernels, which take every register, keep some in memory, outside their K loop"""
    import os
    import re
    import subprocess

    lib = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cutile-rs_amd", "lib")
    for image in ("mxfp4", "mxfp4flat"):
        notes = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--notes", os.path.join(lib, image + ".hsaco")], stdout=subprocess.PIPE, text=True, check=True).stdout
        for kernel in notes.split("- .agpr_count")[1:]:
            symbol = re.search(r"\n    \.name: +(\S+)", kernel)[1]
            most = 0 if "256x256x256" not in symbol else 3 if "bf16" in symbol else 5
            assert int(re.search(r"\.vgpr_spill_count: (\d+)", kernel)[1]) <= most, symbol


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,shares", SHARED)
def test_gpu_mxfp4_shared_k(ct, dev, m, n, k, shares):
    """the same sums launch after launch, on two streams at once, and captured (where nobody may share)"""
    args = operands(m, n, k, k, dev)
    want, size = product(*args)
    zs = [torch.full((m, n), math.nan, device=dev) for _ in range(4)]
    run = lambda i, stream=None: ct.linear_tile_mxfp4(ct.partition(zs[i], [128, 128]), *args, variant="f32_128x128x256_e2x2", stream=stream)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        run(0), run(1, streams[0].cuda_stream), run(2, streams[1].cuda_stream)
    torch.cuda.synchronize()
    for z in zs[:3]:
        assert_product(z, want, size, k)
    assert torch.equal(zs[0], zs[1]) and torch.equal(zs[0], zs[2])                             # shares are added in their order
    graph = ct.CapturedGraph().capture(lambda s: run(3, s))
    for _ in range(3):
        zs[3].fill_(math.nan)
        run(0)
        torch.cuda.synchronize()
        graph.launch()
        graph.synchronize()
        assert_product(zs[3], want, size, k)
    graph.close()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,variant", [(2100, 2052, 1152, "128x128x256_e2x2"), (2100, 2052, 640, None), (4300, 4100, 384, "256x256x256_e4x2"), (300, 34000, 256, None)])
def test_gpu_mxfp4_more_tiles_than_compute_units(ct, dev, m, n, k, variant):
    args = operands(m, n, k, 3, dev)
    want, size = product(*args)
    z = torch.full((m, n), math.nan, dtype=torch.bfloat16, device=dev)
    ct.linear_tile_mxfp4(ct.partition(z, [256, 256] if variant and variant[0] == "2" else [128, 128]), *args, variant=variant and "bf16_" + variant)
    assert_product(z, want, size, k)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [128, 256])
@pytest.mark.parametrize("k", [256, 2176])
def test_gpu_mxfp4_part_of_z(ct, dev, tile, k):
    """a grid over some tiles of z leaves the others alone"""
    m, n = 2 * tile + 40, 2 * tile + 36
    args = operands(m, n, k, 8, dev)
    want, size = product(*args)
    z = torch.full((m, n), 7.0, device=dev)
    ct.linear_tile_mxfp4(ct.partition(z, [tile, tile], prefix=True), *args, grid=(2, 1, 1))
    assert_product(z[: 2 * tile, :tile], want[: 2 * tile, :tile], size[: 2 * tile, :tile], k)
    assert bool((z[2 * tile:] == 7.0).all()) and bool((z[:, tile:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_gpu_mxfp4(ct, dev, m, n, k, out):
    dt = torch.float32 if out == "f32" else torch.bfloat16
    args = operands(m, n, k, m + n + k, dev)
    want, size = product(*args, 0.75)
    for variant in variants_of(ct, out) + [None]:
        for tile in ([128, 128], [256, 256]):
            z = torch.full((m + 1, n), 7.0, dtype=dt, device=dev)       # a row behind z that nothing may touch
            for _ in range(2):                                           # the second launch finds the first one's counters at 0
                z[:m] = math.nan
                try:
                    ct.linear_tile_mxfp4(ct.partition(z[:m], tile), *args, 0.75, variant=variant)
                except ct.CutileError as e:                              # a tile of 256 is no kernel of a partition of 128
                    assert variant is not None and "does not fit" in str(e) and "flat" not in variant
                    break
                torch.cuda.synchronize()
                assert_product(z[:m], want, size, k)
                assert bool((z[m] == 7.0).all()), variant


@pytest.mark.gpu
@pytest.mark.parametrize("k", [128, 384, 640, 1152])
def test_gpu_mxfp4_nan_scales_stay_in_their_row(ct, dev, k):
    """K that ends inside a 256-value step, beside rows whose scales are NaN: no other row sees them.  A row and a column far from 1, inside f32."""
    m, n = 40, 136
    x, y, xs, ys = operands(m, n, k, 9, dev)
    xs[3], ys[40], xs[39], ys[135, 0] = 255, 255, 255, 255
    xs[7], ys[50] = 227, 20
    want, size = product(x, y, xs, ys)
    for variant in variants_of(ct, "f32") + [None]:
        z = torch.zeros(m, n, device=dev)
        ct.linear_tile_mxfp4(ct.partition(z, [256, 256] if variant and "256x256" in variant else [128, 128]), x, y, xs, ys, variant=variant)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(z), nan), variant
        assert_product(torch.where(nan, 0.0, z), torch.where(nan, 0.0, want), torch.where(nan, 1.0, size), k)


@pytest.mark.gpu
def test_gpu_mxfp4_strided_operands(ct, dev):
    """rows of a wider buffer, their scales too, z a part of a wider one"""
    m, n, k = 45, 200, 768
    big = operands(2 * m, 2 * n, 2 * k, 5, dev)
    x, y, xs, ys = big[0][::2, 64:64 + k // 2], big[1][::2, : k // 2], big[2][1::2, 4:4 + k // 32], big[3][::2, 8:8 + k // 32]
    want, size = product(x.contiguous(), y.contiguous(), xs.contiguous(), ys.contiguous())
    for variant in variants_of(ct, "bf16") + [None]:
        wide = torch.full((m, n + 24), 7.0, dtype=torch.bfloat16, device=dev)
        ct.linear_tile_mxfp4(ct.partition(wide[:, 8:n + 8], [256, 256] if variant and "256x256" in variant else [128, 128]), x, y, xs, ys, variant=variant)
        assert_product(wide[:, 8:n + 8], want, size, k)
        assert bool((wide[:, :8] == 7.0).all()) and bool((wide[:, n + 8:] == 7.0).all())


# ---- a gated MLP in 4 bits, as it is used --------------------------------------------------------------------------------------
class Mlp:
    """residual + x -> norm -> gate and up -> silu * -> down, every product on MXFP4 operands; widths that fill no block"""

    def __init__(self, ct, dev, rows, hidden, inter, seed, device_stream=None):
        self.ct, self.rows, self.hidden, self.inter = ct, rows, hidden, inter
        g = torch.Generator(device="cpu")
        g.manual_seed(seed)
        bf = torch.bfloat16
        rand = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to(bf).to(dev)
        self.kh, self.ki = -(-hidden // 128) * 128, -(-inter // 128) * 128
        self.x, self.r, self.w = rand(rows, hidden), rand(rows, hidden), 1 + rand(hidden, std=0.1)
        self.weights = {}
        for name, (n, k, kp) in {"gate_up": (2 * inter, hidden, self.kh), "down": (hidden, inter, self.ki)}.items():
            w = rand(k, n, std=k ** -0.5).t()                             # kept as [K, N]
            q = self.bytes(n, kp)
            ct.block_quantize(w, whole(ct, q[0]), whole(ct, q[1]), "mxfp4")
            self.weights[name] = q
        self.a, self.h = self.bytes(rows, self.kh), self.bytes(rows, self.ki)
        self.residual_out, self.both, self.out = torch.zeros(rows, hidden, dtype=bf, device=dev), torch.zeros(rows, 2 * inter, dtype=bf, device=dev), torch.zeros(rows, hidden, dtype=bf, device=dev)

    def bytes(self, rows, k):
        return ref.buffers(rows, k, "mxfp4", "cuda")

    def run(self, stream=None):
        ct, kw = self.ct, {"stream": stream}
        ct.add_rms_norm_quantize(self.r, self.x, self.w, whole(ct, self.a[0]), whole(ct, self.a[1]), whole(ct, self.residual_out), 1e-6, "mxfp4", **kw)
        ct.linear_tile_mxfp4(ct.partition(self.both, [128, 128]), self.a[0], self.weights["gate_up"][0], self.a[1], self.weights["gate_up"][1], **kw)
        ct.silu_mul_quantize(self.both[:, : self.inter], self.both[:, self.inter:], whole(ct, self.h[0]), whole(ct, self.h[1]), "mxfp4", **kw)
        ct.linear_tile_mxfp4(ct.partition(self.out, [128, 128]), self.h[0], self.weights["down"][0], self.h[1], self.weights["down"][1], **kw)

    def check(self):
        """each step against 64 bits on what the step before it left"""
        c = self.x.double() + self.r.double()
        assert torch.equal(self.residual_out, (self.x.float() + self.r.float()).bfloat16())
        ref.assert_quantised(*self.a, c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * self.w.double(), "mxfp4", slack=64 * 2.0 ** -24)
        want, size = product(self.a[0], self.weights["gate_up"][0], self.a[1], self.weights["gate_up"][1])
        assert_product(self.both, want, size, self.kh)
        gate, up = self.both[:, : self.inter].double(), self.both[:, self.inter:].double()
        ref.assert_quantised(*self.h, gate / (1 + torch.exp(-gate)) * up, "mxfp4", slack=6 * 2.0 ** -24, tiny=2.0 ** -126)
        want, size = product(self.h[0], self.weights["down"][0], self.h[1], self.weights["down"][1])
        assert_product(self.out, want, size, self.ki)


def whole(ct, t):
    return ct.partition(t, [1, t.shape[1]])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,inter", [(1, 512, 1408), (7, 500, 1300), (130, 1024, 2050)])
def test_gpu_mlp(ct, dev, rows, hidden, inter):
    m = Mlp(ct, dev, rows, hidden, inter, rows)
    m.run()
    torch.cuda.synchronize()
    m.check()


@pytest.mark.gpu
def test_gpu_mlp_captured_and_on_two_streams(ct, dev):
    """two layers captured into graphs of their own, replayed side by side with eager runs and new inputs between the replays"""
    layers = [Mlp(ct, dev, 5, 512, 1408, s) for s in (1, 2)]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in layers]
    for m in layers:
        m.run()                                                            # loads what a capture may not
    torch.cuda.synchronize()
    for m in layers:
        graphs.append(ct.CapturedGraph().capture(lambda s, m=m: m.run(s)))
    other = Mlp(ct, dev, 64, 512, 1408, 3)
    for turn in range(4):
        for m in layers:
            m.x.normal_(generator=torch.Generator(device="cuda").manual_seed(turn))
            m.out.zero_(), m.both.zero_(), m.a[0].zero_(), m.h[0].zero_()
        torch.cuda.synchronize()
        for g in graphs:
            g.launch()
        with torch.cuda.stream(streams[0]):
            other.run()
        for g in graphs:
            g.synchronize()
        torch.cuda.synchronize()
        for m in layers + [other]:
            m.check()
    for m, s in zip(layers, streams):                                       # eager on streams of their own, at once
        m.out.zero_(), m.both.zero_()
    torch.cuda.synchronize()
    for m, s in zip(layers, streams):
        for _ in range(3):
            m.run(s.cuda_stream)
    torch.cuda.synchronize()
    for m in layers:
        m.check()
    for g in graphs:
        g.close()
