"""Block-scaled rows: quantisation, reading back, and the norm and gated activation that end in it (block_scale.hip)."""
import math

import pytest
import torch

import block_ref as ref

FORMATS = ["mxfp8", "mxfp4", "nvfp4"]
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# one value, one short of a block, a block, one more, lengths that are no multiple of a unit, several workgroups, a long row
LENGTHS = [1, 15, 16, 31, 32, 33, 100, 256, 1000, 5001, 8192, 20000]


# of nvfp4's scale, relative: f32 roundings of tensor_scale, of 6 tensor_scale, of its reciprocal and of the product with it (what follows in
# the elements is in assert_quantised)
NVFP4_SLACK = 4 * 2.0 ** -24


def whole(ct, t):
    return ct.partition(t, [1, t.shape[1]])


def normal(shape, seed, device, dtype=torch.float32, std=1.0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(device).to(dtype)


def g_of(x, fmt):
    return float(x[torch.isfinite(x)].abs().max().float()) / (6 * 448.0) if fmt == "nvfp4" else 1.0


# ---- refusals, without a GPU ---------------------------------------------------------------------------------------------
def test_refusals(fake_hip):
    ct = fake_hip
    n0 = ct.lib().cutile_testing_launch_count()
    x = torch.zeros(4, 64, dtype=torch.half)
    data, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    q = lambda x=x, d=data, s=scales, fmt="mxfp8", *a, **kw: ct.block_quantize(x, whole(ct, d), whole(ct, s), fmt, *a, **kw)
    w = torch.zeros(64, dtype=torch.half)
    norm = lambda r=x, x=x, w=w, d=data, s=scales, ro=x, **kw: ct.add_rms_norm_quantize(r, x, w, whole(ct, d), whole(ct, s), whole(ct, ro), 1e-6, "mxfp8", **kw)
    silu = lambda g=x, u=x, **kw: ct.silu_mul_quantize(g, u, whole(ct, data), whole(ct, scales), "mxfp8", **kw)
    deq = lambda d=data, s=scales, o=x, fmt="mxfp8", *a: ct.block_dequantize(d, s, whole(ct, o), fmt, *a)
    wide = torch.zeros(4, 80, dtype=torch.uint8)
    cases = [
        (lambda: q(fmt="mxfp6"), "unknown block-scaled format"),
        (lambda: q(d=data.float()), "tensors of bytes"),
        (lambda: q(x=x.double()), "x must be f16, bf16 or f32"),
        (lambda: q(x=x.to(torch.uint8)), "x must be f16, bf16 or f32"),
        (lambda: q(x=torch.zeros(64, dtype=torch.half)), "expected rank 2"),
        (lambda: q(s=torch.zeros(4, 4, dtype=torch.uint8)), "whole blocks of 32 and scales"),
        (lambda: q(d=torch.zeros(4, 48, dtype=torch.uint8)), "whole blocks of 32"),
        (lambda: q(s=torch.zeros(3, 2, dtype=torch.uint8)), "whole blocks of 32 and scales"),
        (lambda: q(x=torch.zeros(4, 65, dtype=torch.half)), "out holds 4 rows of 64 values"),
        (lambda: q(x=torch.zeros(3, 64, dtype=torch.half)), "out holds 4 rows of 64 values"),
        (lambda: q(d=torch.zeros(64, 4, dtype=torch.uint8).t()), "contiguous rows"),
        (lambda: q(d=torch.zeros(4, 65, dtype=torch.uint8)[:, :64]), "8-byte boundaries"),
        (lambda: q(d=torch.zeros(4, 72, dtype=torch.uint8)[:, 1:65]), "8-byte boundaries"),
        (lambda: q(d=torch.zeros(1, 64, dtype=torch.uint8).expand(4, 64)), "do not overlap"),
        (lambda: q(s=torch.zeros(1, 2, dtype=torch.uint8).expand(4, 2)), "do not overlap"),
        (lambda: q(s=torch.zeros(2, 4, dtype=torch.uint8).t()), "contiguous rows"),
        (lambda: q(x, data, scales, "mxfp8", 2.0), "no tensor_scale"),
        (lambda: q(x, data[:, :32], torch.zeros(4, 4, dtype=torch.uint8), "nvfp4", 0.0), "tensor_scale must lie"),
        (lambda: q(x, data[:, :32], torch.zeros(4, 4, dtype=torch.uint8), "nvfp4", -1.0), "tensor_scale must lie"),
        (lambda: q(x, data[:, :32], torch.zeros(4, 4, dtype=torch.uint8), "nvfp4", math.nan), "tensor_scale must lie"),
        (lambda: q(x, data[:, :32], torch.zeros(4, 4, dtype=torch.uint8), "nvfp4", math.inf), "tensor_scale must lie"),
        (lambda: q(generics=[32]), "generic N"),
        (lambda: q(grid=(3, 1, 1)), "does not match the inferred partition grid"),
        (lambda: q(variant="mxfp4_f16_any"), "does not fit these arguments"),
        (lambda: ct.block_quantize(x, ct.partition(data, [1, 32]), whole(ct, scales), "mxfp8"), "whole row"),
        (lambda: ct.block_quantize(x, ct.partition(data, [2, 64]), whole(ct, scales), "mxfp8"), "whole row"),
        (lambda: ct.block_quantize(x, ct.partition(data, [1, 64], prefix=True), ct.partition(scales, [1, 2], prefix=True), "mxfp8"), "Launch grid required"),
        (lambda: norm(w=w[:32]), "must be shared by all tensors"),
        (lambda: norm(w=w.float()), "all be f16 or all bf16"),
        (lambda: norm(x=x.bfloat16()), "all be f16 or all bf16"),
        (lambda: norm(r=x[:2]), "residual must have its rows"),
        (lambda: norm(r=x[:, :32]), "must be shared by all tensors"),
        (lambda: norm(ro=x[:2]), "same rows"),
        (lambda: norm(ro=x.float()), "all be f16 or all bf16"),
        (lambda: norm(ro=x[:1].expand(4, 64)), "elements of residual_out overlap"),
        (lambda: norm(ro=x[:, :1].expand(4, 64)), "elements of residual_out overlap"),
        (lambda: norm(variant="none"), "does not fit these arguments"),
        (lambda: ct.rms_norm_quantize(x.float(), w.float(), whole(ct, data), whole(ct, scales), 1e-6, "mxfp8"), "all be f16 or all bf16"),
        (lambda: silu(u=x[:, :32]), "up has another shape"),
        (lambda: silu(u=x.bfloat16()), "both be f16 or both bf16"),
        (lambda: silu(g=x.float(), u=x.float()), "both be f16 or both bf16"),
        (lambda: deq(o=torch.zeros(4, 65, dtype=torch.half)), "x holds 4 rows of 64 values"),
        (lambda: deq(o=torch.zeros(5, 64, dtype=torch.half)), "x holds 4 rows of 64 values"),
        (lambda: deq(o=torch.zeros(4, 64, dtype=torch.double)), "out must be f16, bf16 or f32"),
        (lambda: deq(o=x[:1].expand(4, 64)), "elements of out overlap"),
        (lambda: deq(o=x.flatten()[:130].as_strided((4, 64), (20, 1))), "elements of out overlap"),
        (lambda: deq(s=wide), "whole blocks of 32 and scales"),
        (lambda: deq(data, scales, x, "mxfp4", 3.0), "whole blocks of 32 and scales"),
    ]
    for i, (fn, msg) in enumerate(cases):
        with pytest.raises(ct.CutileError, match=msg):
            fn()
            print("case", i, msg)
    assert ct.lib().cutile_testing_launch_count() == n0


def test_null_arguments_of_the_c_entries(fake_hip):
    """every pointer of the C entries may be null by mistake: an error, not a fault"""
    import ctypes as C

    ct = fake_hip
    x, data, scales, w = (torch.zeros(4, 64, dtype=torch.half), torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), torch.zeros(64, dtype=torch.half))
    t = lambda v, d=None: C.pointer(ct.tensor_arg(v, d))
    p = lambda v, d=None: C.pointer(ct.Partition(v, [1, v.shape[1]], False, d).arg())
    f32 = C.c_float
    calls = {
        "block_quantize": [t(x), p(data, ct.F8E4M3FN), p(scales, ct.F8E8M0FNU), f32(1.0)],
        "block_dequantize": [t(data, ct.F8E4M3FN), t(scales, ct.F8E8M0FNU), f32(1.0), p(x)],
        "rms_norm_quantize": [t(x), t(w), p(data, ct.F8E4M3FN), p(scales, ct.F8E8M0FNU), f32(1e-6), f32(1.0)],
        "add_rms_norm_quantize": [t(x), t(x), t(w), p(data, ct.F8E4M3FN), p(scales, ct.F8E8M0FNU), p(x), f32(1e-6), f32(1.0)],
        "silu_mul_quantize": [t(x), t(x), p(data, ct.F8E4M3FN), p(scales, ct.F8E8M0FNU), f32(1.0)],
    }
    for name, args in calls.items():
        fn = getattr(ct.lib(), "cutile_launch_" + name)
        assert fn(None, *args, None) == 0, name
        for i, a in enumerate(args):
            if isinstance(a, C.c_float):
                continue
            assert fn(None, *[None if j == i else b for j, b in enumerate(args)], None) == -2, (name, i)


def test_launch_modes_and_coverage(fake_hip):
    """a prefix partition covers the rows that its grid says; compile-only launches enqueue nothing"""
    import struct

    ct = fake_hip
    x = torch.zeros(10, 64, dtype=torch.half)
    data, scales = torch.zeros(10, 64, dtype=torch.uint8), torch.zeros(10, 2, dtype=torch.uint8)
    ct.block_quantize(x, ct.partition(data, [4, 64], prefix=True), ct.partition(scales, [4, 2], prefix=True), "mxfp8", grid=(2, 1, 1), generics=[64])
    from test_host_abi import _last
    rec, args = _last(ct)
    assert rec.symbol.startswith(b"block_quantize_entry__mxfp8_f16")
    n0 = ct.lib().cutile_testing_launch_count()
    ct.check(ct.lib().cutile_set_launch_mode(1))
    try:
        ct.block_quantize(x, whole(ct, data), whole(ct, scales), "mxfp8")
        assert ct.last_resolved()["function"] == "block_quantize"
    finally:
        ct.check(ct.lib().cutile_set_launch_mode(0))
    assert ct.lib().cutile_testing_launch_count() == n0


def test_rows_beyond_one_dispatch(fake_hip):
    """fewer than 2^32 lanes make a grid: what has more rows goes to the kernels that stride over them"""
    from test_host_abi import _last

    ct = fake_hip
    rows = (1 << 26) + 5
    data, scales = torch.empty(rows, 16, dtype=torch.uint8), torch.empty(rows, 1, dtype=torch.uint8)      # (never touched)
    x, w = torch.empty(1, 32, dtype=torch.half).expand(rows, 32), torch.empty(32, dtype=torch.half)
    ct.rms_norm_quantize(x, w, whole(ct, data), whole(ct, scales), 1e-6, "mxfp4")
    rec, _ = _last(ct)
    assert rec.symbol.decode().endswith("mxfp4_f16_any") and rec.grid[0] * rec.block[0] < 1 << 32
    ct.rms_norm_quantize(x[:-5], w, whole(ct, data[:-5]), whole(ct, scales[:-5]), 1e-6, "mxfp4")
    assert _last(ct)[0].symbol.decode().endswith("mxfp4_f16_any")
    ct.rms_norm_quantize(x[:-9], w, whole(ct, data[:-9]), whole(ct, scales[:-9]), 1e-6, "mxfp4")
    assert _last(ct)[0].symbol.decode().endswith("mxfp4_f16_w1v1")


# ---- quantisation ----------------------------------------------------------------------------------------------------------
def quantised(ct, x, fmt, k=None, g=1.0, rows=None, **kw):
    rows = x.shape[0] if rows is None else rows
    data, scales = ref.buffers(rows, ref.padded(x.shape[1], fmt) if k is None else k, fmt, x.device, extra_rows=1)
    ct.block_quantize(x, whole(ct, data[:rows]), whole(ct, scales[:rows]), fmt, g, **kw)
    torch.cuda.synchronize()
    assert int((data[rows:] != 0xA5).sum() + (scales[rows:] != 0xA5).sum()) == 0, "rows behind the last"
    return data[:rows], scales[:rows]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", LENGTHS)
def test_gpu_quantize(ct, dev, fmt, dtype, n):
    """rows of any length, from tight to wide apart; the input is exact, so every code is the rounding (nvfp4: its scale is found with
    roundings of f32)"""
    for rows, pad in ((1, 0), (5, 0), (37, 3)):
        x = normal((rows, n + pad), 100 + n + rows, dev, TYPES[dtype]) * torch.exp2(torch.arange(rows, device=dev) % 13 - 6.0).to(TYPES[dtype])[:, None]
        x = x[:, pad:]
        g = g_of(x, fmt)
        k = ref.padded(n, fmt) + (ref.BLOCK[fmt] * 3 if rows == 5 else 0)      # blocks of nothing but padding
        data, scales = quantised(ct, x, fmt, k, g)
        ref.assert_quantised(data, scales, x.double(), fmt, g, slack=NVFP4_SLACK if fmt == "nvfp4" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gpu_quantize_strides(ct, dev, fmt, dtype):
    """transposed, every second column, one row repeated, a part of wider rows whose start is on no boundary"""
    base = normal((300, 517), 7, dev, TYPES[dtype])
    wide = normal((70, 1030), 8, dev, TYPES[dtype])
    for x in (base.t(), base[:, ::2], base[:1].expand(9, 517), wide[:, 3:1027], wide[1:, 1:130], wide[:, 6:70], base.t()[5:, 3:200], base[::3].t()):
        g = g_of(x, fmt)
        data, scales = quantised(ct, x, fmt, None, g)
        ref.assert_quantised(data, scales, x.double(), fmt, g, slack=NVFP4_SLACK if fmt == "nvfp4" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_gpu_quantize_special_values(ct, dev, fmt):
    """zeros of both signs, NaN, infinities, subnormals, the type's extremes, values halfway between two codes: each in a block of its own"""
    b = ref.BLOCK[fmt]
    for name, dt in TYPES.items():
        info = torch.finfo(dt)
        grid = ref.grid_of(fmt)
        mids = ((grid[1:] + grid[:-1]) / 2)[-b + 1:]
        rows = [torch.zeros(b), -torch.zeros(b), torch.full((b,), info.max), torch.full((b,), -info.max), torch.full((b,), info.tiny), torch.full((b,), info.smallest_normal / 4),
                torch.cat((torch.tensor([float(grid[-1])]), torch.nn.functional.pad(mids.float(), (0, b - 1 - mids.numel())))),
                torch.cat((torch.tensor([-float(grid[-1])]), torch.nn.functional.pad(-mids.float(), (0, b - 1 - mids.numel()))))]
        for at in (0, b // 2, b - 1):
            for bad in (math.nan, math.inf, -math.inf):
                rows.append(torch.ones(b))
                rows[-1][at] = bad
        rows.append(torch.ones(b))                                        # a block beside those
        x = torch.stack(rows).to(dt).reshape(1, -1).to(dev)
        g = 2.0 ** -9 if fmt == "nvfp4" else 1.0
        data, scales = quantised(ct, x, fmt, None, g)
        ref.assert_quantised(data, scales, x.double(), fmt, g, slack=NVFP4_SLACK if fmt == "nvfp4" else 0.0)
        back = torch.zeros(x.shape, device=dev)
        ct.block_dequantize(data, scales, whole(ct, back), fmt, g)
        lost = ~torch.isfinite(x.view(-1, b)).all(-1)
        assert bool(torch.isnan(back.view(-1, b)[lost]).all()) and bool(torch.isfinite(back.view(-1, b)[~lost]).all()), name


@pytest.mark.gpu
def test_gpu_quantize_tensor_scale_range(ct, dev):
    """nvfp4: the ends of tensor_scale, values too small for any scale and too large for the largest"""
    x = torch.cat([normal((1, 64), 3, dev) * s for s in (1e-30, 1e-6, 1.0, 1e6, 1e30)], 1)
    for g in (2.0 ** -100, 1.0, 1e3, 2.0 ** 100):
        data, scales = quantised(ct, x, "nvfp4", None, g)
        ref.assert_quantised(data, scales, x.double(), "nvfp4", g, slack=NVFP4_SLACK)


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1.0, 14.0, 81.5, 0.8984375, 3.359375, 110.5])
def test_gpu_quantize_calibrated_tensor_scale(ct, dev, most):
    """g = largest / (6 * 448): many blocks' scales lie on a border between two; the bytes are those of the definition in f32"""
    x = normal((300, 512), 21, dev, torch.bfloat16)
    x = (x / x.abs().max() * most).bfloat16()
    x[7, 9] = most
    g = float(x.abs().max().float()) / (6.0 * 448.0)
    data, scales = quantised(ct, x, "nvfp4", None, g)
    g32 = torch.tensor(g, dtype=torch.float32)
    v = x.float().cpu().view(300, 32, 16)
    s = (v.abs().amax(-1) * (1.0 / (6.0 * g32))).clamp(max=448.0).to(torch.float8_e4m3fn)
    assert torch.equal(scales.cpu(), s.view(torch.uint8))
    unit = s.float()
    q = torch.where(unit > 0, 1.0 / (unit * g32), 0.0).unsqueeze(-1) * v
    codes = ref.nearest(q.double(), ref.grid_of("nvfp4")).view(300, 512)
    assert torch.equal(ref.unpack(data, "nvfp4").cpu().long() & 7, codes)


@pytest.mark.gpu
def test_gpu_quantize_covers_the_rows_of_its_grid(ct, dev):
    x = normal((10, 96), 5, dev, torch.half)
    data, scales = ref.buffers(10, 96, "mxfp8", dev)
    ct.block_quantize(x, ct.partition(data, [4, 96], prefix=True), ct.partition(scales, [4, 3], prefix=True), "mxfp8", grid=(2, 1, 1))
    torch.cuda.synchronize()
    ref.assert_quantised(data[:8], scales[:8], x[:8].double(), "mxfp8")
    assert int((data[8:] != 0xA5).sum() + (scales[8:] != 0xA5).sum()) == 0
    data, scales = ref.buffers(7, 96, "mxfp8", dev)                         # fewer rows than x
    ct.block_quantize(x, ct.partition(data, [3, 96]), ct.partition(scales, [3, 3]), "mxfp8")
    ref.assert_quantised(data, scales, x[:7].double(), "mxfp8")


@pytest.mark.gpu
def test_gpu_quantize_and_back_beyond_32_bit_offsets(ct, dev):
    """more than 2^32 bytes of input: the last rows are where their offsets say"""
    rows, n = 300000, 8192
    x = torch.zeros((rows, n), dtype=torch.bfloat16, device=dev)
    tail = normal((64, n), 11, dev, torch.bfloat16)
    x[-64:] = tail
    x[:64] = tail
    for fmt in ("mxfp8", "mxfp4"):
        data, scales = ref.buffers(rows, n, fmt, dev)
        ct.block_quantize(x, whole(ct, data), whole(ct, scales), fmt)
        for part in (slice(0, 64), slice(rows - 64, rows)):
            ref.assert_quantised(data[part], scales[part], tail.double(), fmt)
        assert int(scales[64:-64].view(torch.uint8).max()) == 0
        x.fill_(1.0)
        ct.block_dequantize(data, scales, whole(ct, x), fmt)
        assert torch.equal(x[-64:].double(), ref.values(data[-64:], scales[-64:], fmt)) and int(torch.count_nonzero(x[64:-64])) == 0
        x[-64:] = tail
        x[:64] = tail
        del data, scales


# ---- reading back ----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gpu_dequantize_every_code_and_scale(ct, dev, fmt, dtype):
    """each scale byte against each data byte, one rounding to out's type (f32: exact but for 2^-149, and nvfp4's factor)"""
    b = ref.BLOCK[fmt]
    per_row = 256 if fmt == "mxfp8" else 512
    data = torch.arange(256, dtype=torch.uint8, device=dev).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device=dev)[:, None].repeat(1, per_row // b)
    g = 0.37 if fmt == "nvfp4" else 1.0
    out = torch.full((257, per_row), 7.0, dtype=TYPES[dtype], device=dev)
    ct.block_dequantize(data, scales, whole(ct, out[:256]), fmt, g)
    want = ref.values(data, scales, fmt, torch.tensor(g, dtype=torch.float32).double().item())
    got = out[:256].double()
    assert bool((out[256] == 7.0).all())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    info = torch.finfo(TYPES[dtype])
    over = want.abs() >= info.max * (1 + info.eps / 4)
    assert torch.equal(got[over], torch.copysign(torch.full_like(want, math.inf), want)[over])
    fine = torch.isfinite(want) & ~over
    # a step is eps of the value, or of the smallest normal number below it; f32 holds the product before the rounding to out
    step = info.eps / 2 * want.abs().clamp(min=info.smallest_normal) + 2.0 ** -24 * want.abs() * (fmt == "nvfp4") + 2.0 ** -150
    assert bool(((got - want).abs() <= step)[fine].all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_gpu_dequantize_lengths_and_strides(ct, dev, fmt):
    for rows, n in ((1, 1), (3, 33), (2, 100), (40, 1000), (7, 5001)):
        x = normal((rows, n), rows + n, dev)
        g = g_of(x, fmt)
        data, scales = quantised(ct, x, fmt, None, g)
        want = ref.values(data, scales, fmt, torch.tensor(g, dtype=torch.float32).double().item())[:, :n]
        for out in (torch.full((rows + 1, n), 7.0, device=dev)[:rows], torch.zeros((n, rows), device=dev).t(), torch.full((rows, n + 5), 7.0, device=dev)[:, 3:n + 3],
                    torch.full((rows, 2 * n), 7.0, device=dev)[:, ::2], torch.zeros((rows, max(1, n - 9)), dtype=torch.half, device=dev)):
            ct.block_dequantize(data, scales, whole(ct, out), fmt, g)
            assert bool(((out.double() - want[:, : out.shape[1]]).abs() <= torch.finfo(out.dtype).eps * want[:, : out.shape[1]].abs()).all())
            if out.dtype == torch.float32 and out._base is not None and out._base.shape != out.shape and out.stride(1) == 1:
                assert int((out._base == 7.0).sum()) >= out._base.numel() - out.numel(), "around out"


# ---- norm ------------------------------------------------------------------------------------------------------------------
def norm_slack(n):
    """relative to 2^-24: the sum's own rounding; half of what the sum of squares collects - 2 per square and one per addition, of which a
    value passes at most n / 256 in its thread and 16 across lanes and threads; mean, eps, root and reciprocal; two products"""
    return (1 + 0.5 * (2 + n / 256 + 8 + 16) + 4 + 2) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS + [40000])
@pytest.mark.parametrize("add", [False, True])
def test_gpu_norm(ct, dev, fmt, dtype, n, add):
    dt = TYPES[dtype]
    for rows, pad in ((1, 0), (6, 0), (11, 5)):
        x, r = (normal((rows, n + pad), 31 * n + rows + i, dev, dt, 1.0 + i)[:, pad:] for i in range(2))
        w = (1 + 0.3 * normal((n,), n, dev)).to(dt)
        c = x.double() + r.double() if add else x.double()
        want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        g = g_of(want, fmt)
        data, scales = ref.buffers(rows, ref.padded(n, fmt) + (ref.BLOCK[fmt] * 2 if rows == 6 else 0), fmt, dev, extra_rows=1)
        outs = whole(ct, data[:rows]), whole(ct, scales[:rows])
        if add:
            ro = torch.full((rows + 1, n), 7.0, dtype=dt, device=dev)
            ct.add_rms_norm_quantize(r, x, w, *outs, whole(ct, ro[:rows]), 1e-6, fmt, g)
            assert bool((ro[rows] == 7.0).all())
            assert torch.equal(ro[:rows], (x.float() + r.float()).to(dt))       # f32 sum, one rounding
        else:
            ct.rms_norm_quantize(x, w, *outs, 1e-6, fmt, g)
        torch.cuda.synchronize()
        assert int((data[rows:] != 0xA5).sum() + (scales[rows:] != 0xA5).sum()) == 0
        g = torch.tensor(g, dtype=torch.float32).double().item()
        ref.assert_quantised(data[:rows], scales[:rows], want, fmt, g, slack=norm_slack(n) + NVFP4_SLACK)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [256, 1001, 8192])
def test_gpu_norm_in_place_and_strided(ct, dev, n):
    """residual_out is residual, then x; rows with a stride, a transposed residual, weights with a stride"""
    dt = torch.bfloat16
    for alias in ("residual", "x", "strided"):
        x, r = normal((9, n), 1, dev, dt), normal((9, n), 2, dev, dt)
        w = (1 + 0.3 * normal((2 * n,), 3, dev)).to(dt)[:n]
        if alias == "strided":
            x, r, w = normal((9, 2 * n), 1, dev, dt)[:, ::2], normal((n, 9), 2, dev, dt).t(), (1 + 0.3 * normal((2 * n,), 3, dev)).to(dt)[::2]
        total = x.float() + r.float()
        c = x.double() + r.double()
        want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w.double()
        ro = {"residual": r, "x": x, "strided": torch.zeros((n, 9), dtype=dt, device=dev).t()}[alias]
        data, scales = ref.buffers(9, ref.padded(n, "mxfp8"), "mxfp8", dev)
        ct.add_rms_norm_quantize(r, x, w, whole(ct, data), whole(ct, scales), whole(ct, ro), 1e-5, "mxfp8")
        torch.cuda.synchronize()
        assert torch.equal(ro, total.to(dt)), alias
        ref.assert_quantised(data, scales, want, "mxfp8", slack=norm_slack(n))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_gpu_norm_special_rows(ct, dev, fmt):
    """a row of zeros (with and without eps), of one NaN, of an infinity (its block is NaN, the others are 0), of the largest values
    (whose squares overflow f32 for bf16: the norm is 0)"""
    n, b = 256, ref.BLOCK[fmt]
    x = normal((6, n), 4, dev, torch.bfloat16)
    x[0] = 0
    x[1, 70] = math.nan
    x[2, 70] = math.inf
    x[3] = torch.finfo(torch.bfloat16).max
    w = torch.ones(n, dtype=torch.bfloat16, device=dev)
    for eps in (1e-6, 0.0):
        data, scales = ref.buffers(6, n, fmt, dev)
        ct.rms_norm_quantize(x, w, whole(ct, data), whole(ct, scales), eps, fmt, 0.01 if fmt == "nvfp4" else 1.0)
        v = ref.values(data, scales, fmt, 0.01 if fmt == "nvfp4" else 1.0)
        assert bool((v[0] == 0).all()) if eps else bool(torch.isnan(v[0]).all())
        assert bool(torch.isnan(v[1]).all())
        at = slice(70 // b * b, 70 // b * b + b)
        assert bool(torch.isnan(v[2, at]).all()) and int(torch.isnan(v[2]).sum()) == b and float(torch.nan_to_num(v[2]).abs().max()) == 0
        assert bool((v[3] == 0).all())
        assert bool(torch.isfinite(v[4:]).all()) and float(v[4:].abs().min(-1).values.max()) >= 0 and float(v[4:].abs().max()) > 1


# ---- gated activation --------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_gpu_silu_mul(ct, dev, fmt, dtype, n):
    dt = TYPES[dtype]
    for rows, halves in ((1, True), (5, True), (19, False)):
        both = normal((rows, 2 * n), n + rows, dev, dt, 3.0)
        gate, up = (both[:, :n], both[:, n:]) if halves else (both[:, ::2], both[:, 1::2])
        x = gate.double()
        want = x / (1 + torch.exp(-x)) * up.double()
        g = g_of(want, fmt)
        data, scales = ref.buffers(rows, ref.padded(n, fmt), fmt, dev, extra_rows=1)
        ct.silu_mul_quantize(gate, up, whole(ct, data[:rows]), whole(ct, scales[:rows]), fmt, g)
        torch.cuda.synchronize()
        assert int((data[rows:] != 0xA5).sum() + (scales[rows:] != 0xA5).sum()) == 0
        g = torch.tensor(g, dtype=torch.float32).double().item()
        # exponential (2 steps), sum, quotient (2), product, each relative to the result at most; nvfp4's scale
        ref.assert_quantised(data[:rows], scales[:rows], want, fmt, g, slack=6 * 2.0 ** -24 + NVFP4_SLACK, tiny=2.0 ** -126)


@pytest.mark.gpu
def test_gpu_silu_mul_far_gates(ct, dev):
    """gates from -300 to 300: nothing overflows on the way; a NaN or an infinity takes its block"""
    gate = torch.linspace(-300, 300, 1024, device=dev).to(torch.bfloat16)[None].clone()
    up = normal((1, 1024), 6, dev, torch.bfloat16)
    gate[0, 512 + 5], up[0, 640 + 7], gate[0, 704 + 2] = math.nan, math.inf, -math.inf
    data, scales = ref.buffers(1, 1024, "mxfp8", dev)
    ct.silu_mul_quantize(gate, up, whole(ct, data), whole(ct, scales), "mxfp8")
    x = gate.double()
    want = x / (1 + torch.exp(-x)) * up.double()
    assert [int(i) for i in torch.nonzero(~torch.isfinite(want[0]))] == [517, 647, 706]
    ref.assert_quantised(data, scales, want, "mxfp8", slack=6 * 2.0 ** -24, tiny=2.0 ** -126)


# ---- every kernel by its name, where the size rule would take another ---------------------------------------------------------
def variants_of(ct, function, prefix):
    return [v.split(":")[1] for v in ct.kernel_list() if v.startswith(function + ":" + prefix)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n", [1, 257, 1024])
def test_gpu_norm_by_name(ct, dev, fmt, dtype, n):
    x, r, w = normal((13, n), n, dev, TYPES[dtype]), normal((13, n), n + 1, dev, TYPES[dtype]), normal((n,), n + 2, dev, TYPES[dtype])
    for function in ("rms_norm_quantize", "add_rms_norm_quantize"):
        names = variants_of(ct, function, fmt + "_" + dtype + "_")
        assert len(names) == 8
        c = x.double() + r.double() if function[0] == "a" else x.double()
        want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        g = g_of(want, fmt)
        for variant in names:
            if variant.endswith("w1v1") and n > 512:                      # holds 512 values
                continue
            data, scales = ref.buffers(13, ref.padded(n, fmt), fmt, dev)
            ro = torch.full_like(x, 7.0)
            args = (whole(ct, data), whole(ct, scales))
            if function[0] == "a":
                ct.add_rms_norm_quantize(r, x, w, *args, whole(ct, ro), 1e-6, fmt, g, variant=variant)
                assert torch.equal(ro, (x.float() + r.float()).to(x.dtype)), variant
            else:
                ct.rms_norm_quantize(x, w, *args, 1e-6, fmt, g, variant=variant)
            ref.assert_quantised(data, scales, want, fmt, torch.tensor(g, dtype=torch.float32).double().item(), slack=norm_slack(n) + NVFP4_SLACK)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gpu_units_by_name(ct, dev, fmt, dtype):
    """the three ways through a matrix give the same bytes, and the two ways back the same values"""
    base = normal((333, 417), 17, dev, TYPES[dtype])
    plain, column = base, base.t().contiguous().t()
    g = g_of(base, fmt)
    prefix = fmt + "_" + dtype + "_"
    results = [quantised(ct, x, fmt, None, g, variant=prefix + kind) for x, kind in ((plain, "rows"), (plain, "any"), (column, "columns"), (column, "any"), (column[:, :417], "columns"))]
    for data, scales in results[1:]:
        assert torch.equal(data, results[0][0]) and torch.equal(scales, results[0][1])
    ref.assert_quantised(*results[0], base.double(), fmt, g, slack=NVFP4_SLACK if fmt == "nvfp4" else 0.0)
    outs = [torch.full_like(base, 7.0) for _ in range(2)]
    for out, kind in zip(outs, ("rows", "any")):
        ct.block_dequantize(*results[0], whole(ct, out), fmt, g, variant=prefix + kind)
    assert torch.equal(outs[0], outs[1]) and bool(torch.isfinite(outs[0]).all())
    if dtype != "f32":
        up = normal(base.shape, 18, dev, base.dtype)
        got = []
        for kind in ("rows", "any"):
            data, scales = ref.buffers(333, ref.padded(417, fmt), fmt, dev)
            ct.silu_mul_quantize(base, up, whole(ct, data), whole(ct, scales), fmt, g, variant=prefix + kind)
            got.append((data, scales))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("image,entries", [("blockscale", 153), ("mxfp4", 6), ("mxfp4flat", 6)])
def test_lds_bytes_and_registers(fake_hip, image, entries):
    """LDS of the code objects is what the table says; no kernel of block-scaled rows spills"""
    import os
    import re
    import subprocess

    ct = fake_hip
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    notes = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--notes", os.path.join(root, "cutile-rs_amd", "lib", image + ".hsaco")],
                           stdout=subprocess.PIPE, text=True, check=True).stdout
    kernels = notes.split("- .agpr_count")[1:]
    assert len(kernels) == entries
    by_symbol = {}
    for kernel in kernels:
        symbol = re.search(r"\n    \.name: +(\S+)", kernel)[1]
        function, variant = symbol.split("_entry__")
        lds = int(re.search(r"\.group_segment_fixed_size: (\d+)", kernel)[1])
        assert ct.kernel_lookup(function, variant=variant.replace("_lone", "+lone")).lds_bytes == lds, symbol
        assert image != "blockscale" or int(re.search(r"\.vgpr_spill_count: (\d+)", kernel)[1]) == 0, symbol


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(3000, 480), (700, 4096), (90, 20000)])
def test_gpu_norm_rounds_the_value_itself(ct, dev, fmt, dtype, rows, n):
    """Next to a border between two codes or two scales f32 roundings decide wrongly: with two of them about one value in 2^21 (4 of the
    formats' steps against 2^-24), here of 1.4 to 2.9 million none: the norm is held to 2^-45"""
    x, r, w = normal((rows, n), 51, dev, TYPES[dtype]), normal((rows, n), 52, dev, TYPES[dtype], 3.0), (1 + 0.3 * normal((n,), 53, dev)).to(TYPES[dtype])
    c = (x.float() + r.float()).double()
    want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    k = ref.padded(n, fmt)
    data, scales = ref.buffers(rows, k, fmt, dev)
    ct.add_rms_norm_quantize(r, x, w, whole(ct, data), whole(ct, scales), whole(ct, torch.empty_like(x)), 1e-6, fmt)
    full = torch.zeros((rows, k), dtype=torch.float64, device=dev)
    full[:, :n] = want
    blocks = full.view(rows, k // 32, 32)
    exponents = ref._scale_codes(blocks.abs().amax(-1), fmt, 1.0)
    assert torch.equal(scales.long(), exponents)
    codes = ref.nearest(blocks / torch.exp2(exponents.double() - 127).unsqueeze(-1), ref.grid_of(fmt)).view(rows, k)
    assert torch.equal(codes, (ref.unpack(data, fmt) & (127 if fmt == "mxfp8" else 7)).long())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(3000, 480), (700, 4096), (90, 20001)])
def test_gpu_silu_mul_rounds_the_value_itself(ct, dev, fmt, dtype, rows, n):
    """as above; gates within 12 of 0, where the f32 result is within 32 steps, and some far above: their products with 1 are a power of two less a
    little, which f32 does not hold"""
    gate = normal((rows, n), 61, dev, torch.float32, 2.5).clamp(-11.9, 40.0).to(TYPES[dtype])
    up = normal((rows, n), 62, dev, TYPES[dtype])
    gate[:, 5], up[:, 5] = 16.0, 2.0
    gate[:, 70], up[:, 70] = 32.0, -4.0
    g = gate.double()
    want = g / (1 + torch.exp(-g)) * up.double()
    k = ref.padded(n, fmt)
    for view in (lambda t: t, lambda t: t.t().contiguous().t()):
        data, scales = ref.buffers(rows, k, fmt, dev)
        ct.silu_mul_quantize(view(gate), view(up), whole(ct, data), whole(ct, scales), fmt)
        full = torch.zeros((rows, k), dtype=torch.float64, device=dev)
        full[:, :n] = want
        blocks = full.view(rows, k // 32, 32)
        exponents = ref._scale_codes(blocks.abs().amax(-1), fmt, 1.0)
        assert torch.equal(scales.long(), exponents)
        codes = ref.nearest(blocks / torch.exp2(exponents.double() - 127).unsqueeze(-1), ref.grid_of(fmt)).view(rows, k)
        assert torch.equal(codes, (ref.unpack(data, fmt) & (127 if fmt == "mxfp8" else 7)).long())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("n", [32, 100, 5120])
def test_gpu_norm_of_equal_values(ct, dev, fmt, n):
    """rows of one value c each and eps = 0: the norm is w, wherever w lies - on a power of two (a border between scales), between two codes, above or below"""
    c = torch.tensor([3.0, 1.0, -0.375, 100.0, 3.3, -7.1, 1e-3, 250.0], device=dev)
    for w in (1.0, 2.0, 1.0625, 1.1875, 0.99609375, 5.0, 1.75):                         # (1.0625, 1.1875: halfway between two e4m3 codes)
        x = c.bfloat16()[:, None].expand(-1, n).contiguous()
        weights = torch.full((n,), w, dtype=torch.bfloat16, device=dev)
        for last in (1.0, 4.0):
            weights[0] = last * w
            want = torch.sign(x.double()) * weights.double()
            data, scales = ref.buffers(8, ref.padded(n, fmt), fmt, dev)
            ct.rms_norm_quantize(x, weights, whole(ct, data), whole(ct, scales), 0.0, fmt)
            ref.assert_quantised(data, scales, want, fmt)
            other = ref.buffers(8, ref.padded(n, fmt), fmt, dev)
            ct.rms_norm_quantize(x.t().contiguous().t(), weights, whole(ct, other[0]), whole(ct, other[1]), 0.0, fmt)
            assert torch.equal(other[0], data) and torch.equal(other[1], scales)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "nvfp4"])
@pytest.mark.parametrize("rows", [1, 70, 300])
def test_gpu_operands_of_the_products(ct, dev, fmt, rows):
    """norm -> product -> gated activation -> product on 8-bit, and on nvfp4 operands made here: each product is that of the values its bytes
    stand for, to what its own kernels are held to (1e-4 and 1e-5 of the norm in f32)"""
    hidden, inter, kh, ki = 500, 700, 512, 768
    dt = torch.bfloat16
    x, r, w = normal((rows, hidden), 71, dev, dt), normal((rows, hidden), 72, dev, dt), (1 + 0.3 * normal((hidden,), 73, dev)).to(dt)
    gate_up, down = normal((hidden, 2 * inter), 74, dev, dt, hidden ** -0.5).t(), normal((hidden, inter), 75, dev, dt, inter ** -0.5)

    def operand(count, k, make, g):
        data, scales = ref.buffers(count, k, fmt, dev)
        make(whole(ct, data), whole(ct, scales), g)
        return data, scales, ref.values(data, scales, fmt), torch.tensor(g, dtype=torch.float32).double().item()

    def product(a, b, out):
        run, alpha = (ct.linear_tile_mxfp8, 1.0) if fmt == "mxfp8" else (ct.linear_tile_nvfp4, a[3] * b[3])
        run(ct.partition(out, [128, 128]), a[0], b[0], a[1], b[1], alpha)
        want = alpha * (a[2] @ b[2].t())
        assert float((out.double() - want).norm() / want.norm()) <= (1e-4 if fmt == "mxfp8" else 1e-5)

    scale = lambda t: g_of(t, fmt)
    wa = operand(2 * inter, kh, lambda d, s, g: ct.block_quantize(gate_up, d, s, fmt, g), scale(gate_up))
    wd = operand(hidden, ki, lambda d, s, g: ct.block_quantize(down, d, s, fmt, g), scale(down))
    a = operand(rows, kh, lambda d, s, g: ct.add_rms_norm_quantize(r, x, w, d, s, whole(ct, r), 1e-6, fmt, g), 8.0 / (6 * 448) if fmt == "nvfp4" else 1.0)
    both = torch.zeros(rows, 2 * inter, device=dev)
    product(a, wa, both)
    half = both.to(dt)
    h = operand(rows, ki, lambda d, s, g: ct.silu_mul_quantize(half[:, :inter], half[:, inter:], d, s, fmt, g), 16.0 / (6 * 448) if fmt == "nvfp4" else 1.0)
    product(h, wd, torch.zeros(rows, hidden, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["rows", "any", "silu", "norm", "add_norm"])
def test_gpu_rows_padded_beyond_32_bit_columns(ct, dev, kind):
    """4-bit rows of more than 2^31 values, a short row in front of zeros: what lies behind the row is neither read nor, in residual_out, written"""
    k = (1 << 31) + 256
    n = 100
    data, scales = torch.full((1, k // 2), 0xA5, dtype=torch.uint8, device=dev), torch.full((1, k // 32), 0xA5, dtype=torch.uint8, device=dev)
    outs = whole(ct, data), whole(ct, scales)
    base = normal((2 * n, 4), 81, dev, torch.bfloat16)
    x = base[::2, 1:2].t()                                                   # a stride between the columns
    want = x.double()
    if kind == "rows":
        ct.block_quantize(x.contiguous(), *outs, "mxfp4", variant="mxfp4_bf16_rows")
    elif kind == "any":
        ct.block_quantize(x, *outs, "mxfp4", variant="mxfp4_bf16_any")
    elif kind == "silu":
        up = base[1::2, 2:3].t()
        want = want / (1 + torch.exp(-want)) * up.double()
        ct.silu_mul_quantize(x, up, *outs, "mxfp4", variant="mxfp4_bf16_any")
    else:
        w = torch.ones(n, dtype=torch.bfloat16, device=dev)
        around = torch.full((1, n + 2000), 7.0, dtype=torch.bfloat16, device=dev)
        if kind == "norm":
            ct.rms_norm_quantize(x, w, *outs, 1e-6, "mxfp4")
        else:
            r = base[1::2, 2:3].t()
            want = (x.float() + r.float()).double()
            ct.add_rms_norm_quantize(r, x, w, *outs, whole(ct, around[:, 1000:1000 + n]), 1e-6, "mxfp4")
            assert torch.equal(around[:, 1000:1000 + n], want.to(torch.bfloat16))
        want = want / torch.sqrt(want.square().mean(-1, keepdim=True) + 1e-6)
        assert bool((around[:, :1000] == 7.0).all()) and bool((around[:, 1000 + n:] == 7.0).all())
    assert ct.last_resolved()["variant"].endswith("_rows" if kind == "rows" else "_any")
    torch.cuda.synchronize()
    ref.assert_quantised(data[:, :64], scales[:, :4], want, "mxfp4", slack=32 * 2.0 ** -24 if kind in ("silu", "norm", "add_norm") else 0.0)
    assert int(torch.count_nonzero(data[:, 64:])) == 0 and int(torch.count_nonzero(scales[:, 4:])) == 0


def assert_codes_of(data, scales, want, fmt):
    """data and scales (mx formats) are the rounding of `want` itself, code by code"""
    rows, n = want.shape
    k = scales.shape[1] * 32
    full = torch.zeros((rows, k), dtype=torch.float64, device=want.device)
    full[:, :n] = want
    blocks = full.view(rows, k // 32, 32)
    exponents = ref._scale_codes(blocks.abs().amax(-1), fmt, 1.0)
    assert torch.equal(scales.long(), exponents), int((scales.long() != exponents).sum())
    codes = ref.nearest(blocks / torch.exp2(exponents.double() - 127).unsqueeze(-1), ref.grid_of(fmt)).view(rows, k)
    got = (ref.unpack(data, fmt) & (127 if fmt == "mxfp8" else 7)).long()
    assert torch.equal(codes, got), int((codes != got).sum())


def silu_steps(gate):
    """what an nvfp4 gated product is off by, relative: exponential twice 4 steps of 2^-24, products with it 2, sum 1, quotient 1, product 1, and for negative gates
    1.23 |g|, the rounding of the exponential's argument"""
    return (9 + 1.23 * float(gate.abs().max())) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sign", [-1, 1])
def test_gpu_silu_mul_of_every_gate(ct, dev, fmt, dtype, sign):
    """Every gate of the type from 1/2 to 84 of one sign, a row each, times every factor from 1 to 2, by both kernels: in the mx formats every code is the rounding of the
    product itself, next to borders (36 x 1.5 is 2^-52 below one) and however far below 0 the gate is; nvfp4 within its roundings of f32"""
    dt = TYPES[dtype]
    every = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dt)
    every = sign * every[(every >= 0.5) & (every <= 84)].to(dev)
    up = (1 + torch.arange(1 << (10 if dtype == "f16" else 7), device=dev) * torch.finfo(dt).eps).to(dt)
    gate, up = every[:, None].expand(-1, up.numel()).contiguous(), up[None].expand(every.numel(), -1).contiguous()
    x = gate.double()
    want = x / (1 + torch.exp(-x)) * up.double()
    rows, n = gate.shape
    g = 2.0 ** (-60 if sign < 0 else -6) if fmt == "nvfp4" else 1.0
    for view in (lambda t: t, lambda t: t.t().contiguous().t()):
        data, scales = ref.buffers(rows, n, fmt, dev)
        ct.silu_mul_quantize(view(gate), view(up), whole(ct, data), whole(ct, scales), fmt, g)
        if fmt == "nvfp4":
            ref.assert_quantised(data, scales, want, fmt, g, slack=silu_steps(gate) + NVFP4_SLACK)
        else:
            assert_codes_of(data, scales, want, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_gpu_silu_mul_of_far_gates_and_large_factors(ct, dev, fmt):
    """exp(g) below what f32 holds, times a factor that brings the product back: gates from -64 to -150, factors up to 2^127; beside them far positive gates"""
    rows, n = 300, 512
    gate = (-64 - 86 * torch.rand((rows, n), generator=torch.Generator().manual_seed(93))).to(dev).bfloat16()
    up = (torch.exp2(torch.floor(-gate.double() * 1.442) - 20).clamp(max=2.0 ** 126) * (1 + normal((rows, n), 94, dev).double().abs().clamp(max=0.99))).bfloat16()
    steps = silu_steps(gate)
    gate[:, 64:96] = 3e38
    up[:, 64:96] = 0.1
    x = gate.double()
    want = x / (1 + torch.exp(-x)) * up.double()
    for view in (lambda t: t, lambda t: t.t().contiguous().t()):
        data, scales = ref.buffers(rows, n, fmt, dev)
        ct.silu_mul_quantize(view(gate), view(up), whole(ct, data), whole(ct, scales), fmt, 2.0 ** -20 if fmt == "nvfp4" else 1.0)
        if fmt == "nvfp4":
            ref.assert_quantised(data, scales, want, fmt, 2.0 ** -20, slack=steps + NVFP4_SLACK)
        else:
            assert_codes_of(data, scales, want, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("add", [False, True])
def test_gpu_norm_of_small_rows(ct, dev, fmt, add):
    """eps = 0 and rows whose mean square f32 holds badly (below 2^-126) or not at all, down to rows of nothing but subnormals: an ordinary norm of about w, by every kernel"""
    exponents = [-40, -55, -62, -64, -70, -75, -90, -120, -126, -130, -132]
    n = 500
    x, r = (torch.stack([normal((n,), 100 * i + j, dev) * 2.0 ** e for j, e in enumerate(exponents)]).bfloat16() for i in (1, 2))
    w = (1 + 0.3 * normal((n,), 3, dev)).bfloat16()
    c = (x.float() + r.float()).double() if add else x.double()
    want = c / torch.sqrt(c.square().mean(-1, keepdim=True)) * w.double()
    k, g = 512, 2.0 ** -9 if fmt == "nvfp4" else 1.0
    function = "add_rms_norm_quantize" if add else "rms_norm_quantize"
    for variant in variants_of(ct, function, fmt + "_bf16_"):
        data, scales = ref.buffers(len(exponents), k, fmt, dev)
        if add:
            ct.add_rms_norm_quantize(r, x, w, whole(ct, data), whole(ct, scales), whole(ct, torch.empty_like(x)), 0.0, fmt, g, variant=variant)
        else:
            ct.rms_norm_quantize(x, w, whole(ct, data), whole(ct, scales), 0.0, fmt, g, variant=variant)
        if fmt == "nvfp4":
            ref.assert_quantised(data, scales, want, fmt, g, slack=2.0 ** -24 + NVFP4_SLACK)       # one rounding to f32
        else:
            assert_codes_of(data, scales, want, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("n", [5000, 32768, 40000, 262144])
def test_gpu_norm_of_equal_values_whose_squares_do_not_add_up(ct, dev, fmt, n):
    """as test_gpu_norm_of_equal_values, with c of 24 bits: sums of its squares are rounded (by 2^-47 of themselves and more where each thread adds a thousand), and the norm is w
    all the same - on a border between two codes or scales"""
    r = torch.tensor([1.0, -1.0, 1.5, 1.25, 1.0], device=dev).bfloat16()[:, None].expand(-1, n).contiguous()
    x = torch.tensor([2.0 ** -23, -2.0 ** -23, 2.0 ** -23, 1.5 * 2.0 ** -22, 2.0 ** -22], device=dev).bfloat16()[:, None].expand(-1, n).contiguous()
    k = ref.padded(n, fmt)
    for w in (1.0, 2.0, 1.0625, 1.1875, 2.5, 5.0, 1.75):
        weights = torch.full((n,), w, dtype=torch.bfloat16, device=dev)
        for last in (1.0, 4.0):
            weights[::32] = last * w
            want = torch.sign(r.double()) * weights.double()
            for view in (lambda t: t, lambda t: t.t().contiguous().t()):
                data, scales = ref.buffers(5, k, fmt, dev)
                ct.add_rms_norm_quantize(view(r), view(x), weights, whole(ct, data), whole(ct, scales), whole(ct, torch.empty_like(x)), 0.0, fmt)
                assert_codes_of(data, scales, want, fmt)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,strided", [(300, 4096, True), (60, 20001, True), (40, 40000, False), (12, 100003, True)])
def test_gpu_norm_of_any_rows_rounds_the_value_itself(ct, dev, fmt, dtype, rows, n, strided):
    """test_gpu_norm_rounds_the_value_itself where no kernel holds the row: strides, and more than 32768 values"""
    dt = TYPES[dtype]
    x, r, w = normal((rows, n), 55, dev, dt), normal((rows, n), 56, dev, dt, 3.0), (1 + 0.3 * normal((n,), 57, dev)).to(dt)
    c = (x.float() + r.float()).double()                                     # the sum is one of f32
    want = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    view = (lambda t: t.t().contiguous().t()) if strided else (lambda t: t)
    data, scales = ref.buffers(rows, ref.padded(n, fmt), fmt, dev)
    ct.add_rms_norm_quantize(view(r), view(x), w, whole(ct, data), whole(ct, scales), whole(ct, torch.empty_like(x)), 1e-6, fmt)
    assert ct.last_resolved()["variant"].endswith("_any")
    assert_codes_of(data, scales, want, fmt)
