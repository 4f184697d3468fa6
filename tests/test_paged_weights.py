"""paged_attention on softmax weights far below the largest one: many keys of small weight in front of one that outweighs each of them."""
import math

import pytest
import torch

import paged_ref as ref
from paged_ref import TYPES, Batch
from test_paged_attention import attend
from test_paged_cache import args, caches

LIFT = 11   # f16 weights are held 2^11 times what they are against the row's reference point (paged_attention.hip)


def bound(dtype, parts, d, keys):
    """How far an output may be off, with u = half a step in the type (relative, 2^-11 f16, 2^-8 bf16).  The output is rounded once, u |o| and, in f16, half its least
    step, 2^-25.  The weights are rounded and their sum is that of the rounded ones, so that a relative error e of every weight moves o by e sum(w |v - o|) <= e (near + |o|):
    u of the rounding; (d + 2) 2^-24 of the scores' magnitude twice (a key's and the reference point's); 2^-21 of the exponential and (keys / 16 + 64) 2^-24 of the sums.  An f16
    weight below the type's normal range is off by half of its least step instead: 2^-25 / 2^LIFT of the row's reference point, which is the largest weight or less: every
    key moves o by that times |v - o| at most, |v| summed is `far`."""
    out, near, far, reach = parts
    half = dtype == torch.float16
    u = 2.0 ** -11 if half else 2.0 ** -8
    e = u + 2 * reach * (d + 2) * 2.0 ** -24 + 2.0 ** -21 + (keys / 16 + 64) * 2.0 ** -24
    tol = u * out.abs() + e.unsqueeze(-1) * (near + out.abs()) * (1 + u)
    return tol + (2.0 ** -(25 + LIFT) * (far + keys * out.abs()) + 2.0 ** -25 if half else 1e-38)


def one_key_above_many(ct, dev, dtype, mx, d, new, held, at, gap, group=1, page=16, **kw):
    """the key at position `at` has a score of `gap` (log2) above the others', whose scores are all 0, and values of 0; the second head of a group half of it"""
    b = Batch([new], [held], page, seed=held + d)
    q = torch.zeros(new, group, d, dtype=TYPES[dtype])
    q[:, :, 1] = 4.0 / torch.arange(1, group + 1)
    k, v, scales = caches(b, 1, d, dtype, mx, dev)
    kx, vx = torch.zeros(b.pages, page, 1, d), 1.0 + b.normal(b.pages, page, 1, d)
    place = (int(b.table[0, at // page]), at % page)
    kx[place][0, 1] = 4.0
    vx[place] = 0.0
    real = []
    for cache, name, x in ((k, "k_scales", kx), (v, "v_scales", vx)):
        x = x.to(TYPES[dtype])
        if mx:
            data, byte = ref.quantized(x)
            cache.copy_(data)
            scales[name].copy_(byte)
            real.append(ref.values(data, byte))
        else:
            cache.copy_(x)
            real.append(x.double())
    scale = gap * math.log(2.0) / 16
    out = torch.full_like(q, 9.0).to(dev)
    ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), scale, **scales, **kw)
    parts = ref.attention(b, q, *real, float(torch.tensor(scale, dtype=torch.float32)))
    off = (out.cpu().double() - parts[0]).abs() / bound(q.dtype, parts, d, held)
    assert bool((off <= 1.0).all()), f"worst {float(off.nan_to_num(1e9).max()):.3g} of the bound; {float((out.cpu().double() / parts[0]).mean()):.4f} of the result"
    return out


# ---- without a GPU --------------------------------------------------------------------------------------------------------
def test_scales_that_f32_does_not_hold(fake_hip):
    """scores are taken in units of log 2: the scale times 1.4427 has to be a number of f32 as well"""
    ct, t = fake_hip, args()
    n0 = ct.lib().cutile_testing_launch_count()
    for scale in (2.4e38, -2.4e38, 3.4e38, float("inf"), float("nan")):
        with pytest.raises(ct.CutileError, match="finite number"):
            attend(ct, t, scale=scale)
    assert ct.lib().cutile_testing_launch_count() == n0
    for scale in (2.3e38, -2.3e38, 1e-45, 0.0):
        attend(ct, t, scale=scale)
    assert ct.lib().cutile_testing_launch_count() == n0 + 4


# ---- on a GPU ---------------------------------------------------------------------------------------------------------------
GAPS = [12.0, 15.0, 17.4, 17.6, 20.3, 22.0, 22.6, 24.5, 26.0, 30.0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,mx", [("f16", False), ("f16", True), ("bf16", False)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("gap", GAPS)
def test_gpu_one_key_above_many_others(ct, dev, dtype, mx, d, shared, gap):
    """a single token behind 40000 keys, shared by workgroups or (a workspace without room) walked by one"""
    ws = None if shared else torch.zeros(16384 + 16, dtype=torch.uint8, device=dev)
    for at in (0, 20011):
        one_key_above_many(ct, dev, dtype, mx, d, 1, 40000, at, gap, group=2, max_new=1, max_context=40000, workspace=ws)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,mx", [("f16", False), ("f16", True), ("bf16", False)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("gap", [15.0, 17.6, 20.3, 22.6, 24.5, 30.0])
def test_gpu_one_key_above_many_others_in_a_chunk(ct, dev, dtype, mx, d, gap):
    one_key_above_many(ct, dev, dtype, mx, d, 150, 6000, 100, gap, max_new=150, max_context=6000)
    one_key_above_many(ct, dev, dtype, mx, d, 20, 3000, 2000, gap, group=1, max_new=20, max_context=3000)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rise", [0.2, 1.0, 3.9, 4.1, 7.9, 8.1])
def test_gpu_scores_that_rise_from_key_to_key(ct, dev, d, rise):
    """every block of 32 keys has scores `rise` (log2) above those of the last, so that the reference point lags behind as far as it may: finite, and right"""
    held = 1600
    b = Batch([1], [held], 16, seed=d)
    q = torch.zeros(1, 1, d).half()
    q[..., 0] = 1.0
    k, v, _ = caches(b, 1, d, "f16", False, dev)
    kx, vx = torch.zeros(b.pages, 16, 1, d), b.normal(b.pages, 16, 1, d).half()
    p = torch.arange(held)
    kx[b.table[0].long()[p // 16], p % 16, 0, 0] = (p // 32).float()
    k.copy_(kx.half()), v.copy_(vx)
    for sign in (1.0, -1.0):
        scale = sign * rise * math.log(2.0)
        out = torch.full_like(q, 9.0).to(dev)
        for ws in (None, torch.zeros(16384 + 16, dtype=torch.uint8, device=dev)):
            ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), scale, max_new=1, max_context=held, workspace=ws)
            parts = ref.attention(b, q, kx.half().double(), vx.double(), float(torch.tensor(scale, dtype=torch.float32)))
            off = (out.cpu().double() - parts[0]).abs() / bound(q.dtype, parts, d, held)
            assert bool((off <= 1.0).all()), float(off.nan_to_num(1e9).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("log_score", [16, 20, 23, 24, 25])
def test_gpu_scores_of_any_magnitude(ct, dev, dtype, d, log_score):
    """scores of 2^16 to 2^25 (log2 units), all alike or rising by a little from block to block: what f32 leaves of their differences decides, but every output is a mean of values"""
    held = 640
    b = Batch([40, 1], [held, held], 16, seed=d)
    q = torch.zeros(41, 1, d).to(TYPES[dtype])
    q[..., 0], q[..., 1] = 1024.0, 1.0
    k, v, _ = caches(b, 1, d, dtype, False, dev)
    kx, vx = torch.zeros(b.pages, 16, 1, d), (2.0 + b.normal(b.pages, 16, 1, d).clamp(-1, 1)).to(TYPES[dtype])
    v.copy_(vx)
    p = torch.arange(held)
    for i, rise in enumerate([0.0] + [0.25, 0.125, 0.0625, 0.03125] * 4):
        kx[..., 0] = 1024.0
        for s in range(2):
            kx[b.table[s].long()[p // 16], p % 16, 0, 1] = (p // 32).float() * rise
        k.copy_(kx.to(TYPES[dtype]))
        for sign in (1.0, -1.0):
            scale = sign * math.log(2.0) * 2.0 ** (log_score - 20) * (1 + i / 17)
            out = torch.full_like(q, 9.0).to(dev)
            ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), scale, max_new=40, max_context=held)
            got = out.cpu().double()
            assert bool(((got >= 1.0 - 2.0 ** -8) & (got <= 3.0 + 3 * 2.0 ** -8)).all()), (rise, scale, got.min(), got.max())
            if rise == 0.0:   # equal scores, whatever they are rounded to: the mean, with weights of no error but that of f32 sums
                for row, s, at, _, _ in b.places():
                    mean = vx[b.table[s].long()[p[:at + 1] // 16], p[:at + 1] % 16, 0].double().mean(0)
                    u = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
                    assert bool(((got[row, 0] - mean).abs() <= u * mean + (held / 16 + 64) * 2.0 ** -24 * 3).all()), (row, scale)
