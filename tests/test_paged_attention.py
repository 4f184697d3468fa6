"""paged_attention (paged_attention.hip): against 64 bits within a bound that counts its roundings, and the refusals."""
import pytest
import torch

import paged_ref as ref
from paged_ref import TYPES, Batch
from test_paged_cache import args, caches


def attend(ct, t, **o):
    v = {"out": t["new"].clone(), "vc": t["kc"], "ks": t["sc"], "vs": t["sc"], "tile": None, "grid": None, "window": 0, "max_new": 0, "max_context": 0, "workspace": None, "variant": None, "scale": 0.1, **t, **o}
    ct.paged_attention(v["new"], v["kc"], v["vc"], v["table"], v["starts"], v["lens"], ct.partition(v["out"], v["tile"] or [1, 1, v["out"].shape[-1]]), v["scale"], window=v["window"],
                       max_new=v["max_new"], max_context=v["max_context"], k_scales=v["ks"], v_scales=v["vs"], workspace=v["workspace"], grid=v["grid"], variant=v["variant"])


# ---- without a GPU --------------------------------------------------------------------------------------------------------
def test_refusals(fake_hip):
    ct = fake_hip
    t, m = args(), args(mx=True)
    z, half = torch.zeros, torch.half
    attend(ct, t), attend(ct, m), attend(ct, t, new=z(6, 6, 64, dtype=half), out=z(6, 6, 64, dtype=half), max_new=3)
    n0 = ct.lib().cutile_testing_launch_count()
    cases = [
        (lambda: attend(ct, t, new=z(6, 2, 64), out=z(6, 2, 64)), "must be f16 or bf16"),
        (lambda: attend(ct, t, new=z(6, 3, 64, dtype=half), out=z(6, 3, 64, dtype=half)), "3 query heads are no multiple of the cache's 2"),
        (lambda: attend(ct, t, new=z(6, 1, 64, dtype=half), out=z(6, 1, 64, dtype=half)), "no multiple"),
        (lambda: attend(ct, t, out=z(5, 2, 64, dtype=half)), "out must be q's shape"),
        (lambda: attend(ct, t, out=z(6, 2, 64).bfloat16()), "out must be q's shape"),
        (lambda: attend(ct, t, tile=[1, 1, 32]), "out must be q's shape"),
        (lambda: attend(ct, t, out=z(1, 2, 64, dtype=half).expand(6, 2, 64)), "elements of out overlap"),
        (lambda: attend(ct, t, out=z(6, 2, 68, dtype=half)[..., :64]), "aligned rows of out"),
        (lambda: attend(ct, t, new=z(6, 2, 68, dtype=half)[..., :64]), "aligned rows of q"),
        (lambda: attend(ct, t, new=z(6, 64, 2, dtype=half).transpose(1, 2)), "unit inner stride"),
        (lambda: attend(ct, t, window=-1), "must not be negative"),
        (lambda: attend(ct, t, max_new=-1), "must not be negative"),
        (lambda: attend(ct, t, max_context=-5), "must not be negative"),
        (lambda: attend(ct, t, scale=float("inf")), "finite number"),
        (lambda: attend(ct, t, scale=float("nan")), "finite number"),
        (lambda: attend(ct, t, workspace=z(1000)), "more than 16384 bytes"),
        (lambda: attend(ct, t, workspace=z(10000)[1:]), "16-byte aligned"),
        (lambda: attend(ct, t, workspace=z(20000)[::2]), "workspace must be contiguous"),
        (lambda: attend(ct, t, variant="f16_mxfp8_d64"), "does not fit these arguments"),
        (lambda: attend(ct, t, kc=t["kc"].bfloat16(), vc=t["kc"].bfloat16()), "of the rows' type"),
        (lambda: attend(ct, m, vs=None), "come together"),
        (lambda: attend(ct, args(d=32)), "D = 64, 128 or 256"),
        (lambda: attend(ct, t, starts=z(2, dtype=torch.int32)), "starts must be 3"),
        (lambda: attend(ct, t, grid=(5, 2, 1)), "grid"),
    ]
    for i, (fn, msg) in enumerate(cases):
        with pytest.raises(ct.CutileError, match=msg):
            fn()
            print("case", i, msg)
    assert ct.lib().cutile_testing_launch_count() == n0


def test_null_arguments_of_the_c_entry(fake_hip):
    import ctypes as C

    ct = fake_hip
    t = args()
    a = lambda x: C.pointer(ct.tensor_arg(x, None))
    f32, i32 = C.c_float, C.c_int32
    list_ = [a(t["new"]), a(t["kc"]), a(t["kc"]), None, None, a(t["table"]), a(t["starts"]), a(t["lens"]), C.pointer(ct.Partition(t["new"], [1, 1, 64], False, None).arg()), f32(0.1), i32(0), i32(0),
             i32(0), None]
    fn = ct.lib().cutile_launch_paged_attention
    assert fn(None, *list_, None) == 0
    for i, x in enumerate(list_):
        if x is not None and not isinstance(x, (C.c_float, C.c_int32)):
            assert fn(None, *[None if j == i else b for j, b in enumerate(list_)], None) == -2, i


@pytest.mark.parametrize("image,entries", [("pagedcache", 24), ("pagedattention", 32), ("logits", 9)])
def test_lds_bytes_and_registers(fake_hip, image, entries):
    """LDS of the code objects is what the table says"""
    import os
    import re
    import subprocess

    ct = fake_hip
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    notes = subprocess.run(["/opt/rocm/llvm/bin/llvm-readelf", "--notes", os.path.join(root, "cutile-rs_amd", "lib", image + ".hsaco")], stdout=subprocess.PIPE, text=True, check=True).stdout
    kernels = notes.split("- .agpr_count")[1:]
    assert len(kernels) == entries
    for kernel in kernels:
        symbol = re.search(r"\n    \.name: +(\S+)", kernel)[1]
        function, variant = symbol.split("_entry__")
        assert ct.kernel_lookup(function, variant=variant.replace("_few", "+few")).lds_bytes == int(re.search(r"\.group_segment_fixed_size: (\d+)", kernel)[1]), symbol


# ---- on a GPU ---------------------------------------------------------------------------------------------------------------
def problem(b, heads, group, d, dtype, mx, dev, layout="nhd"):
    """q, caches and scales on the device, and the caches' values in 64 bits"""
    q = b.normal(b.rows, heads * group, d).to(TYPES[dtype])
    k, v, scales = caches(b, heads, d, dtype, mx, dev, layout)
    real = []
    for cache, name in ((k, "k_scales"), (v, "v_scales")):
        x = b.normal(b.pages, b.page, heads, d).to(TYPES[dtype])
        if mx:
            data, byte = ref.quantized(x)
            cache.copy_(data)
            scales[name].copy_(byte)
            real.append(ref.values(data, byte))
        else:
            cache.copy_(x)
            real.append(x.double())
    return q, k, v, scales, real


def check(ct, dev, b, q, k, v, scales, real, d, window=0, scale=None, out=None, **kw):
    scale = d ** -0.5 if scale is None else scale
    qd = q.to(dev)
    out = torch.full_like(qd, 9.0) if out is None else out
    ct.paged_attention(qd, k, v, *b.where(dev), ct.partition(out, [1, 1, d]), scale, window=window, **scales, **kw)
    parts = ref.attention(b, q, *real, scale, window)
    tol = ref.bound(q.dtype, parts, d, max(max(b.held), 1))
    got, n = out.cpu().double(), sum(b.new)
    assert bool((got[n:] == 9.0).all()), "rows that are nobody's"
    off = (got[:n] - parts[0][:n]).abs()
    bad = ~(off <= tol[:n])
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}, worst {float((off / tol[:n]).nan_to_num(1e9).max()):.3g} of the bound"
    return out


SHAPES = [(2, 4, 64, 16, "nhd"), (1, 8, 128, 1, "hnd"), (2, 1, 128, 48, "both"), (1, 3, 256, 5, "nhd"), (3, 6, 64, 7, "hnd")]
BATCHES = [([1], [1]), ([1, 1, 1, 1], [7, 1, 300, 33]), ([5, 0, 1, 40, 0, 2], [5, 0, 17, 100, 3, 700]), ([3, 70], [2, 70]), ([130], [650]), ([1, 300, 4], [31, 300, 260])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("heads,group,d,page,layout", SHAPES)
@pytest.mark.parametrize("new,held", BATCHES)
def test_gpu_attention(ct, dev, dtype, mx, heads, group, d, page, layout, new, held):
    b = Batch(new, held, page, seed=d + group, rows=sum(new) + 3)
    check(ct, dev, b, *problem(b, heads, group, d, dtype, mx, dev, layout), d)


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("window", [1, 2, 31, 64, 100, 1000])
@pytest.mark.parametrize("group,d", [(4, 64), (1, 128), (2, 256)])
def test_gpu_sliding_window(ct, dev, mx, window, group, d):
    b = Batch([1, 6, 90, 200], [400, 333, 90, 500], 16, seed=window)
    check(ct, dev, b, *problem(b, 2, group, d, "f16", mx, dev), d, window=window, max_new=200, max_context=500)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 70])
def test_gpu_drafts_of_a_few_tokens(ct, dev, dtype, mx, d, window):
    """up to 32 rows to every sequence, behind short and long contexts; the same bits every time"""
    b = Batch([7, 3, 0, 1, 8], [2900, 30, 0, 700, 8], 16, seed=12, rows=21)
    p = problem(b, 2, 4, d, dtype, mx, dev)
    out = check(ct, dev, b, *p, d, window=window, max_new=8, max_context=2900)
    assert torch.equal(out, check(ct, dev, b, *p, d, window=window, max_new=8, max_context=2900))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{"max_new": 1, "max_context": 9000}, {"max_new": 1, "max_context": 1000}, {}, {"max_new": 1, "max_context": 2 ** 31 - 1}])
@pytest.mark.parametrize("mx", [False, True])
def test_gpu_keys_dealt_to_several_workgroups(ct, dev, kw, mx):
    """a few tokens behind long contexts, whatever is said of their length; the same bits every time"""
    b = Batch([1, 1, 1], [9000, 1, 4100], 16, seed=5)
    p = problem(b, 1, 5, 128, "bf16", mx, dev)
    out = check(ct, dev, b, *p, 128, **kw)
    for _ in range(3):
        assert torch.equal(out, check(ct, dev, b, *p, 128, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("new,held,group", [([150], [6000], 2), ([40, 1], [5000, 2000], 4), ([9], [4000], 8), ([300], [2500], 1)])
def test_gpu_keys_of_row_tiles_dealt_out(ct, dev, new, held, group):
    b = Batch(new, held, 32, seed=6)
    p = problem(b, 1, group, 128, "f16", False, dev)
    out = check(ct, dev, b, *p, 128, max_new=max(new), max_context=max(held))
    assert torch.equal(out, check(ct, dev, b, *p, 128, max_new=max(new), max_context=max(held)))


@pytest.mark.gpu
def test_gpu_workspace_of_the_callers(ct, dev):
    """any size of it gives the same within the bound, and it is left as it was found: zeros in front"""
    b = Batch([1, 2], [5000, 3000], 16, seed=7)
    p = problem(b, 2, 4, 128, "f16", True, dev)
    for size in (16384 + 16, 70000, 400000, ct.PAGED_ATTENTION_WORKSPACE_BYTES):
        ws = torch.zeros(size, dtype=torch.uint8, device=dev)
        for _ in range(2):
            check(ct, dev, b, *p, 128, workspace=ws, max_new=2, max_context=5000)
            assert int(ws[:16384].count_nonzero()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [True, False])
def test_gpu_captured(ct, dev, shared):
    """a graph replayed for other contents of q, the cache and the metadata, with eager work between, equals the eager launch that it is"""
    b = Batch([1, 1, 3], [700, 2000, 40], 16, seed=8)
    q, k, v, scales, real = problem(b, 2, 4, 128, "f16", False, dev)
    table, starts, lens = b.where(dev)
    qd, out, eager = q.to(dev), torch.zeros_like(q, device=dev), torch.zeros_like(q, device=dev)
    ws = torch.zeros(ct.PAGED_ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=dev) if shared else None
    launch = lambda o, **kw: ct.paged_attention(qd, k, v, table, starts, lens, ct.partition(o, [1, 4, 128]), 0.09, max_new=3, max_context=2000, workspace=ws, **kw)
    launch(out)
    torch.cuda.synchronize()
    g = ct.CapturedGraph().capture(lambda s: launch(out, stream=s))
    for i in range(4):
        qd.copy_(b.normal(*q.shape))
        lens.copy_(torch.tensor([700 - 300 * i if i < 2 else 1, 2000 - i, 40 + i]))
        out.fill_(5.0)
        torch.cuda.synchronize()
        g.launch()
        g.synchronize()
        launch(eager)
        torch.cuda.synchronize()
        if shared:
            assert torch.equal(out, eager)
        else:   # two orders of summation, each within its bound
            assert float((out.float() - eager.float()).abs().max()) <= 2 * 2.0 ** -11 * 4 + 1e-3
    g.close()


def unseen(ct, dev, dtype, mx, new, held, group, window, d, page):
    """NaN and infinities behind the context, in later tokens and in front of the window change nothing for the rows that do not see them; rows that do get what
    the definition gives"""
    b = Batch(new, held, page, seed=9)
    q, k, v, scales, real = problem(b, 2, group, d, dtype, mx, dev)
    first = check(ct, dev, b, q, k, v, scales, real, d, window)
    kinds = [float("nan")] if mx else [float("nan"), float("inf"), float("-inf")]
    table = b.table.long()
    poisoned = []
    for s, (n, h) in enumerate(zip(new, held)):
        last = int(table[s, (h - 1) // page])
        for r in range((h - 1) % page + 1, page):          # behind the context
            if mx:
                scales["v_scales"][last, r], scales["k_scales"][last, r] = 255, 255
            else:
                v[last, r], k[last, r] = float("nan"), float("inf")
        p = h - max(1, n // 3)                        # among the new tokens
        for i, kind in enumerate(kinds):
            at, r = int(table[s, (p + i) // page]), (p + i) % page
            if p + i >= h:
                continue
            if mx:
                scales["v_scales"][at, r, 1, 0] = 255
            else:
                v[at, r, 1, 3] = kind
            poisoned.append((s, p + i, kind))
    out = torch.full_like(first, 9.0)
    ct.paged_attention(q.to(dev), k, v, *b.where(dev), ct.partition(out, [1, 1, d]), d ** -0.5, window=window, **scales)
    out, first = out.cpu(), first.cpu()
    rows = {}
    for row, s, p, _, _ in b.places():
        for ps, pp, kind in poisoned:
            if ps == s and pp <= p and (not window or pp > p - window):
                rows.setdefault(row, []).append(kind)
    cols = slice(0, 32) if mx else slice(3, 4)
    for row in range(sum(new)):
        hit = rows.get(row, [])
        want, got = first[row], out[row]
        spoilt = torch.zeros(want.shape, dtype=torch.bool)
        spoilt[group:, cols] = bool(hit)
        # (a poisoned step's products are added up in another order: twice the bound of one)
        assert bool(((got.double() - want.double()).abs() <= 2 * 2.0 ** -8 * 4)[~spoilt].all()), row
        if hit:
            inf = {float("inf"), float("-inf")}
            kind = "nan" if set(hit) - inf or inf <= set(hit) else hit[0]
            assert bool(got[group:, cols].isnan().all()) if kind == "nan" else bool((got[group:, cols] == kind).all()), (row, hit)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("new,held,group,window", [([40], [40], 2, 0), ([200], [300], 1, 0), ([5], [120], 4, 0), ([64], [200], 8, 50), ([3, 100], [70, 100], 1, 33)])
def test_gpu_what_a_row_does_not_see(ct, dev, dtype, mx, new, held, group, window):
    unseen(ct, dev, dtype, mx, new, held, group, window, 64, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("new,held,group,window,d,page", [([300], [300], 1, 0, 128, 16), ([100], [700], 8, 0, 128, 16), ([200], [900], 2, 333, 128, 16), ([200], [900], 2, 333, 128, 7),
                                                          ([200], [900], 2, 333, 64, 16), ([130], [700], 2, 90, 256, 16), ([130], [700], 2, 90, 256, 7), ([9], [600], 1, 100, 256, 16), ([8], [300], 4, 100, 128, 16),
                                                          ([30], [300], 1, 40, 64, 7)])
def test_gpu_what_a_row_of_a_larger_tile_does_not_see(ct, dev, mx, new, held, group, window, d, page):
    unseen(ct, dev, "f16", mx, new, held, group, window, d, page)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_gpu_every_value_of_an_mxfp8_cache(ct, dev, dtype):
    """one key for each of 256 scales: the output is its V, all 256 codes, rounded once"""
    codes = torch.arange(256, dtype=torch.uint8).reshape(1, 1, 1, 256).repeat(256, 1, 1, 1)
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1, 1, 1).repeat(1, 1, 1, 8)
    want = ref.values(codes, scales).to(TYPES[dtype]).reshape(256, 1, 256)
    one = torch.ones(256, dtype=torch.int32, device=dev)
    table, starts = torch.arange(256, dtype=torch.int32, device=dev).reshape(256, 1), torch.arange(257, dtype=torch.int32, device=dev)
    q = torch.zeros((256, 1, 256), dtype=TYPES[dtype], device=dev)
    out = torch.zeros_like(q)
    ct.paged_attention(q, torch.zeros_like(codes).to(dev), codes.to(dev), table, starts, one, ct.partition(out, [1, 1, 256]), 1.0, max_new=1, max_context=1,
                       k_scales=torch.full_like(scales, 127).to(dev), v_scales=scales.to(dev))
    got = out.cpu()
    assert torch.equal(got.isnan(), want.isnan() | ~want.isfinite() & got.isnan())
    fine = want.isfinite()
    assert torch.equal(got[fine], want[fine])


@pytest.mark.gpu
def test_gpu_metadata_that_names_no_place(ct, dev):
    """pages that the cache lacks are zeros (a score of 0 each), lengths beyond the table end there, starts beyond the rows are cut"""
    for mx in (False, True):
        b = Batch([2, 2, 2], [40, 40, 64], 16, spare=0, table_pages=4, seed=10)
        b.table[0, 1], b.table[1, 0] = -1, b.pages + 7
        p = problem(b, 1, 4, 64, "f16", mx, dev)
        check(ct, dev, b, *p, 64)
        table, starts, lens = b.where(dev)
        q, out = p[0].to(dev), torch.full_like(p[0], 9.0).to(dev)
        starts[3], lens[2], starts[0] = 1000, 2 ** 31 - 1, -5
        ct.paged_attention(q, p[1], p[2], table, starts, lens, ct.partition(out, [1, 1, 64]), 0.125, **p[3])
        assert bool(out.isfinite().all()) and bool((out != 9.0).all())
        starts.copy_(torch.tensor([0, 6, 2, 4]))           # falling: anything finite, in bounds
        ct.paged_attention(q, p[1], p[2], table, starts, lens, ct.partition(out, [1, 1, 64]), 0.125, **p[3])
        torch.cuda.synchronize()
        assert bool(out.isfinite().all())


@pytest.mark.gpu
def test_gpu_many_sequences(ct, dev):
    for n, d in ((70, 64), (1000, 64)):
        new = [(i * 7 + i // 3) % 3 for i in range(n)]
        b = Batch(new, [x + i % 40 for i, x in enumerate(new)], 4, seed=n)
        check(ct, dev, b, *problem(b, 1, 2, d, "bf16", False, dev), d)
    new = [100 if i % 10 == 0 else 1 for i in range(80)]
    b = Batch(new, [x + i for i, x in enumerate(new)], 8, seed=3)
    check(ct, dev, b, *problem(b, 1, 4, 64, "f16", True, dev), 64, max_new=100)


@pytest.mark.gpu
def test_gpu_offsets_beyond_32_bits(ct, dev):
    pages, page, heads, d = 3 * 2 ** 12, 64, 16, 256
    b = Batch([3], [100], page)
    k = torch.empty((pages, page, heads, d), dtype=torch.half, device=dev)
    v = torch.empty_like(k)
    small = torch.randn(2, 2, page, heads, d).half()
    k[pages - 2:], v[pages - 2:] = small[0].to(dev), small[1].to(dev)
    q = b.normal(3, heads, d).half()
    out = torch.zeros_like(q, device=dev)
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=dev)
    ct.paged_attention(q.to(dev), k, v, table, *b.where(dev)[1:], ct.partition(out, [1, 1, d]), d ** -0.5)
    b.table, b.pages = torch.tensor([[0, 1]], dtype=torch.int32), 2
    parts = ref.attention(b, q, small[0].double(), small[1].double(), d ** -0.5)
    assert bool(((out.cpu().double() - parts[0]).abs() <= ref.bound(torch.half, parts, d, 100)).all())


@pytest.mark.gpu
def test_gpu_streams_strides_and_scores(ct, dev):
    """q and out inside wider tensors, on a stream of the caller's; scores of both signs, large, and all alike"""
    b = Batch([7, 1, 50], [300, 900, 50], 16, seed=11)
    q, k, v, scales, real = problem(b, 2, 4, 64, "bf16", False, dev)
    wide = torch.zeros((58, 3, 8, 64), dtype=torch.bfloat16, device=dev)
    wide[:, 1] = q.to(dev)
    out = torch.full((58, 8, 128), 9.0, dtype=torch.bfloat16, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for scale in (0.125, -0.125, 2.0, 0.0):
        with torch.cuda.stream(s):
            ct.paged_attention(wide[:, 1], k, v, *b.where(dev), ct.partition(out[..., 64:], [1, 1, 64]), scale)
        s.synchronize()
        parts = ref.attention(b, q, *real, scale)
        ok = bool(((out[..., 64:].cpu().double() - parts[0]).abs() <= ref.bound(q.dtype, parts, 64, 900)).all())
        assert ok, scale
        assert bool((out[..., :64] == 9.0).all())
