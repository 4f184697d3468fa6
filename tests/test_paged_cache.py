"""paged_cache_write and paged_cache_read (paged_cache.hip): every byte of the cache against the definition, and the refusals."""
import pytest
import torch

import paged_ref as ref
from paged_ref import TYPES, Batch

FLAT = [(dt, mx) for dt in ("f16", "bf16") for mx in (False, True)]


def caches(batch, heads, d, dtype, mx, dev, layout="nhd"):
    """caches and scales [pages, page, heads, ...], filled with a pattern that is no result"""
    def make(width, kind):
        shape = (batch.pages, batch.page, heads, width)
        if layout == "hnd":      # pages of [heads, page, D]
            return torch.full((shape[0], heads, batch.page, width), 0x5A, dtype=torch.uint8).to(dev).view(kind).permute(0, 2, 1, 3) if kind == torch.uint8 else \
                torch.full((shape[0], heads, batch.page, width), 3.25, dtype=kind, device=dev).permute(0, 2, 1, 3)
        if layout == "both":     # K and V of a page side by side: strides over twice a page
            both = torch.full((shape[0], 2, *shape[1:]), 0x5A if kind == torch.uint8 else 3.25, dtype=kind, device=dev)
            return both[:, 1]
        return torch.full(shape, 0x5A if kind == torch.uint8 else 3.25, dtype=kind, device=dev)
    if not mx:
        return make(d, TYPES[dtype]), make(d, TYPES[dtype]), {}
    return make(d, torch.uint8), make(d, torch.uint8), {"k_scales": make(d // 32, torch.uint8), "v_scales": make(d // 32, torch.uint8)}


def args(rows=6, heads=2, d=64, page=16, pages=5, dtype=torch.float16, mx=False):
    """small tensors on the CPU for launches that nothing runs"""
    t = {"new": torch.zeros(rows, heads, d, dtype=dtype), "kc": torch.zeros(pages, page, heads, d, dtype=torch.uint8 if mx else dtype), "table": torch.zeros(2, 4, dtype=torch.int32),
         "starts": torch.zeros(3, dtype=torch.int32), "lens": torch.zeros(2, dtype=torch.int32)}
    t["sc"] = torch.zeros(pages, page, heads, d // 32, dtype=torch.uint8) if mx else None
    return t


def write(ct, t, **o):
    v = {"new_v": t["new"], "vc": t["kc"].clone(), "ks": t["sc"], "vs": t["sc"] if t["sc"] is None else t["sc"].clone(), "variant": None, **t, **o}
    ct.paged_cache_write(v["new"], v["new_v"], v["kc"], v["vc"], v["table"], v["starts"], v["lens"], k_scales=v["ks"], v_scales=v["vs"], variant=v["variant"])


def read(ct, t, **o):
    v = {"out_v": t["new"].clone(), "vc": t["kc"], "ks": t["sc"], "vs": t["sc"], "tile": None, "grid": None, **t, **o}
    tile = v["tile"] or [1, *v["new"].shape[1:]]
    ct.paged_cache_read(v["kc"], v["vc"], v["table"], v["starts"], v["lens"], ct.partition(v["new"], tile), ct.partition(v["out_v"], tile), k_scales=v["ks"], v_scales=v["vs"], grid=v["grid"])


# ---- without a GPU --------------------------------------------------------------------------------------------------------
def test_refusals(fake_hip):
    ct = fake_hip
    n0 = ct.lib().cutile_testing_launch_count()
    t, m = args(), args(mx=True)
    z = torch.zeros
    half = torch.half
    odd = z(5, 16, 2, 72, dtype=half)[..., 1:65]
    cases = [
        (lambda f: f(t, new=z(6, 2, 64)), "must be f16 or bf16"),
        (lambda f: f(t, kc=t["kc"].bfloat16(), vc=t["kc"].bfloat16()), "of the rows' type f16"),
        (lambda f: f(t, vc=t["kc"].bfloat16()), "of the rows' type f16"),
        (lambda f: f(m, ks=None), "come together"),
        (lambda f: f(m, vs=None), "come together"),
        (lambda f: f(t, ks=m["sc"], vs=m["sc"]), "tensors of bytes"),
        (lambda f: f(m, ks=m["sc"].float(), vs=m["sc"].float()), "tensors of bytes"),
        (lambda f: f(m, ks=m["sc"][..., :1], vs=m["sc"][..., :1]), "scales must be"),
        (lambda f: f(m, ks=m["sc"][:4], vs=m["sc"][:4]), "scales must be"),
        (lambda f: f(m, ks=m["sc"].permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)), "unit inner stride"),
        (lambda f: f(m, ks=z(5, 2, 16, 2, dtype=torch.uint8).permute(0, 2, 1, 3)), "laid out alike"),
        (lambda f: f(t, vc=z(5, 2, 16, 64, dtype=half).permute(0, 2, 1, 3)), "laid out alike"),
        (lambda f: f(t, kc=odd, vc=odd), "16-byte aligned rows of k_cache"),
        (lambda f: f(t, kc=z(5, 16, 2, 128, dtype=half)[..., ::2], vc=z(5, 16, 2, 128, dtype=half)[..., ::2]), "unit inner stride"),
        (lambda f: f(t, vc=z(4, 16, 2, 64, dtype=half)), "must have one shape"),
        (lambda f: f(t, new=z(6, 2, 128, dtype=half)), "that of the rows"),
        (lambda f: f(args(d=96)), "D = 64, 128 or 256, got 96"),
        (lambda f: f(t, kc=z(5, 16, 128, dtype=half)), "expected rank 4"),
        (lambda f: f(t, new=z(6, 128, dtype=half)), "rank"),
        (lambda f: f(t, new=z(0, 2, 64, dtype=half)), "must be positive"),
        (lambda f: f(t, table=z(2, 4)), "page_table must be"),
        (lambda f: f(t, table=z(4, 2, dtype=torch.int32).t()), "page_table must be"),
        (lambda f: f(t, table=z(2, 0, dtype=torch.int32)), "must be positive"),
        (lambda f: f(t, starts=z(2, dtype=torch.int32)), "starts must be 3"),
        (lambda f: f(t, starts=z(3, dtype=torch.int64)), "starts must be"),
        (lambda f: f(t, starts=z(6, dtype=torch.int32)[::2]), "starts must be"),
        (lambda f: f(t, lens=z(1, dtype=torch.int32)), "context_lens must be 2"),
        (lambda f: f(t, lens=z(2, dtype=torch.int64)), "context_lens must be"),
        (lambda f: f(m, kc=torch.empty(2 ** 31 + 4096, dtype=torch.uint8).as_strided((2, 16, 2, 64), (2 ** 31, 128, 64, 1))), "below 2\\^31"),   # (never touched)
    ]
    only_write = [
        (lambda f: f(t, new_v=z(5, 2, 64, dtype=half)), "must be \\[tokens, 2, 64\\]"),
        (lambda f: f(t, new_v=t["new"].bfloat16()), "must be \\[tokens, 2, 64\\]"),
        (lambda f: f(t, new=z(6, 4, 64, dtype=half), new_v=z(6, 4, 64, dtype=half)), "must be \\[tokens, 2, 64\\]"),
        (lambda f: f(t, new=z(6, 2, 68, dtype=half)[..., :64]), "aligned rows of new_k"),
        (lambda f: f(t, kc=z(1, 16, 2, 64, dtype=half).expand(5, 16, 2, 64), vc=z(1, 16, 2, 64, dtype=half).expand(5, 16, 2, 64)), "elements of k_cache overlap"),
        (lambda f: f(m, ks=z(1, 16, 2, 2, dtype=torch.uint8).expand(5, 16, 2, 2), vs=z(1, 16, 2, 2, dtype=torch.uint8).expand(5, 16, 2, 2)), "elements of k_scales overlap"),
        (lambda f: f(t, variant="f16_d128"), "does not fit these arguments"),
    ]
    only_read = [
        (lambda f: f(t, out_v=z(5, 2, 64, dtype=half)), "must be \\[tokens, 2, 64\\]|differ"),
        (lambda f: f(t, tile=[1, 1, 64]), "partitioned"),
        (lambda f: f(t, tile=[1, 2, 32]), "partitioned"),
        (lambda f: f(t, out_v=z(1, 2, 64, dtype=half).expand(6, 2, 64)), "elements of out_v overlap"),
        (lambda f: f(t, out_v=z(6, 2, 68, dtype=half)[..., :64]), "aligned rows of out_v"),
        (lambda f: f(t, grid=(5, 1, 1)), "grid"),
    ]
    for op, listed in ((write, cases + only_write), (read, cases + only_read)):
        for i, (case, msg) in enumerate(listed):
            with pytest.raises(ct.CutileError, match=msg):
                case(lambda *a, **k: op(ct, *a, **k))
                print(op.__name__, "case", i, msg)
    assert ct.lib().cutile_testing_launch_count() == n0
    write(ct, t), write(ct, m), read(ct, t), read(ct, m)
    read(ct, t, kc=z(1, 16, 2, 64, dtype=half).expand(5, 16, 2, 64), vc=z(1, 16, 2, 64, dtype=half).expand(5, 16, 2, 64))   # reading may share
    assert ct.lib().cutile_testing_launch_count() == n0 + 5


def test_null_arguments_of_the_c_entries(fake_hip):
    """every pointer of the C entries that must not be null may be so by mistake: an error, not a fault"""
    import ctypes as C

    ct = fake_hip
    t = args()
    a = lambda x: C.pointer(ct.tensor_arg(x, None))
    part = lambda x: C.pointer(ct.Partition(x, [1, *x.shape[1:]], False, None).arg())
    calls = {
        "paged_cache_write": [a(t["new"]), a(t["new"]), a(t["kc"]), a(t["kc"]), None, None, a(t["table"]), a(t["starts"]), a(t["lens"])],
        "paged_cache_read": [a(t["kc"]), a(t["kc"]), None, None, a(t["table"]), a(t["starts"]), a(t["lens"]), part(t["new"]), part(t["new"])],
    }
    for name, list_ in calls.items():
        fn = getattr(ct.lib(), "cutile_launch_" + name)
        assert fn(None, *list_, None) == 0, name
        for i, x in enumerate(list_):
            if x is not None:
                assert fn(None, *[None if j == i else b for j, b in enumerate(list_)], None) == -2, (name, i)


# ---- on a GPU ---------------------------------------------------------------------------------------------------------------
# (new tokens, tokens in all): nothing new, nothing at all, one token of each, chunks over page borders, a position before 0
BATCHES = [([1], [1]), ([1, 1, 1], [7, 1, 300]), ([5, 0, 1, 40, 0], [5, 0, 17, 100, 3]), ([3, 70], [2, 70])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,mx", FLAT)
@pytest.mark.parametrize("heads,d,page,layout", [(2, 64, 16, "nhd"), (8, 128, 1, "hnd"), (1, 256, 5, "both"), (3, 128, 48, "nhd")])
@pytest.mark.parametrize("new,held", BATCHES)
def test_gpu_write_and_read(ct, dev, dtype, mx, heads, d, page, layout, new, held):
    """the places of the batch's tokens hold them, every other byte of the cache stays, and read gives them back"""
    b = Batch(new, held, page, seed=heads + page, rows=sum(new) + 2)
    qkv = b.normal(b.rows, heads, 3, d, std=2.0).to(TYPES[dtype])
    new_k, new_v = qkv[:, :, 1], qkv[:, :, 2]           # strided
    k, v, scales = caches(b, heads, d, dtype, mx, dev, layout)
    want = [x.cpu().clone() for x in (k, v, *scales.values())]
    ct.paged_cache_write(qkv.to(dev)[:, :, 1], qkv.to(dev)[:, :, 2], k, v, *b.where(dev), **scales)
    back_k, back_v = torch.full((b.rows, heads, d), 9.0), torch.full((b.rows, heads, d), 9.0)
    for row, _, _, at, r in b.places():
        back_k[row], back_v[row] = 0.0, 0.0
        if at < 0:
            continue
        for x, to, s_to, back in ((new_k, want[0], 2, back_k), (new_v, want[1], 3, back_v)):
            if mx:
                data, byte = ref.quantized(x[row])
                to[at, r], want[s_to][at, r] = data, byte
                back[row] = ref.values(data, byte).to(TYPES[dtype]).float()
            else:
                to[at, r] = x[row]
                back[row] = x[row].float()
    for got, w in zip((k, v, *scales.values()), want):
        assert torch.equal(got.cpu().view(torch.uint8) if mx else got.cpu(), w)
    out = torch.full((2, b.rows, heads, d), 9.0, dtype=TYPES[dtype], device=dev)
    ct.paged_cache_read(k, v, *b.where(dev), ct.partition(out[0], [4, heads, d]), ct.partition(out[1], [4, heads, d]), **scales)
    assert torch.equal(out[0].cpu().float(), back_k) and torch.equal(out[1].cpu().float(), back_v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_gpu_every_value_of_an_mxfp8_cache(ct, dev, dtype):
    """all 256 codes under all 256 scales, rounded once"""
    codes = torch.arange(256, dtype=torch.uint8).reshape(1, 1, 1, 256).repeat(256, 1, 1, 1)
    scales = torch.arange(256, dtype=torch.uint8).reshape(256, 1, 1, 1).repeat(1, 1, 1, 8)
    want = ref.values(codes, scales).to(TYPES[dtype]).reshape(256, 1, 256)
    # through f32, as the kernel goes, is no second rounding: 4 significant bits are exact in f32 down to its subnormals
    table = torch.arange(256, dtype=torch.int32).reshape(1, 256)
    where = [x.to(dev) for x in (table, torch.tensor([0, 256], dtype=torch.int32), torch.tensor([256], dtype=torch.int32))]
    out = torch.zeros((2, 256, 1, 256), dtype=TYPES[dtype], device=dev)
    c, s = codes.to(dev), scales.to(dev)
    ct.paged_cache_read(c, c, *where, ct.partition(out[0], [1, 1, 256]), ct.partition(out[1], [1, 1, 256]), k_scales=s, v_scales=s)
    for got in out.cpu():
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got[~got.isnan()], want[~want.isnan()])


@pytest.mark.gpu
def test_gpu_values_that_are_no_finite_numbers(ct, dev):
    """a block with a NaN or an infinity stands for NaN, its neighbours do not; 16-bit caches keep the bits"""
    x = torch.randn(4, 1, 64).half()
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 63] = float("nan"), float("inf"), float("-inf")
    b = Batch([4], [4], 2)
    for mx in (False, True):
        k, v, scales = caches(b, 1, 64, "f16", mx, dev)
        ct.paged_cache_write(x.to(dev), x.to(dev), k, v, *b.where(dev), **scales)
        out = torch.zeros((2, 4, 1, 64), dtype=torch.half, device=dev)
        ct.paged_cache_read(k, v, *b.where(dev), ct.partition(out[0], [1, 1, 64]), ct.partition(out[1], [1, 1, 64]), **scales)
        want = ref.values(*ref.quantized(x)).half() if mx else x
        assert torch.equal(out[0].cpu().nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)) and torch.equal(out[0].isnan(), out[1].isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("mx", [False, True])
def test_gpu_metadata_that_names_no_place(ct, dev, mx):
    """pages that the cache lacks, lengths beyond the table, starts beyond the rows: nothing else is written, and such rows read as zeros"""
    b = Batch([4, 4, 4, 4], [4, 4, 4, 4], 4, spare=0)
    b.table[0, 0], b.table[1, 0] = -1, b.pages
    table, starts, lens = b.where(dev)
    lens[2] = 2 ** 31 - 1
    starts[4] = 99
    x = torch.randn(16, 2, 64).half().to(dev)
    k, v, scales = caches(b, 2, 64, "f16", mx, dev)
    before = [t.clone() for t in (k, v, *scales.values())]
    ct.paged_cache_write(x, x, k, v, table, starts, lens, **scales)
    mine = int(b.table[3, 0])   # starts[4] is cut to the 16 rows: the last sequence is whole
    for t, w in zip((k, v, *scales.values()), before):
        keep = [p for p in range(b.pages) if p != mine]
        assert torch.equal(t[keep], w[keep]) and not torch.equal(t[mine], w[mine])
    out = torch.full((2, 16, 2, 64), 9.0, dtype=torch.half, device=dev)
    ct.paged_cache_read(k, v, table, starts, lens, ct.partition(out[0], [16, 2, 64]), ct.partition(out[1], [16, 2, 64]), **scales)
    assert int(out[:, :12].count_nonzero()) == 0 and int(out[:, 12:].count_nonzero()) > 0


@pytest.mark.gpu
def test_gpu_many_sequences(ct, dev):
    """the search for a token's sequence over more than 64 and more than 4096 of them, empty ones among them"""
    for n in (65, 200, 5000):
        new = [(i * 7 + i // 3) % 3 for i in range(n)]
        b = Batch(new, [x + i % 2 for i, x in enumerate(new)], 3, seed=n)
        x = b.normal(b.rows, 1, 64).bfloat16().to(dev)
        k, v, _ = caches(b, 1, 64, "bf16", False, dev)
        ct.paged_cache_write(x, -x, k, v, *b.where(dev))
        places = b.places()
        at, r = (torch.tensor([p[i] for p in places], device=dev) for i in (3, 4))
        assert torch.equal(k[at, r], x[:len(places)]) and torch.equal(v[at, r], -x[:len(places)])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [20000, 70000, 140000])
@pytest.mark.parametrize("heads,d", [(1, 64), (3, 64), (1, 128)])
def test_gpu_many_short_tokens(ct, dev, tokens, heads, d):
    """wavefronts that take several tokens each, of one sequence, of many, and with more than 64 empty ones between them"""
    new = [(i * 7) % 13 for i in range(500)] + [0] * 150 + [1] * 70 + [tokens] + [0, 0, 5]
    b = Batch(new, [x + i % 3 for i, x in enumerate(new)], 64, seed=tokens, rows=sum(new) + 7)
    x = b.normal(b.rows, heads, d).half()
    for mx in (False, True):
        k, v, scales = caches(b, heads, d, "f16", mx, dev)
        ct.paged_cache_write(x.to(dev), (-x).to(dev), k, v, *b.where(dev), **scales)
        places = b.places()
        at, r = (torch.tensor([p[i] for p in places]) for i in (3, 4))
        want = x[:len(places)]
        if mx:
            data, byte = ref.quantized(want)
            assert torch.equal(k.cpu().view(torch.uint8)[at, r], data) and torch.equal(scales["k_scales"].cpu().view(torch.uint8)[at, r], byte)
            want = ref.values(data, byte).half()
        else:
            assert torch.equal(k.cpu()[at, r], want) and torch.equal(v.cpu()[at, r], -want)
        out = torch.full((2, b.rows, heads, d), 9.0, dtype=torch.half, device=dev)
        ct.paged_cache_read(k, v, *b.where(dev), ct.partition(out[0], [4, heads, d]), ct.partition(out[1], [4, heads, d]), **scales)
        got = out.cpu()
        assert torch.equal(got[0, :len(places)], want) and torch.equal(got[1, :len(places)], -want) and bool((got[:, len(places):] == 9.0).all())


@pytest.mark.gpu
def test_gpu_offsets_beyond_32_bits(ct, dev):
    """a cache of 6 GiB whose last pages are used: byte and element offsets pass 2^32"""
    pages, page, heads, d = 3 * 2 ** 12, 64, 16, 256
    b = Batch([40], [100], page)
    k = torch.empty((pages, page, heads, d), dtype=torch.half, device=dev)
    v = torch.empty_like(k)
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=dev)
    k[pages - 2:], v[pages - 2:] = 1.0, 2.0
    x = b.normal(40, heads, d).half().to(dev)
    _, starts, lens = b.where(dev)
    ct.paged_cache_write(x, x + 1, k, v, table, starts, lens)
    got = k[pages - 2:].reshape(2 * page, heads, d)
    assert torch.equal(got[60:100], x) and bool((got[:60] == 1).all()) and bool((got[100:] == 1).all())
    out = torch.zeros((2, 40, heads, d), dtype=torch.half, device=dev)
    ct.paged_cache_read(k, v, table, starts, lens, ct.partition(out[0], [8, heads, d]), ct.partition(out[1], [8, heads, d]))
    assert torch.equal(out[0], x) and torch.equal(out[1], x + 1)


@pytest.mark.gpu
def test_gpu_captured_launches_take_what_the_metadata_holds(ct, dev):
    """one graph of a write and a read, replayed for other tokens, pages and lengths"""
    b = Batch([1, 1], [5, 9], 4, spare=6)
    table, starts, lens = b.where(dev)
    x = torch.zeros((2, 2, 64), dtype=torch.half, device=dev)
    k, v, scales = caches(b, 2, 64, "f16", True, dev)
    out = torch.zeros((2, 2, 2, 64), dtype=torch.half, device=dev)
    parts = [ct.partition(o, [1, 2, 64]) for o in out]
    ct.paged_cache_write(x, x, k, v, table, starts, lens, **scales)
    ct.paged_cache_read(k, v, table, starts, lens, *parts, **scales)
    torch.cuda.synchronize()
    g = ct.CapturedGraph().capture(lambda s: (ct.paged_cache_write(x, x, k, v, table, starts, lens, stream=s, **scales), ct.paged_cache_read(k, v, table, starts, lens, *parts, stream=s, **scales)))
    for i in range(4):
        x.copy_(torch.randn(2, 2, 64))
        lens.copy_(torch.tensor([1 + i, 7 + i]))
        table[0, 0] = (i * 2) % b.pages
        torch.cuda.synchronize()
        g.launch()
        g.synchronize()
        want = ref.values(*ref.quantized(x.cpu())).half()
        assert torch.equal(out[0].cpu(), want) and torch.equal(out[1].cpu(), want)
        torch.randn(1000, device=dev).sum().item()
    g.close()
