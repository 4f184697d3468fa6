"""adjust_logits (adjust_logits.hip): penalties, biases and masks against 64 bits, and a serving step that uses it."""
import math

import pytest
import torch

import paged_ref as ref
from paged_ref import Batch

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def plain(logits, tokens=None, prompt_lens=None, token_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None, allowed=None):
    """the definition in 64 bits, and the sum of the magnitudes of what each value is added up from"""
    l = logits.double()
    size = l.abs()
    rows, vocab = l.shape
    for r in range(rows):
        if tokens is not None:
            n = tokens.shape[1] if token_lens is None else min(max(int(token_lens[r]), 0), tokens.shape[1])
            p = 0 if prompt_lens is None else min(max(int(prompt_lens[r]), 0), n)
            inside = lambda t: t[(t >= 0) & (t < vocab)].long()
            seen = inside(tokens[r, :n]).unique()
            by = 1.0 if repetition is None else float(repetition[r])
            l[r, seen] = torch.where(l[r, seen] > 0, l[r, seen] / by, l[r, seen] * by)
            size[r, seen] = torch.maximum(size[r, seen], l[r, seen].abs())
            made, count = inside(tokens[r, p:n]).unique(return_counts=True)
            less = (0.0 if presence is None else float(presence[r])) + (0.0 if frequency is None else float(frequency[r])) * count.double()
            more = (0.0 if presence is None else abs(float(presence[r]))) + (0.0 if frequency is None else abs(float(frequency[r]))) * count.double()
            l[r, made] -= less
            size[r, made] += more
        if bias_ids is not None:
            for i, x in zip(bias_ids[r].tolist(), bias_values[r].double().tolist()):
                if 0 <= i < vocab:
                    l[r, i] += x
                    size[r, i] += abs(x)
        if allowed is not None:
            t = torch.arange(vocab)
            l[r, (allowed[r, t // 32].long() >> (t % 32)) & 1 == 0] = -math.inf
    return l, size


def check(got, want, size, biases=0):
    """rounded once to the type; before that up to 5 + the number of biases roundings to f32 of numbers no larger than `size`"""
    u = torch.finfo(got.dtype).eps / 2
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got == -math.inf, want == -math.inf) and torch.equal(got == math.inf, want == math.inf)
    fine = want.isfinite()
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 2.0 ** -140
    tol = u * want.abs() + (5 + biases) * 2.0 ** -24 * (1 + u) * size + tiny
    assert bool(((got - want).abs() <= tol)[fine].all()), float(((got - want).abs() / tol)[fine].max())


def make(rows, vocab, dtype, history, biases, mask, seed):
    g = torch.Generator().manual_seed(seed)
    ints = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, dtype=torch.int64).int()
    x = {"logits": (torch.randn(rows, vocab, generator=g) * 4).to(TYPES[dtype])}
    if history:
        x.update(tokens=ints(-3, min(vocab + 5, 400), rows, history), token_lens=ints(-1, history + 3, rows), prompt_lens=ints(-1, history, rows), repetition=torch.rand(rows, generator=g) + 0.6,
                 presence=torch.rand(rows, generator=g) - 0.3, frequency=torch.rand(rows, generator=g) - 0.3)
    if biases:
        x.update(bias_ids=ints(-2, min(vocab + 2, 3 * biases + 3), rows, biases), bias_values=torch.randn(rows, biases, generator=g) * 5)
    if mask:
        x["allowed"] = ints(-2 ** 31, 2 ** 31, rows, -(-vocab // 32) + 1)
    return x


def launch(ct, x, out, **kw):
    ct.adjust_logits(x["logits"], ct.partition(out, [1, out.shape[1]]), **{k: v for k, v in x.items() if k != "logits"}, **kw)


# ---- without a GPU --------------------------------------------------------------------------------------------------------
def test_refusals(fake_hip):
    ct = fake_hip
    x = make(3, 100, "f16", 8, 4, True, 1)
    out = torch.zeros(3, 100, dtype=torch.half)
    go = lambda o=out, tile=None, kw={}, **c: ct.adjust_logits({**x, **c}["logits"], ct.partition(o, tile or [1, o.shape[1]]), **{k: v for k, v in {**x, **c}.items() if k != "logits"}, **kw)
    go()
    n0 = ct.lib().cutile_testing_launch_count()
    z, i32 = torch.zeros, torch.int32
    cases = [
        (lambda: go(logits=z(3, 100).double()), "logits must be"),
        (lambda: go(logits=z(100, 3).half().t()), "unit inner stride"),
        (lambda: go(o=z(3, 100)), "out must be"),
        (lambda: go(o=z(2, 100).half()), "out must be"),
        (lambda: go(tile=[1, 50]), "partitioned"),
        (lambda: go(o=z(1, 100).half().expand(3, 100)), "elements of out overlap"),
        (lambda: go(tokens=None), "nothing without tokens"),
        (lambda: go(tokens=z(3, 8, dtype=torch.int64)), "tokens must be"),
        (lambda: go(tokens=z(2, 8, dtype=i32)), "tokens must be"),
        (lambda: go(tokens=z(8, 3, dtype=i32).t()), "tokens must be"),
        (lambda: go(token_lens=z(2, dtype=i32)), "token_lens must be"),
        (lambda: go(prompt_lens=z(3)), "prompt_lens must be"),
        (lambda: go(repetition=z(3).half()), "repetition must be"),
        (lambda: go(presence=z(2)), "presence must be"),
        (lambda: go(frequency=z(6)[::2]), "frequency must be"),
        (lambda: go(bias_values=None), "come together"),
        (lambda: go(bias_values=z(3, 5)), "as many ids as values"),
        (lambda: go(bias_ids=z(3, 1025, dtype=i32), bias_values=z(3, 1025)), "up to 1024 biases"),
        (lambda: go(bias_values=z(3, 4).half()), "bias_values must be"),
        (lambda: go(allowed=z(3, 3, dtype=i32)), "needs 4 words"),
        (lambda: go(allowed=z(3, 4, dtype=torch.int64)), "allowed must be"),
        (lambda: go(kw={"variant": "bf16_1024"}), "does not fit these arguments"),
        (lambda: go(kw={"grid": (2, 1, 1)}), "grid"),
    ]
    for i, (fn, msg) in enumerate(cases):
        with pytest.raises(ct.CutileError, match=msg):
            fn()
            print("case", i, msg)
    assert ct.lib().cutile_testing_launch_count() == n0
    fn, p, t = ct.lib().cutile_launch_adjust_logits, __import__("ctypes").pointer, lambda v: __import__("ctypes").pointer(ct.tensor_arg(v, None))
    part = p(ct.Partition(out, [1, 100], False, None).arg())
    assert fn(None, t(x["logits"]), part, *[None] * 10) == 0
    assert fn(None, None, part, *[None] * 10) == -2 and fn(None, t(x["logits"]), None, *[None] * 10) == -2
    many = ct.tensor_arg(x["tokens"], None)
    many.shape[1], many.strides[0] = 2 ** 30, 2 ** 30
    n0 = ct.lib().cutile_testing_launch_count()
    assert fn(None, t(x["logits"]), part, p(many), *[None] * 9) != 0 and b"fewer than 2^30 tokens" in ct.lib().cutile_last_error_message()
    assert ct.lib().cutile_testing_launch_count() == n0


# ---- on a GPU ---------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab,history,biases,mask", [(1, 1, 1, 1, True), (3, 100, 8, 4, True), (2, 1025, 50, 0, False), (5, 4099, 3000, 300, True), (2, 40000, 700, 1024, False), (1, 16384, 0, 3, False),
                                                             (40, 9000, 1, 0, True), (1, 128256, 5000, 20, True)])
def test_gpu_adjusted(ct, dev, dtype, rows, vocab, history, biases, mask):
    x = make(rows, vocab, dtype, history, biases, mask, rows + vocab)
    on = {k: v.to(dev) for k, v in x.items()}
    out = torch.full_like(on["logits"], 7.0)
    launch(ct, on, out)
    want, size = plain(**x)
    check(out.cpu(), want, size, biases)
    for v in (1024, 4096, 8192):
        other = torch.full_like(out, 7.0)
        launch(ct, on, other, variant=f"{dtype}_{v}")
        assert torch.equal(other, out)
    launch(ct, on, on["logits"])            # in place
    assert torch.equal(on["logits"], out)


@pytest.mark.gpu
def test_gpu_each_by_itself_and_strides(ct, dev):
    x = make(4, 3001, "f16", 60, 7, True, 3)
    wide = torch.zeros(4, 3100, dtype=torch.half, device=dev)
    for keep in (("tokens",), ("tokens", "repetition"), ("tokens", "presence", "token_lens"), ("tokens", "frequency", "prompt_lens"), ("bias_ids", "bias_values"), ("allowed",), ()):
        some = {"logits": x["logits"], **{k: x[k] for k in keep}}
        on = {k: v.to(dev) for k, v in some.items()}
        wide.fill_(7.0)
        wide[:, 3:3004] = on["logits"]
        if "tokens" in on:
            on["tokens"] = torch.cat((on["tokens"], on["tokens"]), 1)[:, :60]
        ct.adjust_logits(wide[:, 3:3004], ct.partition(wide[:, 3:3004], [1, 3001]), **{k: v for k, v in on.items() if k != "logits"})
        want, size = plain(**some)
        check(wide[:, 3:3004].cpu(), want, size, 7)
        assert bool((wide[:, :3] == 7.0).all()) and bool((wide[:, 3004:] == 7.0).all())


@pytest.mark.gpu
def test_gpu_values_that_are_no_finite_numbers(ct, dev):
    """infinities and NaN pass the penalties; a bias of -infinity forbids a token; nothing allowed leaves -infinity everywhere"""
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[inf, -inf, nan, 0.0, -0.0, 1.0, 60000.0, -60000.0]]).half()
    x = {"logits": logits, "tokens": torch.arange(8, dtype=torch.int32).reshape(1, 8), "repetition": torch.tensor([2.0]), "presence": torch.tensor([0.5]), "bias_ids": torch.tensor([[5, 3, 5]], dtype=torch.int32),
         "bias_values": torch.tensor([[1.0, -inf, 2.0]])}
    on = {k: v.to(dev) for k, v in x.items()}
    out = torch.zeros_like(on["logits"])
    launch(ct, on, out)
    assert torch.equal(out.cpu().nan_to_num(123.0, inf, -inf), torch.tensor([[inf, -inf, 123.0, -inf, -0.5, 3.0, 29999.5, -inf]]).half().nan_to_num(123.0, inf, -inf))
    launch(ct, {**on, "allowed": torch.zeros(1, 1, dtype=torch.int32, device=dev)}, out)
    assert bool((out == -inf).all())


@pytest.mark.gpu
def test_gpu_serving_steps(ct, dev):
    """Three greedy steps of a batch as a server takes them: the new tokens' K and V into an mxfp8 cache, attention over it, logits adjusted and the token chosen,
    against the same in 64 bits from the cache that the launches wrote"""
    heads, group, d, vocab, page = 2, 4, 64, 4096, 16
    held, new = [40, 7, 65], [40, 7, 65]
    torch.manual_seed(5)
    table_of = lambda h: Batch([0, 0, 0], [x + 3 for x in h], page, seed=2)
    b = table_of(held)
    k, v = (torch.zeros((b.pages, page, heads, d), dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((b.pages, page, heads, d // 32), dtype=torch.uint8, device=dev) for _ in range(2))
    head = (torch.randn(heads * group * d, vocab) * 0.1).to(dev)
    embed = torch.randn(vocab, heads * (group + 2), d).half().to(dev)
    tokens = torch.randint(0, vocab, (3, 80), dtype=torch.int32)
    lens = torch.tensor(held, dtype=torch.int32)
    for step in range(3):
        b.new, b.held = new, lens.tolist()
        b.starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
        b.lens = lens
        ids = torch.cat([tokens[s, int(lens[s]) - n:int(lens[s])] for s, n in enumerate(new)]).long().to(dev)
        qkv = embed[ids]
        where = b.where(dev)
        scales = {"k_scales": ks, "v_scales": vs}
        ct.paged_cache_write(qkv[:, -2 * heads:-heads], qkv[:, -heads:], k, v, *where, **scales)
        out = torch.zeros((len(ids), heads * group, d), dtype=torch.half, device=dev)
        q = qkv[:, :heads * group]
        ct.paged_attention(q, k, v, *where, ct.partition(out, [1, group, d]), d ** -0.5, max_new=max(new), max_context=int(lens.max()), **scales)
        parts = ref.attention(b, q.cpu(), ref.values(k.cpu(), ks.cpu()), ref.values(v.cpu(), vs.cpu()), d ** -0.5)
        assert bool(((out.cpu().double() - parts[0]).abs() <= ref.bound(torch.half, parts, d, 70)).all())
        last = b.starts[1:].long() - 1
        logits = (out[last.to(dev)].flatten(1).float() @ head).half()
        x = {"tokens": tokens, "prompt_lens": torch.tensor(held, dtype=torch.int32), "token_lens": lens, "repetition": torch.full((3,), 1.2), "frequency": torch.full((3,), 0.5),
             "allowed": torch.randint(-2 ** 31, 2 ** 31, (3, vocab // 32), dtype=torch.int64).int()}
        want, size = plain(logits.cpu(), **x)
        ct.adjust_logits(logits, ct.partition(logits, [1, vocab]), **{n: t.to(dev) for n, t in x.items()})
        check(logits.cpu(), want, size)
        top, where_, best = torch.zeros(4, device=dev), torch.zeros(4, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
        for s in range(3):
            ct.argmax_blocks_f16(logits[s], ct.partition(top, [1]), ct.partition(where_, [1]), vocab)
            ct.argmax_reduce_blocks_to_u32(top, where_, ct.partition(best[s:s + 1], [1]), 4)
        assert torch.equal(best.cpu().long(), logits.float().argmax(-1).cpu())
        for s in range(3):
            tokens[s, int(lens[s])] = int(best[s])
        lens, new = lens + 1, [1, 1, 1]
