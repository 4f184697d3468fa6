"""A serving step over a paged cache: writing new tokens' keys and values into pages, reading pages back, attention of new tokens over them, and the
adjustment of the logits in front of the choice of a token.

Every case is one pass of one operator on the current stream.  ``listed()`` holds representatives of each, ``draw()`` spreads over the
ranges they stand for.  ``run`` computes the definition with elementary torch operations in f32, or (``own``) makes the framework's calls.

A batch of sequences shares one cache of pages.  ``starts`` says which rows of the new tokens are whose, ``context_lens`` how many tokens of
each sequence the cache holds with the new ones, ``page_table`` on which pages they are.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32                                      # values of an mxfp8 cache that share a scale
MOST_PAIRS = 32 * 8192 * 8192 * 128             # padded (query head, query, key) pairs times D: no drawn attention has more than the largest listed one
MOST_CACHE = 64 * 8192 * 8 * 128                # nor a drawn cache more values of K
MOST_LOGITS = 256 * 128256


def listed():
    cache = {"kv_heads": 8, "d": 128, "page": 16, "dtype": "bf16", "cache": "same"}
    attend = {**cache, "op": "attend", "group": 4, "chunks": 0, "chunk": 1, "window": 0}
    return [
        # the new tokens of a decode batch into an 8-bit cache: the smallest call, where the launch is the cost
        {"name": "write_mxfp8_64x1", **cache, "op": "write", "cache": "mxfp8", "batch": 64, "chunks": 0, "chunk": 1, "ctx": 2048},
        # four long prompts into a cache of 16-bit values
        {"name": "write_f16_4x4096", **cache, "op": "write", "dtype": "f16", "page": 64, "batch": 4, "chunks": 4, "chunk": 4096, "ctx": 4096},
        # one conversation's 8-bit cache back to 16 bits, as it moves to another program; its pages are no power of two
        {"name": "read_mxfp8_1x2000", **cache, "op": "read", "cache": "mxfp8", "page": 48, "batch": 1, "ctx": 2000},
        # the caches of a batch of long conversations
        {"name": "read_mxfp8_16x8192", **cache, "op": "read", "cache": "mxfp8", "dtype": "f16", "page": 64, "batch": 16, "ctx": 8192},
        # one token for each of a few short conversations, a KV head to every query head: latency
        {"name": "decode_f16_16x1000_d64", **attend, "dtype": "f16", "kv_heads": 16, "group": 1, "d": 64, "batch": 16, "ctx": 1000},
        # one token behind one very long context: keys have to be dealt out to fill the chip
        {"name": "decode_bf16_1x131072", **attend, "page": 64, "batch": 1, "ctx": 131072},
        # the decode batch of a busy server, lengths of all sorts, 8-bit cache
        {"name": "decode_mxfp8_64x8192", **attend, "cache": "mxfp8", "batch": 64, "ctx": 8192},
        # decodes and two chunks of prompts in one batch, a sliding window
        {"name": "mixed_f16_24x6000_window", **attend, "dtype": "f16", "group": 8, "kv_heads": 4, "page": 32, "batch": 24, "chunks": 2, "chunk": 600, "ctx": 6000, "window": 4096},
        # a chunk of a long prompt behind what is already there, 8-bit cache
        {"name": "chunk_mxfp8_512_behind_16384", **attend, "cache": "mxfp8", "batch": 1, "chunks": 1, "chunk": 512, "ctx": 16896},
        # a whole prompt from nothing: the matrix cores bound it
        {"name": "prompt_bf16_8192", **attend, "page": 64, "batch": 1, "chunks": 1, "chunk": 8192, "ctx": 8192},
        # the logits of one conversation under a grammar
        {"name": "logits_f16_1x128256", "op": "logits", "dtype": "f16", "rows": 1, "vocab": 128256, "history": 2000, "biases": 20, "mask": True},
        # of a large decode batch with long histories
        {"name": "logits_bf16_256x128256", "op": "logits", "dtype": "bf16", "rows": 256, "vocab": 128256, "history": 6000, "biases": 0, "mask": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "attend", "logits"])
    if op == "logits":
        vocab = _log(rng, 20000, 200000)
        return {"op": op, "dtype": rng.choice(["f16", "bf16", "f32"]), "rows": min(_log(rng, 1, 256), MOST_LOGITS // vocab), "vocab": vocab if rng.random() < 0.5 else vocab // 64 * 64,
                "history": _log(rng, 10, 8000), "biases": rng.choice([0, _log(rng, 1, 300)]), "mask": rng.random() < 0.5}
    c = {"op": op, "dtype": rng.choice(["f16", "bf16"]), "cache": rng.choice(["same", "mxfp8"]), "kv_heads": rng.choice([1, 2, 4, 8, 16]), "d": rng.choice([64, 128, 128, 256]),
         "page": rng.choice([16, 16, 32, 64, 128, _log(rng, 1, 256)]), "batch": _log(rng, 1, 128)}
    most = max(16, MOST_CACHE // (c["batch"] * c["kv_heads"] * c["d"]))      # tokens of a context
    if op == "read":
        c["ctx"] = min(_log(rng, 16, 32768), most // 2)
        return c
    c.update(chunks=0, chunk=1, ctx=min(_log(rng, 16, 131072), most))
    if op == "attend":
        c.update(group=rng.choice([1, 2, 4, 6, 8]), window=rng.choice([0, 0, 0, _log(rng, 16, 8192)]))
    kind = rng.choice(["decode", "chunks", "few", "mixed"])
    if kind != "decode":
        c["chunk"] = min(_log(rng, 2, 8) if kind == "few" else _log(rng, 16, 8192), c["ctx"])
        c["chunks"] = max(1, c["batch"] // 8) if kind == "mixed" else c["batch"]
    if op == "attend":
        while c["batch"] > 1 and c["batch"] * c["kv_heads"] * c["group"] * c["chunk"] * c["ctx"] * c["d"] > MOST_PAIRS:
            c["batch"] = (c["batch"] + 1) // 2
            c["chunks"] = min(c["chunks"], c["batch"])
        while c["chunk"] > 1 and work(c)["flops"] > 2.0 * MOST_PAIRS:
            c["chunk"] //= 2
    elif c["batch"] * c["chunk"] * c["kv_heads"] * c["d"] > MOST_CACHE // 4:
        c["chunk"] = max(1, MOST_CACHE // 4 // (c["batch"] * c["kv_heads"] * c["d"]))
    return c


def _lengths(case):
    """(new tokens, tokens in the cache) of each sequence, by the case alone"""
    rng = random.Random(7919 * case["batch"] + case["ctx"])
    b, ctx = case["batch"], case["ctx"]
    if case["op"] == "read":
        held = [ctx if b == 1 else rng.randint(max(1, ctx // 4), ctx) for _ in range(b)]
        return held, held
    new = [1] * b
    at = rng.sample(range(b), case["chunks"])
    for i in at:
        new[i] = case["chunk"] if b == 1 or case["chunk"] < 16 else rng.randint(case["chunk"] // 2, case["chunk"])
    held = [max(n, ctx if b == 1 else rng.randint(max(1, ctx // 4), ctx)) for n in new]
    return new, held


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class _Make:
    """seeded inputs on the GPU"""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, dtype, std=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=self.g)

    def uniform(self, *shape, lo=0.0, hi=1.0):
        return torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(lo, hi, generator=self.g)

    def integers(self, *shape, lo, hi, dtype):
        return torch.randint(lo, hi, shape, dtype=dtype, device="cuda", generator=self.g)

    def held(self, case, pages):
        """what the cache holds beforehand, (data, scales or None)"""
        shape = (pages, case["page"], case["kv_heads"], case["d"])
        if case["cache"] == "same":
            return self.normal(*shape, dtype=DTYPES[case["dtype"]]), None
        return _quantize(self.normal(*shape, dtype=torch.float32))


def _prepare_logits(case, mk):
    rows, vocab, history = case["rows"], case["vocab"], case["history"]
    s = {"case": case, "logits": mk.normal(rows, vocab, dtype=DTYPES[case["dtype"]], std=3.0)}
    s["out"] = torch.zeros_like(s["logits"])
    # a few tokens make up most of a text: rank r about as often as 1 / r
    s["tokens"] = (mk.uniform(rows, history) * math.log(vocab)).exp().long().clamp(max=vocab - 1).mul(7919).remainder(vocab).int()
    s["token_lens"] = mk.integers(rows, lo=history // 2, hi=history + 1, dtype=torch.int32)
    s["prompt_lens"] = s["token_lens"] // 2
    s["repetition"], s["presence"], s["frequency"] = mk.uniform(rows, lo=1.0, hi=1.3), mk.uniform(rows), mk.uniform(rows, hi=0.3)
    s["bias_ids"] = s["bias_values"] = s["allowed"] = None
    if case["biases"]:
        s["bias_ids"] = mk.integers(rows, case["biases"], lo=0, hi=vocab, dtype=torch.int32)
        s["bias_values"] = mk.uniform(rows, case["biases"], lo=-5.0, hi=5.0)
    if case["mask"]:
        s["allowed"] = mk.integers(rows, -(-vocab // 32), lo=-2 ** 31, hi=2 ** 31, dtype=torch.int64).int()
    return s


def prepare(case, seed):
    mk = _Make(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, mk)
    new, held = _lengths(case)
    tokens, dtype, page = sum(new), DTYPES[case["dtype"]], case["page"]
    counts = [-(-h // page) for h in held]
    pages = sum(counts) + sum(counts) // 8 + 1                                            # a server has some to spare
    order = torch.randperm(pages, device="cuda", generator=mk.g).int()
    table = torch.zeros((case["batch"], max(counts)), dtype=torch.int32, device="cuda")
    where = torch.arange(max(counts), device="cuda").unsqueeze(0) < _ints(counts).unsqueeze(1)
    table[where] = order[:sum(counts)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"case": case, "new": new, "held": held, "page_table": table, "starts": _ints(starts), "context_lens": _ints(held), "max_new": max(new), "max_context": max(held)}
    s["k_cache"], s["k_scales"] = mk.held(case, pages)
    s["v_cache"], s["v_scales"] = mk.held(case, pages)
    heads, d = case["kv_heads"], case["d"]
    if case["op"] == "write":
        qkv = mk.normal(tokens, 6 * heads, d, dtype=dtype)                                # q, k and v come out of one product side by side
        s.update(new_k=qkv[:, 4 * heads:5 * heads], new_v=qkv[:, 5 * heads:])
    elif case["op"] == "read":
        s.update(out_k=torch.zeros((tokens, heads, d), dtype=dtype, device="cuda"), out_v=torch.zeros((tokens, heads, d), dtype=dtype, device="cuda"))
    else:
        s["q"] = mk.normal(tokens, heads * case["group"], d, dtype=dtype)
        s["out"] = torch.zeros_like(s["q"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _places(s):
    """of every row of the new tokens: its sequence, its position, its page and its row on that page"""
    case = s["case"]
    row = torch.arange(sum(s["new"]), device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    at = row - s["starts"][1:].long()[seq] + s["context_lens"].long()[seq]
    return seq, at, s["page_table"].long()[seq, at // case["page"]], at % case["page"]


def _quantize(v):
    """rows of values in f32 -> (e4m3, e8m0) in blocks along the last axis"""
    b = v.unflatten(-1, (-1, BLOCK))
    most = b.abs().amax(-1, keepdim=True)
    byte = (torch.frexp(most).exponent - 1 - 8 + 127).clamp(0, 254)
    byte = torch.where(most == 0, torch.zeros_like(byte), byte)
    data = torch.ldexp(b, 127 - byte).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return data.flatten(-2), byte.squeeze(-1).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(data, scales, dtype=torch.float32):
    if scales is None:
        return data.to(dtype)
    return (data.to(dtype).unflatten(-1, (-1, BLOCK)) * scales.to(dtype).unsqueeze(-1)).flatten(-2)


def _bytes(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t


def _picked(t, page, row):
    return None if t is None else _bytes(t)[page, row].view(t.dtype)


def _write(s):
    _, _, page, row = _places(s)
    if s["k_scales"] is None:
        s["k_cache"][page, row] = s["new_k"]
        s["v_cache"][page, row] = s["new_v"]
        return s["k_cache"], s["v_cache"]
    (k, ks), (v, vs) = _quantize(s["new_k"].float()), _quantize(s["new_v"].float())
    _bytes(s["k_cache"])[page, row] = _bytes(k)
    _bytes(s["v_cache"])[page, row] = _bytes(v)
    _bytes(s["k_scales"])[page, row] = _bytes(ks)
    _bytes(s["v_scales"])[page, row] = _bytes(vs)
    return s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]


def _read(s):
    _, _, page, row = _places(s)
    k = _values(_picked(s["k_cache"], page, row), _picked(s["k_scales"], page, row))
    v = _values(_picked(s["v_cache"], page, row), _picked(s["v_scales"], page, row))
    return k.to(s["out_k"].dtype), v.to(s["out_v"].dtype)


def _attend(s):
    """all sequences at once, padded to the most new tokens and the longest context"""
    case = s["case"]
    seq, at, _, _ = _places(s)
    batch, heads, group, d, page = case["batch"], case["kv_heads"], case["group"], case["d"], case["page"]
    slot = torch.arange(seq.numel(), device="cuda") - s["starts"].long()[seq]
    key = torch.arange(s["max_context"], device="cuda")
    pages = s["page_table"].long()[:, key // page]
    rows = (key % page).unsqueeze(0).expand_as(pages)
    k = _values(_picked(s["k_cache"], pages, rows), _picked(s["k_scales"], pages, rows)).permute(0, 2, 3, 1).contiguous()   # [batch, heads, d, keys]
    v = _values(_picked(s["v_cache"], pages, rows), _picked(s["v_scales"], pages, rows)).transpose(1, 2).contiguous()
    q = torch.zeros((batch, s["max_new"], heads * group, d), device="cuda")
    q[seq, slot] = s["q"].float()
    q = q.unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).reshape(batch, heads, -1, d)
    p = torch.full((batch, s["max_new"]), -1, dtype=torch.int64, device="cuda")
    p[seq, slot] = at
    sees = key <= p.unsqueeze(-1)
    if case["window"]:
        sees &= key > p.unsqueeze(-1) - case["window"]
    score = (torch.matmul(q, k) * d ** -0.5).unflatten(2, (group, -1)).masked_fill_(~sees[:, None, None], -math.inf)
    score = (score - score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    score = (score / score.sum(-1, keepdim=True).clamp(min=1e-30)).flatten(2, 3)
    o = torch.matmul(score, v).unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[seq, slot].to(s["q"].dtype)


def _adjust(s):
    l, tokens = s["logits"].float(), s["tokens"].long()
    at = torch.arange(tokens.shape[1], device="cuda")
    known, made = at < s["token_lens"].unsqueeze(1), at >= s["prompt_lens"].unsqueeze(1)
    seen = torch.zeros_like(l).scatter_add_(1, tokens, known.float()) > 0
    count = torch.zeros_like(l).scatter_add_(1, tokens, (known & made).float())
    r, presence, frequency = s["repetition"].unsqueeze(1), s["presence"].unsqueeze(1), s["frequency"].unsqueeze(1)
    l = torch.where(seen, torch.where(l > 0, l / r, l * r), l)
    l = l - (presence * (count > 0).float() + frequency * count)
    if s["bias_ids"] is not None:
        l = l + torch.zeros_like(l).scatter_add_(1, s["bias_ids"].long(), s["bias_values"])
    if s["allowed"] is not None:
        bits = (s["allowed"].unsqueeze(-1) >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        l = l.masked_fill(bits.flatten(1)[:, :l.shape[1]] == 0, -math.inf)
    return l.to(s["logits"].dtype)


def _plain(s):
    op = s["case"]["op"]
    if op == "logits":
        return _adjust(s)
    return _write(s) if op == "write" else _read(s) if op == "read" else _attend(s)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
_package = None


def _ct():
    global _package
    if _package is None:
        from __graft_entry__ import load_package
        _package = load_package()
    return _package


def _own(s):
    ct, case = _ct(), s["case"]
    op = case["op"]
    if op == "logits":
        ct.adjust_logits(s["logits"], ct.partition(s["out"], [1, case["vocab"]]), tokens=s["tokens"], prompt_lens=s["prompt_lens"], token_lens=s["token_lens"], repetition=s["repetition"],
                         presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"])
        return s["out"]
    where = (s["page_table"], s["starts"], s["context_lens"])
    scales = {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if op == "write":
        ct.paged_cache_write(s["new_k"], s["new_v"], s["k_cache"], s["v_cache"], *where, **scales)
        return (s["k_cache"], s["v_cache"]) + (() if s["k_scales"] is None else (s["k_scales"], s["v_scales"]))
    if op == "read":
        tile = [1, case["kv_heads"], case["d"]]
        ct.paged_cache_read(s["k_cache"], s["v_cache"], *where, ct.partition(s["out_k"], tile), ct.partition(s["out_v"], tile), **scales)
        return s["out_k"], s["out_v"]
    ct.paged_attention(s["q"], s["k_cache"], s["v_cache"], *where, ct.partition(s["out"], [1, case["group"], case["d"]]), case["d"] ** -0.5, window=case["window"], max_new=s["max_new"],
                       max_context=s["max_context"], **scales)
    return s["out"]


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "logits":
        values = float(case["rows"]) * case["vocab"]
        return {"bytes": 2 * size * values + (values / 8 if case["mask"] else 0.0) + case["rows"] * (3.0 * case["history"] + 8.0 * case["biases"]), "flops": 8.0 * values}
    new, held = _lengths(case)
    kept = size if case["cache"] == "same" else 1 + 1 / BLOCK                               # bytes of a value in the cache
    row = 2.0 * case["kv_heads"] * case["d"]                                              # values of K and V of a token
    if op != "attend":
        return {"bytes": sum(new) * row * (size + kept), "flops": 3.0 * sum(new) * row}
    w = case["window"] or max(held)
    keys = sum(min(h, n + w - 1) for n, h in zip(new, held))
    pairs = sum(_pairs(n, h, w) for n, h in zip(new, held))
    heads = case["kv_heads"] * case["group"]
    return {"bytes": keys * row * kept + 2.0 * size * sum(new) * heads * case["d"], "flops": 4.0 * pairs * heads * case["d"]}


def _pairs(n, h, w):
    """visible (query, key) pairs: new token i of n sees min(h - n + 1 + i, w) keys"""
    first = h - n + 1
    short = max(0, min(n, w - first))                                                     # tokens that see all of fewer than w keys
    return short * first + short * (short - 1) / 2 + (n - short) * float(w)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def _exact_blocks(x):
    """(elements, scales) of mxfp8 blocks along the last axis, as values in 64 bits"""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 9, torch.full_like(top, -127, dtype=torch.int32)).clamp(min=-127)
    scale = torch.exp2(e.double())
    v = b / scale
    at = torch.where(v == 0, torch.full_like(v, -6, dtype=torch.int32), torch.frexp(v)[1] - 1).clamp(min=-6)
    step = torch.exp2(at.double() - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0).flatten(-2), scale.squeeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        l = s["logits"].double()
        for row in range(case["rows"]):
            n, prompt = int(s["token_lens"][row]), int(s["prompt_lens"][row])
            tokens = s["tokens"][row, :n].long()
            said = torch.unique(tokens)
            l[row, said] *= torch.exp2(-torch.sign(l[row, said]) * torch.log2(s["repetition"][row].double()))
            made, times = torch.unique(tokens[prompt:], return_counts=True)
            l[row, made] -= s["presence"][row].double() + s["frequency"][row].double() * times
            if case["biases"]:
                l[row].index_add_(0, s["bias_ids"][row].long(), s["bias_values"][row].double())
        if case["mask"]:
            at = torch.arange(case["vocab"], device="cuda")
            l[torch.bitwise_and(s["allowed"][:, at // 32].long(), 2 ** (at % 32)) == 0] = -math.inf
        return l
    page, group, d = case["page"], case.get("group", 1), case["d"]
    if op == "attend":                                                                    # one sequence and KV head after another, without padding
        out, first = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
        for b, (n, h) in enumerate(zip(s["new"], s["held"])):
            key = torch.arange(h, device="cuda")
            at = (s["page_table"][b].long()[key // page], key % page)
            p = torch.arange(h - n, h, device="cuda").unsqueeze(1)
            hidden = (key > p) | ((key <= p - case["window"]) if case["window"] else torch.zeros_like(key > p))
            k, v = (_values(_picked(s[x + "_cache"], *at), _picked(s[x + "_scales"], *at), torch.float64) for x in "kv")
            for head in range(case["kv_heads"]):
                q = s["q"][first:first + n, head * group:(head + 1) * group].double().reshape(n * group, d)
                score = ((q @ k[:, head].t()) / math.sqrt(d)).masked_fill_(hidden.repeat_interleave(group, 0), -math.inf)
                out[first:first + n, head * group:(head + 1) * group] = (torch.softmax(score, -1) @ v[:, head]).view(n, group, d)
            first += n
        return out
    seq = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(s["new"])])
    at = torch.cat([torch.arange(h - n, h, device="cuda") for n, h in zip(s["new"], s["held"])])
    page, row = s["page_table"].long()[seq, at // page], at % page
    if op == "read":
        return tuple(_values(_picked(s[x + "_cache"], page, row), _picked(s[x + "_scales"], page, row), torch.float64) for x in "kv")
    k, v = s["k_cache"].double(), s["v_cache"].double()
    if case["cache"] == "same":
        k[page, row], v[page, row] = s["new_k"].double(), s["new_v"].double()
        return k, v
    ks, vs = s["k_scales"].double(), s["v_scales"].double()
    (k[page, row], ks[page, row]), (v[page, row], vs[page, row]) = _exact_blocks(s["new_k"]), _exact_blocks(s["new_v"])
    return k, v, ks, vs
