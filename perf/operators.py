"""
The operators of a paged cache, each as its users call it, beside a plain form of the same mathematics:

``rotary``  ``longctx.ops.rotary_``: queries and keys of a ragged batch, every token at its own position, normalised per head
            and rotated; half-split or interleaved pairs, the whole head or its first part.
``write``   ``kvcache.paged.paged_write``: new K and V rows into the slots of their pages.
``store``   ``paged_write`` into 8-bit or 4-bit pages, and ``paged_read`` of whole sequences back: their rows are what is compared.
``read``    ``paged_read`` of sequences on plain pages, as a chunk's attention takes them.
``decode``  ``attention.ops.paged_decode``: one new token a sequence over its pages, sequences of any lengths.
``step``    the three that a layer calls for one new token a sequence: rotary, write, decode.

A case is a dict of plain values; the lengths of its sequences follow from it alone (see ``_lengths``). Shapes are those of the
benchmark's configurations (32 / 8 heads of 128, caches of 16384 to 131072 slots, 8-bit and 4-bit stores), of the tests (other
numbers of heads, head sizes 64 and 256, float16) and what lies between them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BITS = {"plain": 16, "u8": 8, "u4": 4}
HEADS = [(32, 8), (32, 8), (8, 2), (28, 4), (24, 8), (32, 4), (16, 8), (8, 8), (16, 1)]  # query heads / KV heads
EPS = 1.0e-6
MAX_BYTES = 4.6e9


def _rotary(name, tokens, heads, D, rotary_dim, interleaved, norm, context, dtype="bf16", padded=0):
    return {"name": name, "kind": "rotary", "tokens": tokens, "Hq": heads[0], "Hkv": heads[1], "D": D, "rotary_dim": rotary_dim, "interleaved": interleaved,
            "norm": norm, "context": context, "dtype": dtype, "padded": padded}


def _paged(name, kind, B, heads, D, low, high, page, store="plain", dtype="bf16", empty=0, **more):
    return {"name": name, "kind": kind, "B": B, "Hq": heads[0], "Hkv": heads[1], "D": D, "low": low, "high": high, "page": page, "store": store, "dtype": dtype,
            "empty": empty, **more}


def listed():
    return [
        # one new token for each of 32 sequences: what a layer rotates in a step of generation
        _rotary("rotary_tokens", 32, (32, 8), 128, 128, False, True, 131072),
        # the packed prompts of a serving batch
        _rotary("rotary_prompts", 16384, (32, 8), 128, 128, False, True, 32768),
        # interleaved pairs in a part of the head, an odd number of tokens, padding behind the last of them
        _rotary("rotary_part", 5001, (28, 4), 128, 64, True, False, 8192, dtype="fp16", padded=77),
        # the K and V rows of packed prompts, 16-bit pages
        _paged("write_prompts", "write", 5, (32, 8), 128, 1024, 8192, 64),
        # chunks of a few sequences into 8-bit pages, and the sequences back
        _paged("store_u8", "store", 4, (32, 8), 128, 4096, 16384, 64, store="u8"),
        # short ragged sequences on 4-bit pages, two heads of 64
        _paged("store_u4", "store", 7, (8, 2), 64, 5, 700, 16, store="u4", dtype="fp16", empty=1),
        # generation for one user: one sequence, latency is everything
        _paged("decode_one", "decode", 1, (32, 8), 128, 4000, 4000, 16, lse=False, capacity=8192),
        # a serving batch of very different lengths, padded by sequences without a token
        _paged("decode_ragged", "decode", 64, (28, 4), 128, 1, 8192, 16, empty=3, lse=True, capacity=8192),
        # long sequences on 8-bit pages
        _paged("decode_u8", "decode", 16, (32, 8), 128, 16384, 65536, 64, store="u8", lse=False, capacity=131072),
        # the same rows in 4 bits, of a float16 model with many heads over one KV head
        _paged("decode_u4", "decode", 48, (16, 1), 64, 3000, 50000, 32, store="u4", dtype="fp16", lse=True, capacity=65536),
        # the benchmark's decode configuration, paged: 8 sequences of 131072 tokens
        _paged("decode_large", "decode", 8, (32, 8), 128, 131072, 131072, 64, lse=False, capacity=131072),
        # one layer's share of a step of generation for 32 sequences
        _paged("step", "step", 32, (32, 8), 128, 500, 6000, 16, capacity=8192),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; no more work than the largest of the listed ones."""
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= MAX_BYTES and _padded_bytes(case) <= MAX_BYTES:
            return case


def _draw(rng):
    kind = rng.choices(["rotary", "write", "store", "read", "decode", "step"], [18, 9, 14, 9, 40, 10])[0]
    heads = rng.choice(HEADS)
    D = rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rotary":
        tokens = _log_int(rng, 1, 16384)
        case = _rotary("", tokens, heads, D, rng.choice([D, D, D // 2, D // 4]), rng.random() < 0.4, rng.random() < 0.5, _log_int(rng, 256, 131072), dtype,
                       rng.choice([0, 0, _log_int(rng, 1, tokens) // 2]))
    else:
        page = rng.choice([16, 16, 32, 64, 128, 256])
        store = "plain" if kind in ("write", "read", "step") else rng.choice(["u8", "u4"] if kind == "store" else ["plain", "plain", "u8", "u4"])
        most = {"write": 16384, "store": 16384, "read": 16384, "decode": 131072, "step": 32768}[kind]
        high = _log_int(rng, 1, most)
        low = min(high, rng.choice([high, _log_int(rng, 1, high)]))
        B = _log_int(rng, 1, 256 if kind in ("decode", "step") else 16)
        more = {}
        if kind in ("decode", "step"):
            more["capacity"] = rng.choice([high, min(131072, 2 * high)])
        if kind == "decode":
            more["lse"] = rng.random() < 0.5
        case = _paged("", kind, B, heads, D, low, high, page, store, dtype, rng.choice([0, 0, B // 8]), **more)
    del case["name"]
    return case


# -- inputs ---------------------------------------------------------------------------------------------------


def _lengths(c):
    """Tokens of the sequences: even over the logarithm from ``low`` to ``high``, in a fixed disorder, the first ``empty`` of them none."""
    B, low, high = c["B"], c["low"], c["high"]
    lens = [high if B == 1 else int(round(low * (high / low) ** (i / (B - 1)))) for i in range(B)]
    lens = [lens[(i * 7 + 3) % B] if B % 7 else lens[B - 1 - i] for i in range(B)]
    return [0 if i < c["empty"] and B > c["empty"] else n for i, n in enumerate(lens)]


def _pages(c):
    return sum(-(-n // c["page"]) for n in _lengths(c))


def _padded_bytes(c):
    """K or V of all sequences in 32 bits, padded to the longest: what the plain form holds."""
    return 0 if c["kind"] == "rotary" else 4 * c["B"] * c["high"] * c["Hkv"] * c["D"]


def _randn(gen, *shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _keys(gen, *shape, dtype):
    """Keys as a model produces them: unit variance with one value in a hundred eight times as large."""
    x = _randn(gen, *shape, dtype=dtype)
    return x.mul_(torch.where(torch.rand(shape, generator=gen, device="cuda", dtype=dtype) < 0.01, 8.0, 1.0))


def _tables(context, rotary_dim):
    """cos and sin of p * 10^6^(-2j / rotary_dim), formed in 64 bits (the angles of far positions)."""
    inv = 1.0e6 ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device="cuda") / rotary_dim)
    angle = torch.arange(context, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _norm_weights(c, gen):
    return [1.0 + 0.1 * _randn(gen, c["D"], dtype=torch.float32) if c["norm"] else None for _ in range(2)]


def _pack(codes, bits):
    """Byte j of a 4-bit row: value j in the high, value j + D / 2 in the low half."""
    if bits == 8:
        return codes
    half = codes.shape[-1] // 2
    return codes[..., :half] << 4 | codes[..., half:]


def _pool(c, gen):
    """Pages full of rows, the sequences' tables and, behind what a table needs, -1. One page more than the sequences use."""
    lens = torch.tensor(_lengths(c), device="cuda")
    n, page, bits = _pages(c) + 1, c["page"], BITS[c["store"]]
    used = -(-lens // page)
    width = max(1, -(-max(c.get("capacity", 0), c["high"]) // page))
    at = torch.arange(width, device="cuda") < used[:, None]
    table = torch.full((c["B"], width), -1, dtype=torch.int32, device="cuda")
    table[at] = torch.randperm(n - 1, generator=gen, device="cuda").to(torch.int32)
    shape = (n, c["Hkv"], page, c["D"])
    s = {"table": table, "lens": lens.to(torch.int32), "quant": None, "bits": bits}
    if bits == 16:
        s["k"], s["v"] = _keys(gen, *shape, dtype=DTYPES[c["dtype"]]), _randn(gen, *shape, dtype=DTYPES[c["dtype"]])
        return s
    # rows from about -4 to 4 with zero points in the middle of the codes, as quantised rows have
    s["k"], s["v"] = (_pack(torch.randint(0, 1 << bits, shape, generator=gen, device="cuda", dtype=torch.uint8), bits) for _ in range(2))
    state = []
    for _ in range(2):
        state.append((6.0 + 2.0 * torch.rand(shape[:3], generator=gen, device="cuda")) / ((1 << bits) - 1))
        state.append(torch.randint((3 << bits) // 8, (5 << bits) // 8, shape[:3], generator=gen, device="cuda", dtype=torch.int32))
    s["quant"] = tuple(state)
    return s


def _slots(table, page, seq, pos):
    """Slot of token ``pos`` of sequence ``seq``: its page's first slot and its place there."""
    return table[seq, pos // page].long() * page + pos % page


def _prepare_rotary(c, gen):
    cos, sin = _tables(c["context"], c["rotary_dim"])
    n = c["tokens"]
    positions = torch.randint(0, c["context"], (n,), generator=gen, device="cuda", dtype=torch.int32)
    if c["padded"]:
        positions[n - c["padded"] :] = -1
    qw, kw = _norm_weights(c, gen)
    return {"qkv": _randn(gen, n, (c["Hq"] + 2 * c["Hkv"]) * c["D"], dtype=DTYPES[c["dtype"]]), "cos": cos, "sin": sin, "positions": positions, "qw": qw, "kw": kw,
            "interleaved": c["interleaved"]}


def _prepare_rows(c, gen, s):
    """The sequences' tokens, packed one sequence behind the other, and their slots."""
    lens = s["lens"].long()
    seq = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), lens)
    pos = torch.arange(seq.shape[0], device="cuda") - (lens.cumsum(0) - lens)[seq]
    dtype = DTYPES[c["dtype"]]
    # views of a projection's output, as a layer has them
    kv = torch.cat((_keys(gen, seq.shape[0], c["Hkv"], c["D"], dtype=dtype), _randn(gen, seq.shape[0], c["Hkv"], c["D"], dtype=dtype)), 1)
    s["key"], s["value"] = kv[:, : c["Hkv"]], kv[:, c["Hkv"] :]
    s["slots"] = _slots(s["table"], c["page"], seq, pos)


def _prepare_step(c, gen, s):
    last = (s["lens"] - 1).long()
    s["positions"] = last.to(torch.int32)
    s["slots"] = torch.where(last >= 0, _slots(s["table"], c["page"], torch.arange(c["B"], device="cuda"), last.clamp(min=0)), -1)
    s["cos"], s["sin"] = _tables(c["capacity"], c["D"])
    s["qw"], s["kw"] = (1.0 + 0.1 * _randn(gen, c["D"], dtype=torch.float32) for _ in range(2))
    s["interleaved"] = False
    s["qkv"] = _randn(gen, c["B"], (c["Hq"] + 2 * c["Hkv"]) * c["D"], dtype=DTYPES[c["dtype"]])


def prepare(case, seed):
    c, kind = case, case["kind"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _prepare_rotary(c, gen) if kind == "rotary" else _pool(c, gen)
    if kind in ("write", "store"):
        _prepare_rows(c, gen, s)
    if kind == "decode":
        s["q"] = _randn(gen, c["B"], c["Hq"], c["D"], dtype=DTYPES[c["dtype"]])
        s["lse"] = c["lse"]
    if kind == "step":
        _prepare_step(c, gen, s)
    return {**s, "kind": kind, "Hq": c["Hq"], "Hkv": c["Hkv"], "D": c["D"], "length": c.get("high"), "dtype": DTYPES[c["dtype"]], "scale": c["D"] ** -0.5}


# -- one pass -------------------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from keys_values_amd.attention import ops
    from keys_values_amd.kvcache import paged
    from keys_values_amd.longctx import ops as rows

    kind = s["kind"]
    if kind in ("rotary", "step"):
        rows.rotary_(s["qkv"], s["Hq"], s["Hkv"], s["D"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], s["positions"], interleaved=s["interleaved"])
        if kind == "rotary":
            return {"qkv": s["qkv"]}
        heads = s["qkv"].view(-1, s["Hq"] + 2 * s["Hkv"], s["D"])
        paged.paged_write(heads[:, s["Hq"] : -s["Hkv"]], heads[:, -s["Hkv"] :], s["k"], s["v"], s["slots"])
        out, _ = ops.paged_decode(heads[:, : s["Hq"]], s["k"], s["v"], s["table"], s["lens"], s["scale"])
        return {"qkv": s["qkv"], "out": out, "k": s["k"][:-1], "v": s["v"][:-1]}
    if kind == "decode":
        out, lse = ops.paged_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], s["scale"], return_lse=s["lse"], quant=s["quant"])
        return {"out": out, "lse": lse} if s["lse"] else {"out": out}
    if kind != "read":
        paged.paged_write(s["key"], s["value"], s["k"], s["v"], s["slots"], quant=s["quant"])
        if kind == "write":
            return {"k": s["k"][:-1], "v": s["v"][:-1]}
    k, v = paged.paged_read(s["k"], s["v"], s["table"], s["lens"], s["length"], head_size=s["D"], dtype=s["dtype"], quant=s["quant"])
    return {"k": k, "v": v}


def _plain(s):
    kind = s["kind"]
    if kind in ("rotary", "step"):
        _plain_rotary(s)
        if kind == "rotary":
            return {"qkv": s["qkv"]}
        heads = s["qkv"].view(-1, s["Hq"] + 2 * s["Hkv"], s["D"])
        _plain_write({**s, "key": heads[:, s["Hq"] : -s["Hkv"]], "value": heads[:, -s["Hkv"] :]})
        out, _ = _plain_decode({**s, "q": heads[:, : s["Hq"]]})
        return {"qkv": s["qkv"], "out": out, "k": s["k"][:-1], "v": s["v"][:-1]}
    if kind == "decode":
        out, lse = _plain_decode(s)
        return {"out": out, "lse": lse} if s["lse"] else {"out": out}
    if kind != "read":
        _plain_write(s)
        if kind == "write":
            return {"k": s["k"][:-1], "v": s["v"][:-1]}
    there = torch.arange(s["length"], device="cuda") < s["lens"][:, None]
    k, v = (torch.where(there[:, None, :, None], x[:, :, : s["length"]], 0.0).to(s["dtype"]) for x in _sequences(s))
    return {"k": k, "v": v}


def _plain_rotary(s):
    """Query and key heads x: x / (|x| / sqrt(D) + eps) * weight, then (a, b) -> (a cos - b sin, b cos + a sin) for its pairs. In place."""
    D, there = s["D"], (s["positions"] >= 0)[:, None, None]
    heads = s["qkv"].view(-1, s["Hq"] + 2 * s["Hkv"], D)
    x = heads[:, : -s["Hkv"]].float()
    if s["qw"] is not None:
        weight = torch.cat((s["qw"].expand(s["Hq"], D), s["kw"].expand(s["Hkv"], D)))
        x = x / (x.square().sum(-1, keepdim=True).sqrt() / D**0.5 + EPS) * weight
    half = s["cos"].shape[1]
    at = s["positions"].clamp(min=0).long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    if s["interleaved"]:
        a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half : 2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    y = torch.cat((turned, x[..., 2 * half :]), -1).to(heads.dtype)
    heads[:, : -s["Hkv"]] = torch.where(there, y, heads[:, : -s["Hkv"]])


def _plain_write(s):
    """Row i of key and value to slot ``slots[i]``; rows without one to the page that no sequence has."""
    n, Hkv, page, _ = s["k"].shape
    slots = torch.where(s["slots"] >= 0, s["slots"], (n - 1) * page)
    at, place = slots // page, slots % page
    for i, (x, pages) in enumerate(((s["key"], s["k"]), (s["value"], s["v"]))):
        if s["bits"] == 16:
            pages[at, :, place] = x
            continue
        x, top = x.float(), float((1 << s["bits"]) - 1)
        low, high = x.amin(-1), x.amax(-1)
        scale = ((high - low) / torch.full_like(low, top)).clamp(min=1.1920929e-07)  # by a number it would be a product with its reciprocal
        zero = -(low / scale).round().to(torch.int32)
        codes = ((x * (1.0 / scale)[..., None]).round() + zero[..., None]).clamp(0.0, top).to(torch.uint8)
        pages[at, :, place] = _pack(codes, s["bits"])
        s["quant"][2 * i][at, :, place] = scale
        s["quant"][2 * i + 1][at, :, place] = zero


def _sequences(s):
    """The sequences' K and V rows in 32 bits, (B, Hkv, whole pages of the longest, D)."""
    at = s["table"][:, : -(-s["length"] // s["k"].shape[2])].clamp(min=0).long()
    out = []
    for i, pages in enumerate((s["k"], s["v"])):
        x = pages[at]
        if s["bits"] == 4:
            x = torch.cat((x >> 4, x & 15), -1)
        if s["bits"] != 16:
            x = (x.to(torch.int32) - s["quant"][2 * i + 1][at][..., None]).float() * s["quant"][2 * i][at][..., None]
        out.append(x.float().transpose(1, 2).flatten(2, 3))
    return out


def _plain_decode(s):
    """out = softmax(scale q K^T) V over a sequence's first ``lens`` rows, and the base-2 logarithm of the sum; zero and -inf where there are none."""
    B, D = s["q"].shape[0], s["D"]
    k, v = _sequences(s)
    q = s["q"].float().view(B, s["Hkv"], -1, D)
    there = (torch.arange(k.shape[2], device="cuda") < s["lens"][:, None])[:, None, None]
    logits = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    logits = logits.masked_fill(~there, -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (logits - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = ((top + total.log()) / math.log(2.0)).flatten(1)
    return out.view(B, -1, D).to(s["dtype"]), lse


# -- what a pass cannot do without ------------------------------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    if kind == "rotary":
        n, d = c["tokens"] - c["padded"], c["D"]
        heads = c["Hq"] + c["Hkv"]
        return {"bytes": n * (4 * heads * d + 4 * c["rotary_dim"] + 4), "flops": n * heads * (3 * c["rotary_dim"] + (4 * d if c["norm"] else 0))}
    lens, bits = _lengths(c), BITS[c["store"]]
    rows = 2 * sum(lens) * c["Hkv"]
    row, kept = 2 * c["D"], c["D"] * bits // 8 + (0 if bits == 16 else 8)  # a row's bytes, and in its page
    table = 4 * (_pages(c) + c["B"])
    if kind == "write":
        return {"bytes": rows * (row + kept) + 8 * sum(lens), "flops": 0}
    if kind == "store":  # rows in, codes out; codes in, rows out
        return {"bytes": rows * (row + kept) + 8 * sum(lens) + rows * kept + 2 * c["B"] * c["Hkv"] * c["high"] * row + table, "flops": 8 * rows * c["D"]}
    if kind == "read":
        return {"bytes": rows * kept + 2 * c["B"] * c["Hkv"] * c["high"] * row + table, "flops": 0}
    attention = {"bytes": rows * kept + 2 * c["B"] * c["Hq"] * row + table, "flops": 4 * sum(lens) * c["Hq"] * c["D"]}
    if kind == "step":
        new = sum(n > 0 for n in lens)
        attention["bytes"] += new * (4 * (c["Hq"] + c["Hkv"]) * c["D"] + 4 * c["D"]) + new * 2 * c["Hkv"] * 2 * row
    return attention


# -- the definitions in 64 bits ---------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("rotary", "step"):
        qkv = _exact_rotary(s, case)
        if kind == "rotary":
            return {"qkv": qkv}
        # the operators hand each other rows of the model's type
        heads = qkv.to(s["dtype"]).double().view(-1, case["Hq"] + 2 * case["Hkv"], case["D"])
        key, value = heads[:, case["Hq"] : case["Hq"] + case["Hkv"]], heads[:, case["Hq"] + case["Hkv"] :]
        k, v = s["k"].double(), s["v"].double()
        for b in range(case["B"]):
            slot = int(s["slots"][b])
            if slot >= 0:
                k[slot // case["page"], :, slot % case["page"]] = key[b]
                v[slot // case["page"], :, slot % case["page"]] = value[b]
        out, _ = _exact_decode({**s, "k": k, "v": v, "q": heads[:, : case["Hq"]]}, case)
        return {"qkv": qkv, "out": out, "k": k[:-1], "v": v[:-1]}
    if kind == "decode":
        out, lse = _exact_decode(s, case)
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    if kind == "write":
        k, v, first = s["k"].double(), s["v"].double(), 0
        for b, n in enumerate(_lengths(case)):
            for page in range(-(-n // case["page"])):
                at, last = int(s["table"][b, page]), min(n, (page + 1) * case["page"])
                for pages, rows in ((k, s["key"]), (v, s["value"])):
                    pages[at, :, : last - page * case["page"]] = rows[first + page * case["page"] : first + last].double().transpose(0, 1)
            first += n
        return {"k": k[:-1], "v": v[:-1]}
    got = []
    for i, name in enumerate(("key", "value")):
        rows = torch.zeros(case["B"], case["Hkv"], case["high"], case["D"], dtype=torch.float64, device="cuda")
        first = 0
        for b, n in enumerate(_lengths(case)):
            if kind == "read":
                rows[b, :, :n] = _exact_rows(s, case, b, n, i)
            else:
                rows[b, :, :n] = _exact_round_trip(s[name][first : first + n].double(), (1 << s["bits"]) - 1).transpose(0, 1)
            first += n
        got.append(rows)
    return {"k": got[0], "v": got[1]}


def _exact_rotary(s, case):
    """Pairs as complex numbers, turned by cos + i sin."""
    D, rd, Hq, Hkv = case["D"], case["rotary_dim"] if case["kind"] == "rotary" else case["D"], case["Hq"], case["Hkv"]
    x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
    y = x[:, : Hq + Hkv].clone()
    if s["qw"] is not None:
        y /= torch.linalg.vector_norm(y, dim=-1, keepdim=True) * D**-0.5 + EPS
        y[:, :Hq] *= s["qw"].double()
        y[:, Hq:] *= s["kw"].double()
    at = s["positions"].long()
    turn = torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if s["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    x = x.clone()
    x[at >= 0, : Hq + Hkv] = y[at >= 0]
    return x.flatten(1)


def _exact_round_trip(x, top):
    """A code is a whole number, and values often lie on the border of two: which one it is follows from the 32-bit scale that the store
    keeps, from its 32-bit reciprocal and the 32-bit products with that, each rounded once."""

    def once(y):
        return y.float().double()

    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = torch.clamp(once(once(high - low) / top), min=2.0**-23)
    zero = -torch.round(once(low / scale))
    codes = torch.clamp(torch.round(once(x * once(1.0 / scale))) + zero, 0, top)
    return (codes - zero) * scale


def _exact_rows(s, case, b, n, i):
    """K (i = 0) or V (i = 1) rows of sequence b, (Hkv, n, D)."""
    pages = s["table"][b, : -(-n // case["page"])].long()
    x = (s["k"], s["v"])[i][pages]
    if s["bits"] < 16:
        if s["bits"] == 4:
            x = torch.cat((torch.div(x, 16, rounding_mode="floor"), x % 16), -1)
        x = (x.double() - s["quant"][2 * i + 1][pages].double()[..., None]) * s["quant"][2 * i][pages].double()[..., None]
    return x.double().permute(1, 0, 2, 3).reshape(case["Hkv"], -1, case["D"])[:, :n]


def _exact_decode(s, case):
    B, Hq, D = case["B"], case["Hq"], case["D"]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        k, v = (_exact_rows(s, case, b, n, i) for i in (0, 1))
        q = s["q"][b].double().reshape(case["Hkv"], -1, D)
        logits = torch.matmul(k, q.transpose(1, 2).contiguous()).transpose(1, 2) * D**-0.5
        out[b] = torch.matmul(torch.softmax(logits, -1), v).reshape(Hq, D)
        lse[b] = torch.logsumexp(logits, -1).reshape(Hq) / math.log(2.0)
    return out, lse
