"""
The operators of sparse attention over a paged cache, each as its users call it, beside a plain form of the same mathematics:

``append``  ``kvcache.paged.paged_append``: queries of a ragged batch rotated in place, its keys rotated on their way to their slots, its values to theirs;
            plain pages, or pages of codes and then the sequences' rows back (``paged_read``), as a later chunk's attention takes them.
``bounds``  ``kvcache.paged.paged_bounds``: the lowest and the highest of a page's keys, value by value.
``select``  ``attention.ops.paged_select``: the pages that a query attends to, by the largest product with it that their bounds allow.
``attend``  ``attention.ops.paged_decode_chosen``: one new token a sequence over its chosen pages.
``step``    the four that a layer calls for one new token a sequence: append, bounds of the page written to, select, attend.

A case is a dict of plain values; the lengths of its sequences follow from it alone (see ``_lengths``). Shapes are those of the benchmark's
configurations (32 / 8 heads of 128, sequences to 131072 tokens, 8-bit and 4-bit stores), of the tests (other numbers of heads, head sizes 64 and 256,
float16) and what lies between them.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BITS = {"plain": 16, "u8": 8, "u4": 4}
HEADS = [(32, 8), (32, 8), (8, 2), (28, 4), (24, 8), (32, 4), (16, 8), (8, 8), (16, 1)]  # query heads / KV heads
EPS = 1.0e-6
MAX_BYTES = 1.6e9


def _case(name, kind, B, heads, D, low, high, page, store="plain", dtype="bf16", empty=0, **more):
    return {"name": name, "kind": kind, "B": B, "Hq": heads[0], "Hkv": heads[1], "D": D, "low": low, "high": high, "page": page, "store": store, "dtype": dtype,
            "empty": empty, **more}


def _append(name, B, heads, D, low, high, page, rotary_dim, interleaved, norm, store="plain", dtype="bf16", each=0, padded=0):
    """``each``: the newest tokens of a sequence that are appended, 0: all; ``padded``: rows without a token behind them."""
    return _case(name, "append", B, heads, D, low, high, page, store, dtype, rotary_dim=rotary_dim, interleaved=interleaved, norm=norm, each=each, padded=padded)


def listed():
    return [
        # one new token for each of 32 sequences: what a layer writes in a step of generation
        _append("append_tokens", 32, (32, 8), 128, 500, 6000, 16, 128, False, True, each=1),
        # the packed prompts of a serving batch
        _append("append_prompts", 5, (32, 8), 128, 1024, 8192, 64, 128, False, True),
        # prompts into 4-bit pages and their rows back; interleaved pairs in a part of the head, padding behind the last token
        _append("append_codes", 7, (28, 4), 128, 101, 2047, 32, 64, True, False, store="u4", dtype="fp16", padded=77),
        # the page that a step of generation has written to
        _case("bounds_tokens", "bounds", 32, (32, 8), 128, 500, 6000, 16, empty=2, tokens=1),
        # all pages of a batch of prompts
        _case("bounds_prompts", "bounds", 16, (32, 8), 128, 4096, 16384, 16, tokens=16384),
        # generation for one user at the benchmark's longest context: latency is everything
        _case("select_one", "select", 1, (32, 8), 128, 131072, 131072, 16, count=64, first=1, last=1),
        # a serving batch of very different lengths
        _case("select_ragged", "select", 48, (28, 4), 128, 300, 131072, 16, dtype="fp16", empty=3, count=128, first=2, last=4),
        # generation for one user
        _case("attend_one", "attend", 1, (32, 8), 128, 65536, 65536, 16, count=64, lse=False),
        # a serving batch on 8-bit pages
        _case("attend_u8", "attend", 64, (32, 8), 128, 2000, 16384, 64, store="u8", empty=3, count=48, lse=True),
        # many heads over one KV head of a float16 model, 4-bit pages
        _case("attend_u4", "attend", 48, (16, 1), 64, 3000, 50000, 32, store="u4", dtype="fp16", count=65, lse=True),
        # one layer's share of a step of generation for 32 sequences
        _case("step", "step", 32, (32, 8), 128, 500, 16384, 16, empty=2, count=64, first=1, last=2),
        # the same for 8 sequences of the benchmark's decode configuration, 8-bit pages
        _case("step_long", "step", 8, (32, 8), 128, 131072, 131072, 32, store="u8", count=128, first=1, last=1),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; no more work, rows or pages than the largest of the listed ones."""
    while True:
        case = _draw(rng)
        pages = _pages(case) * case["Hkv"]  # (page, head) pairs: of bounds, and of K and V
        if case["kind"] == "select" and max(_of(case, n) for n in _lengths(case)) <= case["count"]:
            continue  # nothing to choose
        rows = 0 if case["kind"] == "select" else pages * case["page"] * case["D"] * BITS[case["store"]] // 4
        if work(case)["bytes"] <= 3.6e8 and rows <= MAX_BYTES and pages * case["D"] <= 1.3e8 and _padded(case) <= 6.0e8:
            return case


def _draw(rng):
    kind = rng.choices(["append", "bounds", "select", "attend", "step"], [22, 14, 22, 24, 18])[0]
    heads = rng.choice(HEADS)
    D = rng.choice([64, 128, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([16, 16, 32, 64, 128])
    store = rng.choice(["plain", "plain", "u8", "u4"])
    high = _log_int(rng, 8 * page if kind == "select" else 1, {"append": 16384, "bounds": 32768}.get(kind, 131072))
    low = min(high, rng.choice([high, _log_int(rng, 1, high)]))
    B = _log_int(rng, 1, 16 if kind in ("append", "bounds") else 128)
    count = _log_int(rng, 4, min(256, high // page // 2) if kind == "select" else 256)
    if kind == "append":
        each = 0 if store != "plain" else rng.choice([0, 1])
        # a 4-bit code is a large part of a row's span: heads are not normalised there, since another order of the squares' sum moves values over codes' borders
        case = _append("", B if each == 0 else 8 * B, heads, D, low, high, page, rng.choice([D, D, D // 2, D // 4]), rng.random() < 0.4, store != "u4" and rng.random() < 0.5,
                       store, dtype, each, rng.choice([0, 0, _log_int(rng, 1, 200)]))
    else:
        empty = rng.choice([0, 0, B // 8])
        if kind == "bounds":
            more = {"tokens": rng.choice([1, high, _log_int(rng, 1, high)])}
        elif kind == "attend":
            more = {"count": count, "lse": rng.random() < 0.5}
        else:
            first = rng.choice([0, 1, 1, 2])
            more = {"count": count, "first": first, "last": rng.randint(1, min(8, count - first - 1))}
        case = _case("", kind, B, heads, D, low, high, page, "plain" if kind == "select" else store, dtype, empty, **more)
    del case["name"]
    return case


# -- inputs ---------------------------------------------------------------------------------------------------


def _lengths(c):
    """Tokens of the sequences: even over the logarithm from ``low`` to ``high``, in a fixed disorder, the first ``empty`` of them none."""
    B, low, high = c["B"], c["low"], c["high"]
    lens = [high if B == 1 else int(round(low * (high / low) ** (i / (B - 1)))) for i in range(B)]
    lens = [lens[(i * 7 + 3) % B] if B % 7 else lens[B - 1 - i] for i in range(B)]
    return [0 if i < c["empty"] and B > c["empty"] else n for i, n in enumerate(lens)]


def _of(c, n):
    """Pages of n tokens."""
    return -(-n // c["page"])


def _pages(c):
    return sum(_of(c, n) for n in _lengths(c))


def _read(c):
    """Tokens that are attended to for one KV head: those of ``count`` pages, the last of which is not full."""
    return sum(n if _of(c, n) <= c["count"] else (c["count"] - 1) * c["page"] + n - (_of(c, n) - 1) * c["page"] for n in _lengths(c))


def _padded(c):
    """Values that the plain form holds at once, padded to the longest sequence."""
    B, h, D = c["B"], c["Hkv"], c["D"]
    if c["kind"] == "append":
        return 0 if c["each"] else B * h * c["high"] * D
    if c["kind"] == "bounds":
        return B * h * min(c["high"], c["tokens"] + 2 * c["page"]) * D
    scores = 0 if c["kind"] == "attend" else 2 * B * h * _of(c, c["high"]) * D
    return max(scores, 0 if c["kind"] == "select" else B * h * min(c["count"], _of(c, c["high"])) * c["page"] * D)


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


def _pack(codes, bits):
    """Byte j of a 4-bit row: value j in the high, value j + D / 2 in the low half."""
    if bits == 8:
        return codes
    half = codes.shape[-1] // 2
    return codes[..., :half] << 4 | codes[..., half:]


def _tables_of_pages(c, gen):
    """The sequences' tables over a pool of one page more than they use; behind what a sequence needs, -1."""
    lens = torch.tensor(_lengths(c), device="cuda")
    n, used = _pages(c) + 1, -(-lens // c["page"])
    at = torch.arange(max(1, _of(c, c["high"])), device="cuda") < used[:, None]
    table = torch.full(at.shape, -1, dtype=torch.int32, device="cuda")
    table[at] = torch.randperm(n - 1, generator=gen, device="cuda").to(torch.int32)
    return {"table": table, "lens": lens.to(torch.int32), "quant": None, "bits": BITS[c["store"]], "pages": n}


def _fill(c, gen, s):
    """Pages full of rows. The keys of a page, which come from one stretch of a text, are nearer to each other than to those of others."""
    n, page, bits = s["pages"], c["page"], s["bits"]
    shape, middle = (n, c["Hkv"], page, c["D"]), (n, c["Hkv"], 1, c["D"])
    if bits == 16:
        dtype = DTYPES[c["dtype"]]
        s["k"], s["v"] = _keys(gen, *shape, dtype=dtype).add_(_randn(gen, *middle, dtype=dtype), alpha=0.5), _randn(gen, *shape, dtype=dtype)
        return
    # rows from about -4 to 4 with zero points in the middle of the codes, as quantised rows have
    half, state = 1 << (bits - 1), []
    for name in ("k", "v"):
        codes = torch.randint(0, half, shape, generator=gen, device="cuda", dtype=torch.uint8)
        codes += torch.randint(0, half + 1, middle if name == "k" else shape, generator=gen, device="cuda", dtype=torch.uint8)
        s[name] = _pack(codes, bits)
        state.append((6.0 + 2.0 * torch.rand(shape[:3], generator=gen, device="cuda")) / ((1 << bits) - 1))
        state.append(torch.randint((3 << bits) // 8, (5 << bits) // 8, shape[:3], generator=gen, device="cuda", dtype=torch.int32))
    s["quant"] = tuple(state)


def _slots(table, page, seq, pos):
    """Slot of token ``pos`` of sequence ``seq``: its page's first slot and its place there."""
    return table[seq, pos // page].long() * page + pos % page


def _prepare_append(c, gen, s):
    """The newest tokens, packed one sequence behind the other, their positions and slots."""
    lens = s["lens"].long()
    new = lens.clamp(max=c["each"]) if c["each"] else lens
    seq = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), new)
    pos = (lens - new)[seq] + torch.arange(seq.shape[0], device="cuda") - (new.cumsum(0) - new)[seq]
    none = torch.full((c["padded"],), -1, device="cuda")
    s["positions"] = torch.cat((pos, none)).to(torch.int32)
    s["slots"] = torch.cat((_slots(s["table"], c["page"], seq, pos), none))
    s["cos"], s["sin"] = _tables(c["high"], c["rotary_dim"])
    s["qw"], s["kw"] = (1.0 + 0.1 * _randn(gen, c["D"], dtype=torch.float32) if c["norm"] else None for _ in range(2))
    s["interleaved"] = c["interleaved"]
    s["qkv"] = _randn(gen, s["slots"].shape[0], (c["Hq"] + 2 * c["Hkv"]) * c["D"], dtype=DTYPES[c["dtype"]])


def _prepare_step(c, gen, s):
    last = (s["lens"] - 1).long()
    s["positions"] = last.to(torch.int32)
    s["slots"] = torch.where(last >= 0, _slots(s["table"], c["page"], torch.arange(c["B"], device="cuda"), last.clamp(min=0)), -1)
    s["cos"], s["sin"] = _tables(c["high"], c["D"])
    # the heads of a step are not normalised: queries that another order of a sum has moved may choose another page
    s["qw"], s["kw"], s["interleaved"] = None, None, False
    s["qkv"] = _randn(gen, c["B"], (c["Hq"] + 2 * c["Hkv"]) * c["D"], dtype=DTYPES[c["dtype"]])
    # the bounds that earlier steps have left
    s["bounds"] = torch.zeros(s["pages"], c["Hkv"], 2, c["D"], dtype=DTYPES[c["dtype"]], device="cuda")
    rows = _rows(s, s["k"], 0, torch.arange(s["pages"], device="cuda"))
    s["bounds"][:, :, 0], s["bounds"][:, :, 1] = rows.amin(2).to(s["bounds"].dtype), rows.amax(2).to(s["bounds"].dtype)


def _prepare_select(c, gen, s):
    """Bounds of keys around a middle of the page's own."""
    shape = (s["pages"], c["Hkv"], c["D"])
    middle, reach = 0.7 * _randn(gen, *shape, dtype=torch.float32), 1.2 + torch.rand(shape, generator=gen, device="cuda")
    s["bounds"] = torch.stack((middle - reach, middle + reach), 2).to(DTYPES[c["dtype"]])
    s["q"] = _randn(gen, c["B"], c["Hq"], c["D"], dtype=DTYPES[c["dtype"]])


def _prepare_attend(c, gen, s):
    """Any pages, the first and the last among them, in order."""
    used, count = -(-s["lens"] // c["page"]), c["count"]
    P = max(count, s["table"].shape[1])
    at = torch.arange(P, device="cuda")
    weight = torch.rand(c["B"], c["Hkv"], P, generator=gen, device="cuda")
    weight[:, :, 0] = 2.0
    weight[(at == used[:, None] - 1)[:, None].expand_as(weight)] = 2.0
    weight[(at >= used[:, None])[:, None].expand_as(weight)] = -1.0
    best = weight.topk(count, -1)
    chosen = torch.where(best.values < 0.0, P, best.indices).sort(-1).values
    s["chosen"] = torch.where(chosen == P, -1, chosen).to(torch.int32)
    s["q"] = _randn(gen, c["B"], c["Hq"], c["D"], dtype=DTYPES[c["dtype"]])
    s["lse"] = c["lse"]


def prepare(case, seed):
    c, kind = case, case["kind"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = _tables_of_pages(c, gen)
    if kind != "select":
        _fill(c, gen, s)
    if kind == "append":
        _prepare_append(c, gen, s)
    elif kind == "bounds":
        s["bounds"] = torch.zeros(s["pages"], c["Hkv"], 2, c["D"], dtype=DTYPES[c["dtype"]], device="cuda")
    elif kind == "select":
        _prepare_select(c, gen, s)
    elif kind == "attend":
        _prepare_attend(c, gen, s)
    else:
        _prepare_step(c, gen, s)
    return {**s, "kind": kind, "Hq": c["Hq"], "Hkv": c["Hkv"], "D": c["D"], "page": c["page"], "length": c["high"], "dtype": DTYPES[c["dtype"]], "scale": c["D"] ** -0.5,
            "tokens": c.get("tokens", 1), "count": c.get("count"), "first": c.get("first"), "last": c.get("last")}


# -- one pass -------------------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from keys_values_amd.attention import ops
    from keys_values_amd.kvcache import paged

    kind = s["kind"]
    if kind in ("append", "step"):
        paged.paged_append(s["qkv"], s["Hq"], s["Hkv"], s["D"], s["qw"], s["kw"], EPS, s["cos"], s["sin"], s["positions"], s["k"], s["v"], s["slots"], quant=s["quant"],
                           interleaved=s["interleaved"])
        if kind == "append":
            if s["quant"] is None:
                return {"qkv": s["qkv"], "k": s["k"][:-1], "v": s["v"][:-1]}
            k, v = paged.paged_read(s["k"], s["v"], s["table"], s["lens"], s["length"], head_size=s["D"], dtype=s["dtype"], quant=s["quant"])
            return {"qkv": s["qkv"], "k": k, "v": v}
    if kind in ("bounds", "step"):
        paged.paged_bounds(s["k"], s["bounds"], s["table"], s["lens"], tokens=s["tokens"], quant=s["quant"])
        if kind == "bounds":
            return {"bounds": s["bounds"][:-1]}
    if kind == "attend":
        out, lse = ops.paged_decode_chosen(s["q"], s["k"], s["v"], s["table"], s["lens"], s["chosen"], s["scale"], return_lse=s["lse"], quant=s["quant"])
        return {"out": out, "lse": lse} if s["lse"] else {"out": out}
    q = s["q"] if kind == "select" else s["qkv"].view(-1, s["Hq"] + 2 * s["Hkv"], s["D"])[:, : s["Hq"]]
    chosen = ops.paged_select(q, s["bounds"], s["table"], s["lens"], s["page"], s["count"], first=s["first"], last=s["last"])
    if kind == "select":
        return {"chosen": chosen}
    out, lse = ops.paged_decode_chosen(q, s["k"], s["v"], s["table"], s["lens"], chosen, s["scale"], return_lse=True, quant=s["quant"])
    return {"qkv": s["qkv"], "bounds": s["bounds"][:-1], "chosen": chosen, "out": out, "lse": lse}


def _plain(s):
    kind = s["kind"]
    if kind in ("append", "step"):
        _plain_append(s)
        if kind == "append":
            if s["quant"] is None:
                return {"qkv": s["qkv"], "k": s["k"][:-1], "v": s["v"][:-1]}
            return dict(zip(("k", "v"), _plain_read(s)), qkv=s["qkv"])
    if kind in ("bounds", "step"):
        _plain_bounds(s)
        if kind == "bounds":
            return {"bounds": s["bounds"][:-1]}
    if kind == "attend":
        out, lse = _plain_attend(s, s["q"], s["chosen"])
        return {"out": out, "lse": lse} if s["lse"] else {"out": out}
    q = s["q"] if kind == "select" else s["qkv"].view(-1, s["Hq"] + 2 * s["Hkv"], s["D"])[:, : s["Hq"]]
    chosen = _plain_select(s, q)
    if kind == "select":
        return {"chosen": chosen}
    out, lse = _plain_attend(s, q, chosen)
    return {"qkv": s["qkv"], "bounds": s["bounds"][:-1], "chosen": chosen, "out": out, "lse": lse}


def _plain_append(s):
    """Query and key heads x: x / (|x| / sqrt(D) + eps) * weight, then (a, b) -> (a cos - b sin, b cos + a sin) for its pairs. Queries stay in place, keys of the
    model's type and values go to their slots; what has no position goes nowhere."""
    D, Hq, Hkv, there = s["D"], s["Hq"], s["Hkv"], s["positions"] >= 0
    heads = s["qkv"].view(-1, Hq + 2 * Hkv, D)
    x = heads[:, :-Hkv].float()
    if s["qw"] is not None:
        weight = torch.cat((s["qw"].expand(Hq, D), s["kw"].expand(Hkv, D)))
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
    heads[:, :Hq] = torch.where(there[:, None, None], y[:, :Hq], heads[:, :Hq])
    # rows without a slot to the page that no sequence has
    n, _, page, _ = s["k"].shape
    slots = torch.where(there & (s["slots"] >= 0), s["slots"], (n - 1) * page)
    at, place = slots // page, slots % page
    for i, (row, pages) in enumerate(((y[:, Hq:], s["k"]), (heads[:, -Hkv:], s["v"]))):
        if s["bits"] == 16:
            pages[at, :, place] = row
            continue
        row, top = row.float(), float((1 << s["bits"]) - 1)
        low, high = row.amin(-1), row.amax(-1)
        scale = ((high - low) / torch.full_like(low, top)).clamp(min=1.1920929e-07)  # by a number it would be a product with its reciprocal
        zero = -(low / scale).round().to(torch.int32)
        codes = ((row * (1.0 / scale)[..., None]).round() + zero[..., None]).clamp(0.0, top).to(torch.uint8)
        pages[at, :, place] = _pack(codes, s["bits"])
        s["quant"][2 * i][at, :, place] = scale
        s["quant"][2 * i + 1][at, :, place] = zero


def _rows(s, pages, i, at, head=()):
    """Rows of K (i = 0) or V (i = 1) pages, in 32 bits; ``head``: an index of heads beside that of pages, or all of them."""
    x, at = pages[(at, *head)], (at, *head)
    if s["bits"] == 16:
        return x.float()
    if s["bits"] == 4:
        x = torch.cat((x >> 4, x & 15), -1)
    return (x.to(torch.int32) - s["quant"][2 * i + 1][at][..., None]).float() * s["quant"][2 * i][at][..., None]


def _plain_read(s):
    """The sequences' rows in the model's type, zeros behind their ends."""
    at = s["table"].clamp(min=0).long()
    there = (torch.arange(s["length"], device="cuda") < s["lens"][:, None])[:, None, :, None]
    return [torch.where(there, _rows(s, pages, i, at).transpose(1, 2).flatten(2, 3)[:, :, : s["length"]], 0.0).to(s["dtype"]) for i, pages in enumerate((s["k"], s["v"]))]


def _plain_bounds(s):
    """Minimum and maximum over the rows of the pages that hold the sequences' last ``tokens`` tokens."""
    page, lens = s["page"], s["lens"][:, None].long()
    most = min(s["table"].shape[1], (s["tokens"] + 2 * page - 2) // page)  # pages that so many tokens lie in
    i = (lens - 1).div(page, rounding_mode="floor") - torch.arange(most, device="cuda")
    there = (i >= 0) & ((i + 1) * page > lens - s["tokens"]) & (lens > 0)
    i = i.clamp(min=0)
    at = torch.where(there, s["table"].gather(1, i).long(), s["pages"] - 1)
    rows = _rows(s, s["k"], 0, at)
    behind = (i[..., None] * page + torch.arange(page, device="cuda") >= lens[..., None])[:, :, None, :, None]
    s["bounds"][at, :, 0] = rows.masked_fill(behind, math.inf).amin(3).to(s["dtype"])
    s["bounds"][at, :, 1] = rows.masked_fill(behind, -math.inf).amax(3).to(s["dtype"])


def _plain_select(s, q):
    """A page's score: the largest over the group's heads of sum_d max(q_d low_d, q_d high_d), in 64 bits, rounded to 32, since it decides between pages."""
    B, P, count = q.shape[0], s["table"].shape[1], s["count"]
    used, i = -(-s["lens"] // s["page"])[:, None], torch.arange(P, device="cuda")
    bounds = s["bounds"][s["table"].clamp(min=0).long()].transpose(1, 2).double()  # (B, Hkv, P, 2, D)
    q = q.double().view(B, s["Hkv"], -1, s["D"])
    top = torch.matmul(bounds[..., 1, :], q.clamp(min=0.0).transpose(-1, -2).contiguous())
    score = (top + torch.matmul(bounds[..., 0, :], q.clamp(max=0.0).transpose(-1, -2).contiguous())).amax(-1).float()
    always = (i < s["first"]) | (i >= used - s["last"])
    score = score.masked_fill(always[:, None], math.inf).masked_fill((i >= used)[:, None], -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True)
    chosen = torch.where(best.values == -math.inf, P, best.indices)[..., :count].sort(-1).values
    chosen = torch.where(chosen == P, -1, chosen).to(torch.int32)
    return torch.nn.functional.pad(chosen, (0, count - chosen.shape[-1]), value=-1)


def _plain_attend(s, q, chosen):
    """out = softmax(scale q K^T) V over the rows of the chosen pages, and the base-2 logarithm of the sum; zero and -inf where there are none."""
    B, Hkv, D, page = q.shape[0], s["Hkv"], s["D"], s["page"]
    chosen = chosen[..., : s["table"].shape[1]]
    i = chosen.clamp(min=0).long()
    at = s["table"][:, None].expand(B, Hkv, -1).gather(2, i).clamp(min=0).long()
    heads = torch.arange(Hkv, device="cuda")[:, None].expand_as(at)
    k, v = (_rows(s, pages, j, at, (heads,)).flatten(2, 3) for j, pages in enumerate((s["k"], s["v"])))
    there = (chosen >= 0)[..., None] & (i[..., None] * page + torch.arange(page, device="cuda") < s["lens"][:, None, None, None])
    logits = torch.matmul(q.float().view(B, Hkv, -1, D), k.transpose(-1, -2).contiguous()) * s["scale"]
    logits = logits.masked_fill(~there.flatten(2)[:, :, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (logits - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return out.view(B, -1, D).to(s["dtype"]), ((top + total.log()) / math.log(2.0)).flatten(1)


# -- what a pass cannot do without ------------------------------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    Hq, Hkv, D, bits, lens = c["Hq"], c["Hkv"], c["D"], BITS[c["store"]], _lengths(c)
    row, kept = 2 * D, D * bits // 8 + (0 if bits == 16 else 8)  # a row's bytes, and in its page

    def append(tokens, rotary_dim, norm):
        return {"bytes": tokens * ((2 * Hq + 2 * Hkv) * row + 2 * Hkv * kept + 4 * rotary_dim + 12), "flops": tokens * (Hq + Hkv) * (3 * rotary_dim + (4 * D if norm else 0))}

    def select(pages):
        return {"bytes": pages * (4 + Hkv * 2 * row) + c["B"] * (Hq * row + 4 * Hkv * c["count"]), "flops": 4 * pages * Hq * D}

    def attend(tokens):
        return {"bytes": 2 * tokens * Hkv * kept + c["B"] * (2 * Hq * row + 4 * Hkv * c["count"]), "flops": 4 * tokens * Hq * D}

    if kind == "append":
        w = append(sum(min(n, c["each"] or n) for n in lens), c["rotary_dim"], c["norm"])
        if bits < 16:  # and the rows back
            w["bytes"] += 2 * Hkv * (sum(lens) * kept + c["B"] * c["high"] * row)
        return w
    if kind == "bounds":
        tokens = [n - max(0, n - c["tokens"]) // c["page"] * c["page"] for n in lens]  # of the pages that are looked at
        return {"bytes": Hkv * (sum(tokens) * kept + sum(_of(c, n) for n in tokens) * 2 * row), "flops": 2 * Hkv * sum(tokens) * D}
    if kind == "select":
        return select(_pages(c))
    if kind == "attend":
        return attend(_read(c))
    new = sum(n > 0 for n in lens)
    parts = [append(new, D, False), {"bytes": Hkv * new * (c["page"] // 2 * kept + 2 * row), "flops": Hkv * new * c["page"] * D}, select(_pages(c)), attend(_read(c))]
    return {key: sum(p[key] for p in parts) for key in ("bytes", "flops")}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------


def exact(case, seed):
    kind = case["kind"]
    if kind == "select":  # whole numbers alone
        return None
    s = prepare(case, seed)
    if kind == "bounds":
        return {"bounds": _exact_bounds(s, case, s["bounds"].double())[:-1]}
    if kind == "attend":
        out, lse = _exact_attend(s, case, s["q"].double(), s["chosen"].tolist())
        return {"out": out, "lse": lse} if case["lse"] else {"out": out}
    return _exact_append(s, case) if kind == "append" else _exact_step(s, case)


def _once(y):
    return y.float().double()


def _exact_rotary(s, case, in_steps=False):
    """All heads with pairs as complex numbers, turned by cos + i sin; ``in_steps``: products and sums of 32 bits, each rounded once, which say on which side of a
    border of the model's type a value lies."""
    D, Hq, Hkv, rd = case["D"], case["Hq"], case["Hkv"], 2 * s["cos"].shape[1]
    x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D).clone()
    y = x[:, : Hq + Hkv].clone()
    if s["qw"] is not None:
        y /= torch.linalg.vector_norm(y, dim=-1, keepdim=True) * D**-0.5 + EPS
        y[:, :Hq] *= s["qw"].double()
        y[:, Hq:] *= s["kw"].double()
    at = s["positions"].long()
    c, d = s["cos"].double()[at][:, None], s["sin"].double()[at][:, None]
    first, second = (slice(0, rd, 2), slice(1, rd, 2)) if s["interleaved"] else (slice(0, rd // 2), slice(rd // 2, rd))
    if in_steps:
        a, b = y[..., first].clone(), y[..., second].clone()
        y[..., first], y[..., second] = _once(_once(a * c) - _once(b * d)), _once(_once(b * c) + _once(a * d))
    else:
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(c, d)
        y[..., first], y[..., second] = z.real, z.imag
    x[at >= 0, : Hq + Hkv] = y[at >= 0]
    return x


def _exact_codes(x, top):
    """Scale, zero point and codes of rows. A code is a whole number, and values often lie on the border of two: which one it is follows from the 32-bit scale
    that the store keeps, from its 32-bit reciprocal and the 32-bit products with that, each rounded once."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = torch.clamp(_once(_once(high - low) / top), min=2.0**-23)
    zero = -torch.round(_once(low / scale))
    return scale, zero, torch.clamp(torch.round(_once(x * _once(1.0 / scale))) + zero, 0, top)


def _queries(s, case, turned):
    """qkv with its queries turned, and its keys and values as they were."""
    heads = s["qkv"].double().view(-1, case["Hq"] + 2 * case["Hkv"], case["D"]).clone()
    heads[:, : case["Hq"]] = turned[:, : case["Hq"]]
    return heads.flatten(1)


def _exact_append(s, case):
    Hq, Hkv = case["Hq"], case["Hkv"]
    turned = _exact_rotary(s, case)
    new = {"k": turned[:, Hq : Hq + Hkv], "v": turned[:, Hq + Hkv :]}
    got = {"qkv": _queries(s, case, turned)}
    for name, rows in new.items():
        if s["quant"] is None:
            pages = s[name].double()
            for i, slot in enumerate(s["slots"].tolist()):
                if slot >= 0:
                    pages[slot // case["page"], :, slot % case["page"]] = rows[i]
            got[name] = pages[:-1]
            continue
        back, first = torch.zeros(case["B"], Hkv, case["high"], case["D"], dtype=torch.float64, device="cuda"), 0
        for b, n in enumerate(_lengths(case)):
            scale, zero, codes = _exact_codes(rows[first : first + n].to(s["dtype"]).double(), (1 << s["bits"]) - 1)
            back[b, :, :n] = ((codes - zero) * scale).transpose(0, 1)
            first += n
        got[name] = back
    return got


def _exact_page(s, i, at):
    """All rows of a K (i = 0) or V (i = 1) page, (Hkv, page, D)."""
    x = (s["k"], s["v"])[i][at]
    if s["bits"] == 4:
        x = torch.cat((torch.div(x, 16, rounding_mode="floor"), x % 16), -1)
    x = x.double()
    return x if s["bits"] == 16 else (x - s["quant"][2 * i + 1][at].double()[..., None]) * s["quant"][2 * i][at].double()[..., None]


def _exact_bounds(s, case, bounds):
    table = s["table"].tolist()
    for b, n in enumerate(_lengths(case)):
        for i in range(max(0, n - s["tokens"]) // case["page"], _of(case, n)):
            rows = _exact_page(s, 0, table[b][i])[:, : n - i * case["page"]]
            bounds[table[b][i]] = torch.stack((rows.min(1).values, rows.max(1).values), 1)
    return bounds


def _exact_attend(s, case, q, chosen):
    B, Hq, D, G = case["B"], case["Hq"], case["D"], case["Hq"] // case["Hkv"]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        for h in range(case["Hkv"] if n else 0):
            pages = torch.tensor([i for i in chosen[b][h] if i >= 0], device="cuda")
            at = s["table"][b, pages].long()
            keep = (pages[:, None] * case["page"] + torch.arange(case["page"], device="cuda") < n).flatten()
            k, v = (_exact_page({**s, "k": s["k"][:, h], "v": s["v"][:, h], "quant": s["quant"] and [x[:, h] for x in s["quant"]]}, i, at).flatten(0, 1)[keep] for i in (0, 1))
            mine = slice(h * G, h * G + G)
            logits = torch.matmul(k, q[b, mine].t().contiguous()).t() * D**-0.5
            out[b, mine] = torch.matmul(torch.softmax(logits, -1), v)
            lse[b, mine] = torch.logsumexp(logits, -1) / math.log(2.0)
    return out, lse


def _exact_step(s, case):
    Hq, Hkv, page, G = case["Hq"], case["Hkv"], case["page"], case["Hq"] // case["Hkv"]
    # the operators hand each other rows of the model's type
    handed = _exact_rotary(s, case, in_steps=True).to(s["dtype"]).double()
    lens, table = _lengths(case), s["table"].tolist()
    s["k"], s["v"] = (x.double() if s["bits"] == 16 else x.clone() for x in (s["k"], s["v"]))
    for b, n in enumerate(lens):
        if n == 0:
            continue
        at, place = table[b][(n - 1) // page], (n - 1) % page
        for i, rows in enumerate((handed[b, Hq : Hq + Hkv], handed[b, Hq + Hkv :])):
            if s["bits"] < 16:
                scale, zero, codes = _exact_codes(rows, (1 << s["bits"]) - 1)
                s["quant"][2 * i][at, :, place], s["quant"][2 * i + 1][at, :, place] = scale[..., 0].float(), zero[..., 0].to(torch.int32)
                rows = _pack(codes.to(torch.uint8), s["bits"])
            (s["k"], s["v"])[i][at, :, place] = rows
    bounds = _exact_bounds(s, case, s["bounds"].double())
    kept = bounds.to(s["dtype"]).double()
    chosen = []
    for b, n in enumerate(lens):
        P = _of(case, n)
        own_pages = kept[s["table"][b, :P].long()]  # (P, Hkv, 2, D)
        q = handed[b, :Hq].view(Hkv, G, 1, 1, -1)
        chosen.append([])
        for h in range(Hkv):
            score = (own_pages[:, h, None] * q[h].view(1, G, 1, -1)).amax(2).sum(-1).amax(1).float().tolist() if P else []
            order = sorted(range(P), key=lambda i: (not (i < case["first"] or i >= P - case["last"]), -score[i], i))
            chosen[-1].append(sorted(order[: case["count"]]))
    out, lse = _exact_attend(s, case, handed[:, :Hq], chosen)
    return {"qkv": _queries(s, case, _exact_rotary(s, case)), "bounds": bounds[:-1], "out": out, "lse": lse}
