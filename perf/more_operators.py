"""Workloads of a serving loop around the paged cache, and of rotary positions in training.

A case is one pass of something that such a program does on the GPU:

* ``resize``: sequences grow by new tokens, which get pages from a free list, positions and places, and
  then give the same tokens back (``paged_cache_resize`` twice): drafted tokens that are all rejected,
  or prompts that are admitted and evicted;
* ``rotary``: queries and keys are turned by the angles of their positions (``rotary_positions``),
  alone or with the gradients of both;
* ``chunk``: rows of new tokens go into a cache of 4-bit numbers, and everything the sequences hold comes
  back (``paged_cache_write``, ``paged_cache_read``);
* ``decode``: one new token of every sequence attends to all that its pages of 4-bit numbers hold
  (``paged_attention``).

The ranges: page tables of 1 to 16,384 sequences with up to 131,072 tokens each, of which 1 to 1,000,000
come in a pass; rows of 1 to 32,768 tokens with 1 to 64 heads of 16 to 256 numbers, all or a part of them
turned; caches of 1 to 128 sequences with 1 to 131,072 tokens, pages of 1 to 256 tokens, 1 to 16 heads of
keys shared by 1 to 16 heads of queries each, even widths of 16 to 256; float32, bfloat16 and float16.

A cache of 4-bit numbers holds, for every 32 neighbouring numbers of a row, the exponent of the smallest power of
two that brings the largest of them to 6, and the numbers divided by it as one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a
sign, the nearest one, half to even, two in a byte (the first in its low bits).

Sizes follow from the case alone; values, the order of the sequences and of the pages follow from the
seed.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}
_E2M1 = torch.float4_e2m1fn_x2
_E8M0 = torch.float8_e8m0fnu


def _resize(name, sequences, length, change, page):
    case = {"op": "resize", "sequences": sequences, "length": length, "change": change, "page": page}
    return case if name is None else {"name": name, **case}


def _rotary(name, tokens, heads, key_heads, width, dims, dtype, *, interleaved=False, furthest=8192, scaling="none",
            fused=False, train=False):
    case = {"op": "rotary", "tokens": tokens, "heads": heads, "key_heads": key_heads, "width": width, "dims": dims,
            "dtype": dtype, "interleaved": interleaved, "furthest": furthest, "scaling": scaling, "fused": fused,
            "train": train}
    return case if name is None else {"name": name, **case}


def _cache(name, op, sequences, length, heads, width, page, dtype, *, new=0, value_width=0, group=1, ragged=True,
           window=0):
    case = {"op": op, "sequences": sequences, "length": length, "new": new, "heads": heads, "group": group,
            "width": width, "value_width": value_width or width, "page": page, "dtype": dtype, "ragged": ragged,
            "window": window}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one drafted token for each sequence of a serving batch: a call of a few numbers, where latency counts
        _resize("resize step", 64, 4096, 1, 16),
        # up to five drafted tokens for each of very many short sequences
        _resize("resize drafts of many", 8192, 600, 5, 16),
        # a batch of long prompts: half a million tokens get their places
        _resize("resize prompts", 24, 100, 40000, 64),
        # the step between two tokens of a small batch: queries and keys as a fused projection leaves them
        _rotary("rotary tokens bf16", 24, 32, 8, 128, 128, "bf16", furthest=131072, fused=True),
        # a training step over packed texts
        _rotary("rotary train bf16", 16384, 32, 8, 128, 128, "bf16", train=True),
        # a long context by stretched angles, a part of every head, neighbours as pairs, an odd count of heads
        _rotary("rotary part f32", 5000, 13, 13, 80, 32, "f32", interleaved=True, furthest=1000000, scaling="ramp"),
        # the next 512 tokens of eight long prompts into a 4-bit cache, which their own attention reads back
        _cache("chunk e2m1 bf16", "chunk", 8, 8000, 8, 128, 64, "bf16", new=512),
        # prompts of up to 3,000 tokens into an empty cache, a width that is no multiple of 32
        _cache("prompts e2m1 f16", "chunk", 12, 0, 10, 72, 12, "f16", new=3000),
        # one sequence, just begun
        _cache("decode first tokens f16", "decode", 1, 17, 4, 64, 16, "f16"),
        # a serving batch of ragged lengths with shared key heads
        _cache("decode batch bf16", "decode", 64, 8192, 8, 128, 16, "bf16", group=4),
        # two very long sequences
        _cache("decode long bf16", "decode", 2, 131072, 8, 128, 64, "bf16", group=8, ragged=False),
        # a small float32 model: widths that are no multiples of 32, pages of 12 tokens, the last tokens only
        _cache("decode window f32", "decode", 12, 1500, 6, 40, 12, "f32", value_width=24, group=2, window=1000),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["resize", "rotary", "rotary", "chunk", "decode", "decode", "decode"])
    if op == "resize":
        sequences, length, change = _log_int(rng, 1, 16384), _log_int(rng, 1, 131072), _log_int(rng, 1, 40000)
        page = rng.choice([1, 8, 12, 16, 16, 32, 64, 128, 256])
        while sequences * change > 1_000_000:
            change = change * 2 // 3
        while sequences * -(-(length + change) // page) > 8_000_000:
            length = length * 2 // 3
        return _resize(None, sequences, max(1, length), max(1, change), page)
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "rotary":
        tokens, key_heads, group = _log_int(rng, 1, 32768), _log_int(rng, 1, 16), rng.choice([1, 1, 2, 3, 4, 8])
        width = _log_int(rng, 16, 256)
        width = max(16, width // 8 * 8) if rng.random() < 0.8 else width
        group = min(group, 64 // key_heads)
        while tokens * key_heads * (group + 1) * width > 40_000_000:
            tokens = tokens * 2 // 3
        dims = width // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, width // 2)
        return _rotary(None, tokens, key_heads * group, key_heads, width, dims, dtype,
                       interleaved=rng.random() < 0.5, furthest=max(tokens, _log_int(rng, 1000, 4_000_000)),
                       scaling=rng.choice(["none", "linear", "base", "ramp"]), fused=rng.random() < 0.5,
                       train=rng.random() < 0.5)

    def width():
        w = _log_int(rng, 16, 256)
        return max(16, w // 32 * 32) if w >= 32 and rng.random() < 0.6 else w // 2 * 2

    page = rng.choice([1, 8, 12, 16, 16, 32, 64, 128, 256])
    sequences, length, heads = _log_int(rng, 1, 128), _log_int(rng, 1, 131072), _log_int(rng, 1, 16)
    group, widths = rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), (width(), width())
    if rng.random() < 0.7:
        widths = (widths[0], widths[0])
    most = 400_000_000 if op == "decode" else 120_000_000
    while sequences * length * heads * (widths[0] + widths[1]) > most:
        if length > sequences:
            length = length * 2 // 3
        else:
            sequences = sequences * 2 // 3
    ragged = sequences > 1 and rng.random() < 0.7
    if op == "decode":
        return _cache(None, op, sequences, length, heads, widths[0], page, dtype, value_width=widths[1], group=group,
                      ragged=ragged, window=_log_int(rng, 16, 4096) if rng.random() < 0.2 else 0)
    new = rng.choice([1, 1, max(1, length // 8)])
    return _cache(None, op, sequences, length, heads, widths[0], page, dtype, new=new, value_width=widths[1],
                  ragged=ragged)


# ------------------------------------------------------------------------------------------------
# Sizes, which follow from the case alone


def _spread(longest, sequences, ragged):
    """Lengths of the sequences: all alike, or from an eighth of the longest up to it."""
    if not ragged or sequences == 1 or longest <= 1:
        return [longest] * sequences
    low = max(1, longest // 8)
    return [low + (longest - low) * i // (sequences - 1) for i in range(sequences)]


def _lengths(case):
    """(tokens of every sequence before the pass, new tokens)."""
    if case["op"] == "resize":
        return (_spread(case["length"], case["sequences"], True),
                [1 + i * 7919 % case["change"] for i in range(case["sequences"])])
    before = _spread(case["length"], case["sequences"], case["ragged"]) if case["length"] else [0] * case["sequences"]
    new = _spread(case["new"], case["sequences"], case["ragged"]) if case["new"] else [0] * len(before)
    return before, new


def _held(case):
    """Bytes of one token and head in a 4-bit cache."""
    return sum(w // 2 + -(-w // 32) for w in (case["width"], case["value_width"]))


def work(case):
    if case["op"] == "rotary":
        rows = case["tokens"] * (case["heads"] + case["key_heads"])
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * rows * case["width"] * _SIZES[case["dtype"]] + 8 * case["tokens"]) +
                4 * case["dims"], "flops": 3 * passes * rows * case["dims"]}
    before, new = _lengths(case)
    page = case["page"]
    pages = sum(-(-(b + n) // page) for b, n in zip(before, new))
    if case["op"] == "resize":
        moved = pages - sum(-(-b // page) for b in before)
        return {"bytes": 2 * (24 * len(before) + 16 * moved) + 8 * len(before) + 16 * sum(new), "flops": 0}
    row, held = case["width"] + case["value_width"], _held(case)
    size, lists = _SIZES[case["dtype"]], 8 * pages + 24 * len(before)
    if case["op"] == "decode":
        seen = sum(min(b, case["window"]) if case["window"] else b for b in before)
        queries = len(before) * case["heads"] * case["group"]
        return {"bytes": seen * case["heads"] * held + queries * row * size + lists,
                "flops": 2 * seen * case["heads"] * case["group"] * row}
    tokens = 2 * sum(new) + sum(before)
    return {"bytes": tokens * case["heads"] * (row * size + held) + lists, "flops": 0}


# ------------------------------------------------------------------------------------------------
# What a program has in hand before the call


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _prepare_resize(case, gen):
    before, new = _lengths(case)
    page, count = case["page"], len(before)
    order = torch.randperm(count, generator=gen, device="cuda")
    before = torch.tensor(before, device="cuda")[order]
    new = torch.tensor(new, device="cuda")[order]
    held = (before + page - 1) // page
    room = int(((before + new + page - 1) // page).max()) + 1
    pages = int(((before + new + page - 1) // page).sum()) + 5
    ids = torch.randperm(pages, generator=gen, device="cuda")
    used = torch.arange(room, device="cuda") < held[:, None]
    table = torch.full((count, room), -1, dtype=torch.long, device="cuda")
    table[used] = ids[:int(held.sum())]
    free = torch.full((pages,), -1, dtype=torch.long, device="cuda")
    free[:pages - int(held.sum())] = ids[int(held.sum()):]
    return {"page_table": table, "lengths": before, "change": new, "free_pages": free,
            "free_count": torch.tensor([pages - int(held.sum())], device="cuda"), "tokens": int(new.sum())}


def _frequencies(case):
    """Radians from one position to the next, a number for each pair, in 64 bits."""
    dims, base = case["dims"], 10000.0
    index = torch.arange(0, dims, 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "base":
        base = base * 8.0 ** (dims / max(dims - 2, 1))
    plain = base ** (-index / dims)
    if case["scaling"] == "linear":
        return plain / 8.0
    if case["scaling"] != "ramp":
        return plain
    # pairs that turn more than 32 times within 4,096 positions stay, those that turn less than once are stretched
    share = ((4096.0 * plain / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return plain * share + plain / 8.0 * (1.0 - share)


def _prepare_rotary(case, gen):
    tokens, heads, key_heads, width = (case[k] for k in ("tokens", "heads", "key_heads", "width"))
    dtype = _DTYPES[case["dtype"]]
    # runs of up to 500 tokens, each from a position of its own on
    at = torch.arange(tokens, device="cuda")
    starts = torch.randint(0, max(1, case["furthest"] - 500), (tokens // 500 + 1,), generator=gen, device="cuda")
    state = {"positions": starts[at // 500] + at % 500, "frequencies": _frequencies(case),
             "magnitude": 0.1 * math.log(8.0) + 1.0 if case["scaling"] == "ramp" else 1.0}
    if case["fused"] and not case["train"]:
        rows = torch.randn(tokens, heads + 2 * key_heads, width, generator=gen, device="cuda").to(dtype)
        state["query"], state["key"] = rows[:, :heads], rows[:, heads:heads + key_heads]
    else:
        state["query"] = torch.randn(tokens, heads, width, generator=gen, device="cuda").to(dtype)
        state["key"] = torch.randn(tokens, key_heads, width, generator=gen, device="cuda").to(dtype)
    if case["train"]:
        for kind in ("query", "key"):
            state["grad_" + kind] = torch.randn(state[kind].shape, generator=gen, device="cuda").to(dtype)
            state[kind].requires_grad_(True)
    return state


def _quantise(x):
    """(codes, two in a byte, exponents with a bias of 127) of rows along the last dimension."""
    groups = torch.nn.functional.pad(x.float(), (0, -x.size(-1) % 32)).unflatten(-1, (-1, 32))
    mantissa, exponent = torch.frexp(groups.abs().amax(-1, keepdim=True))
    exponent = torch.where(mantissa == 0, -127, exponent - 3 + (mantissa > 0.75).to(torch.int32)).clamp_min(-127)
    size = torch.ldexp(groups.abs(), -exponent)
    code = (size > 0.25).to(torch.uint8) + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5)
    code = code + (size >= 3.5) + (size > 5.0) + 8 * groups.signbit()
    code = code.to(torch.uint8).flatten(-2)[..., :x.size(-1)]
    return code[..., ::2] | code[..., 1::2] << 4, (exponent.squeeze(-1) + 127).to(torch.uint8)


def _rows_of_tokens(gen, shape):
    """Keys or values: every token and head has a magnitude of its own."""
    magnitude = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return torch.randn(*shape, generator=gen, device="cuda") * magnitude


def _prepare_cache(case, gen):
    dtype, page, heads = _DTYPES[case["dtype"]], case["page"], case["heads"]
    before, new = _lengths(case)
    order = torch.randperm(len(before), generator=gen, device="cuda").tolist()
    before, new = [before[i] for i in order], [new[i] for i in order]
    counts = [-(-(b + n) // page) for b, n in zip(before, new)]
    pages = sum(counts) + 3
    state = {
        "page_ptr": torch.tensor([0] + counts, device="cuda").cumsum(0),
        "page_idx": torch.randperm(pages, generator=gen, device="cuda")[:sum(counts)].contiguous(),
        "before": torch.tensor(before, device="cuda"),
        "max_length": max(b + n for b, n in zip(before, new)),
    }
    for kind, width in (("key", case["width"]), ("value", case["value_width"])):
        held = torch.empty(pages, heads, page, width // 2, dtype=torch.uint8, device="cuda")
        exponents = torch.empty(pages, heads, page, -(-width // 32), dtype=torch.uint8, device="cuda")
        block = max(1, (1 << 25) // (heads * page * width))
        for at in range(0, pages, block):
            rows = _rows_of_tokens(gen, (min(block, pages - at), heads, page, width)).to(dtype)
            held[at:at + block], exponents[at:at + block] = _quantise(rows)
        state[kind + "_pages"], state[kind + "_exponents"] = held.view(_E2M1), exponents.view(_E8M0)
    if case["op"] == "decode":
        shape = (len(before), heads * case["group"], case["width"])
        state["query"] = torch.randn(*shape, generator=gen, device="cuda").to(dtype)
        return state
    after = [b + n for b, n in zip(before, new)]
    state["key"] = _rows_of_tokens(gen, (sum(new), heads, case["width"])).to(dtype)
    state["value"] = _rows_of_tokens(gen, (sum(new), heads, case["value_width"])).to(dtype)
    state["new_ptr"] = torch.tensor([0] + new, device="cuda").cumsum(0)
    state["zero"] = torch.zeros(len(after), dtype=torch.long, device="cuda")
    state["all_ptr"] = torch.tensor([0] + after, device="cuda").cumsum(0)
    state["tokens"] = sum(after)
    return state


_PREPARE = {"resize": _prepare_resize, "rotary": _prepare_rotary, "chunk": _prepare_cache, "decode": _prepare_cache}


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, _generator(seed))
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------
# One pass


def run(state):
    case = state["case"]
    calls = _OWN if own else _PLAIN
    return calls[case["op"]](case, state)


# ---- through the framework


def _own_resize(case, state):
    import autosage_amd

    table, free, count = state["page_table"], state["free_pages"], state["free_count"]
    grown, token_ptr, positions, slots = autosage_amd.paged_cache_resize(
        table, state["lengths"], state["change"], free, count, page_size=case["page"], tokens=state["tokens"])
    back = autosage_amd.paged_cache_resize(table, grown, -state["change"], free, count, page_size=case["page"],
                                           tokens=0)
    return grown, token_ptr, positions, slots, back[0], table, free, count


def _own_rotary(case, state):
    import autosage_amd

    query, key = state["query"], state["key"]
    turned = autosage_amd.rotary_positions(query, key, state["positions"], state["frequencies"],
                                           interleaved=case["interleaved"], magnitude=state["magnitude"])
    if not case["train"]:
        return turned
    grads = torch.autograd.grad(turned, (query, key), (state["grad_query"], state["grad_key"]))
    return turned[0].detach(), turned[1].detach(), *grads


def _own_chunk(case, state):
    import autosage_amd

    held = {"key_exponents": state["key_exponents"], "value_exponents": state["value_exponents"]}
    autosage_amd.paged_cache_write(state["key"], state["value"], state["key_pages"], state["value_pages"],
                                   state["page_ptr"], state["page_idx"], state["new_ptr"], state["before"], **held)
    return autosage_amd.paged_cache_read(state["key_pages"], state["value_pages"], state["page_ptr"],
                                         state["page_idx"], state["all_ptr"], state["zero"], state["tokens"],
                                         dtype=_DTYPES[case["dtype"]], **held)


def _own_decode(case, state):
    import autosage_amd

    return autosage_amd.paged_attention(
        state["query"], state["key_pages"], state["value_pages"], state["page_ptr"], state["page_idx"],
        state["before"], scale=case["width"] ** -0.5, key_exponents=state["key_exponents"],
        value_exponents=state["value_exponents"], window=case["window"] or None, max_length=state["max_length"])


_OWN = {"resize": _own_resize, "rotary": _own_rotary, "chunk": _own_chunk, "decode": _own_decode}


# ---- in plain form


def _sums(x):
    return torch.nn.functional.pad(x.cumsum(0), (1, 0))


def _plain_resize(case, state):
    """The growth of all sequences, and the way back; there are pages enough for all."""
    table, lengths, change = state["page_table"], state["lengths"], state["change"]
    free, count, page = state["free_pages"], state["free_count"], case["page"]
    grown, token_ptr = lengths + change, _sums(change)
    held, after = (lengths + page - 1) // page, (grown + page - 1) // page
    first = _sums(after - held)[:-1]
    entry = torch.arange(table.size(1), device=table.device)
    taken = (entry >= held[:, None]) & (entry < after[:, None])
    index = count - 1 - (first[:, None] + entry - held[:, None])
    table.copy_(torch.where(taken, free[index.clamp(0, free.numel() - 1)], table))
    count -= (after - held).sum()
    sequence = torch.repeat_interleave(torch.arange(change.numel(), device=table.device), change,
                                       output_size=state["tokens"])
    positions = lengths[sequence] + torch.arange(state["tokens"], device=table.device) - token_ptr[sequence]
    slots = table[sequence, positions // page] * page + positions % page
    # the way back: the first page that goes is the last one on the list
    gone = count + (after - held).sum() - 1 - (first[:, None] + entry - held[:, None])
    free.scatter_(0, torch.where(taken, gone, free.numel() - 1).flatten(),
                  torch.where(taken, table, free[-1]).flatten())
    table.masked_fill_(taken, -1)
    count += (after - held).sum()
    return grown, token_ptr, positions, slots, grown - change, table, free, count


def _plain_turn(x, cos, sin, interleaved, dims):
    x = x.detach()
    part, rest = x[..., :dims].float(), x[..., dims:]
    a, b = (part[..., ::2], part[..., 1::2]) if interleaved else (part[..., :dims // 2], part[..., dims // 2:])
    turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1 if interleaved else -2)
    return torch.cat((turned.flatten(-2).to(x.dtype), rest), -1)


def _plain_rotary(case, state):
    angle = state["positions"].double()[:, None, None] * state["frequencies"]
    cos, sin = (angle.cos() * state["magnitude"]).float(), (angle.sin() * state["magnitude"]).float()
    turned = [_plain_turn(state[kind], cos, sin, case["interleaved"], case["dims"]) for kind in ("query", "key")]
    if not case["train"]:
        return tuple(turned)
    grads = [_plain_turn(state["grad_" + kind], cos, -sin, case["interleaved"], case["dims"])
             for kind in ("query", "key")]
    return (*turned, *grads)


def _plain_places(page_ptr, page_idx, token_ptr, start, tokens, page):
    """(page, place in it) of every token, sequence after sequence from its start on."""
    counts = token_ptr[1:] - token_ptr[:-1]
    sequence = torch.repeat_interleave(torch.arange(counts.numel(), device=start.device), counts, output_size=tokens)
    position = start[sequence] + torch.arange(tokens, device=start.device) - token_ptr[sequence]
    return page_idx[page_ptr[sequence] + position // page], position % page


def _values(codes, exponents):
    """The numbers that codes stand for, in 32 bits."""
    sizes = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    sizes = torch.cat((sizes, -sizes))
    numbers = torch.stack((sizes[(codes & 15).int()], sizes[(codes >> 4).int()]), -1).flatten(-2)
    exponent = (exponents.int() - 127).repeat_interleave(32, -1)[..., :numbers.size(-1)]
    return torch.ldexp(numbers, exponent)


def _plain_chunk(case, state):
    new = _plain_places(state["page_ptr"], state["page_idx"], state["new_ptr"], state["before"], state["key"].size(0),
                        case["page"])
    every = _plain_places(state["page_ptr"], state["page_idx"], state["all_ptr"], state["zero"], state["tokens"],
                          case["page"])

    def one(kind):
        pages, exponents = (state[kind + what].view(torch.uint8) for what in ("_pages", "_exponents"))
        pages[new[0], :, new[1]], exponents[new[0], :, new[1]] = _quantise(state[kind])
        return _values(pages[every[0], :, every[1]], exponents[every[0], :, every[1]]).to(_DTYPES[case["dtype"]])

    return one("key"), one("value")


def _plain_decode(case, state):
    """Every sequence padded to the longest: scores, softmax and sum in 32 bits."""
    heads, group, page = case["heads"], case["group"], case["page"]
    length, longest = state["before"][:, None], state["max_length"]
    time = torch.arange(longest, device=length.device)
    seen = time < length
    if case["window"]:
        seen = seen & (time >= length - case["window"])
    first, last = state["page_ptr"][:-1, None], state["page_ptr"][1:, None]
    where = state["page_idx"][torch.minimum(first + time // page, last - 1)]
    place = (time % page).expand_as(where)

    def rows(kind):
        codes, exponents = (state[kind + what].view(torch.uint8)[where, :, place] for what in ("_pages", "_exponents"))
        return _values(codes, exponents).transpose(1, 2)

    query = state["query"].float().view(-1, heads, group, case["width"])
    scores = (query @ rows("key").transpose(2, 3).contiguous()) * case["width"] ** -0.5
    scores = torch.where(seen[:, None, None], scores, float("-inf"))
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    values = torch.where(seen[:, None, :, None], rows("value"), 0.0)
    out = (weights @ values) / weights.sum(-1, keepdim=True)
    return out.reshape(-1, heads * group, case["value_width"]).to(_DTYPES[case["dtype"]])


_PLAIN = {"resize": _plain_resize, "rotary": _plain_rotary, "chunk": _plain_chunk, "decode": _plain_decode}


# ------------------------------------------------------------------------------------------------
# From the definition, in 64 bits


def _exact_rotary(case, state):
    """A pair is a complex number, multiplied by magnitude * exp(i * position * frequency)."""
    angle = state["positions"].double()[:, None] * state["frequencies"][None]
    turn = torch.polar(torch.full_like(angle, state["magnitude"]), angle)[:, None]
    n = case["dims"] // 2

    def turned(x, by):
        out = x.detach().double().clone()
        pairs = out[..., :2 * n]
        pairs = pairs.unflatten(-1, (n, 2)) if case["interleaved"] else pairs.unflatten(-1, (2, n)).transpose(-1, -2)
        result = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * by)
        out[..., :2 * n] = (result if case["interleaved"] else result.transpose(-1, -2)).flatten(-2)
        return out

    found = [turned(state["query"], turn), turned(state["key"], turn)]
    if case["train"]:
        found += [turned(state["grad_query"], turn.conj()), turned(state["grad_key"], turn.conj())]
    return tuple(found)


def _exact_rows(x):
    """The numbers that a 4-bit cache holds for ``x``: multiples of a step that doubles with the number, from half of
    the group's power of two on."""
    x = torch.nn.functional.pad(x.double(), (0, -x.size(-1) % 32)).unflatten(-1, (-1, 32))
    largest = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(largest.clamp_min(2.0 ** -140) / 6.0)).clamp_min(-127))
    scale = torch.where(largest > 6.0 * scale, 2 * scale, scale)
    scale = torch.where(largest <= 3.0 * scale, scale / 2, scale).clamp_min(2.0 ** -127)
    step = scale * torch.where(x.abs() < 2.0 * scale, 0.5, torch.where(x.abs() < 4.0 * scale, 1.0, 2.0))
    return (torch.round(x / step) * step).flatten(-2)


def _exact_held(state, kind, pages):
    """Rows of the pages, ``[pages, heads, page size, width]``, one number after another."""
    codes = state[kind + "_pages"].view(torch.uint8)[pages]
    both = torch.stack((codes % 16, codes // 16), -1).flatten(-2).double()
    size = both % 8
    # 0, 1 are halves; from 2 on there is one bit behind the leading one
    size = torch.where(size < 2, size / 2, (2 + size % 2) / 2 * torch.exp2(torch.floor(size / 2) - 1))
    scale = torch.exp2(state[kind + "_exponents"].view(torch.uint8)[pages].double() - 127)
    scale = torch.repeat_interleave(scale, 32, -1)[..., :size.size(-1)]
    return torch.where(both >= 8, -size, size) * scale


def _exact_chunk(case, state):
    before, new = state["before"].tolist(), state["new_ptr"].tolist()
    pages, ptr, size = state["page_idx"], state["page_ptr"].tolist(), case["page"]
    results = []
    for kind in ("key", "value"):
        back = []
        for b, length in enumerate(before):
            mine = pages[ptr[b]:ptr[b] + -(-length // size)]
            held = _exact_held(state, kind, mine).transpose(1, 2).flatten(0, 1)[:length]
            fresh = _exact_rows(state[kind][new[b]:new[b + 1]])[..., :state[kind].size(-1)]
            back += [held, fresh]
        results.append(torch.cat(back))
    return tuple(results)


def _exact_decode(case, state):
    heads, group, size = case["heads"], case["group"], case["page"]
    ptr = state["page_ptr"].tolist()
    out = torch.zeros(case["sequences"], heads * group, case["value_width"], dtype=torch.float64, device="cuda")
    for b, length in enumerate(state["before"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        mine = state["page_idx"][ptr[b] + first // size:ptr[b] + -(-length // size)]
        key, value = (_exact_held(state, kind, mine).transpose(1, 2).flatten(0, 1)[first % size:][:length - first]
                      for kind in ("key", "value"))
        for g in range(heads * group):
            score = (key[:, g // group] * state["query"][b, g].double()).sum(1) / math.sqrt(case["width"])
            out[b, g] = (torch.softmax(score, 0)[:, None] * value[:, g // group]).sum(0)
    return out


_EXACT = {"rotary": _exact_rotary, "chunk": _exact_chunk, "decode": _exact_decode}


def exact(case, seed):
    # whole numbers have no value in more bits
    return _EXACT[case["op"]](case, prepare(case, seed)) if case["op"] in _EXACT else None
