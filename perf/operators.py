"""Workloads of the relative position bias and of the paged key-value cache.

A case is one pass of something that a program with attention over lists of keys does on the GPU:

* ``bias``: the learned bias of the distance between the two nodes of every edge of a CSR graph, by
  buckets, for every head (``csr_position_bias``), alone or with the table's gradient;
* ``write``: the keys and values of new tokens go into the pages of their sequences
  (``paged_cache_write``), 1 token of every sequence or whole prompts;
* ``chunk``: a chunk of a prompt goes into a cache of 8-bit floating-point numbers, and everything the
  sequences hold so far comes back (``paged_cache_write``, ``paged_cache_read``), which is what the
  chunk's own attention reads;
* ``read``: everything the sequences hold comes back (``paged_cache_read``);
* ``decode``: one new token of every sequence attends to all that its pages hold (``paged_attention``).

The ranges: graphs of 1,000 to 1,000,000 nodes with 4 to 64 edges each, 1 to 16 heads and 8 to 128
buckets; caches of 1 to 128 sequences with 1 to 131,072 tokens, pages of 1 to 256 tokens, 1 to 16 heads
of keys shared by 1 to 16 heads of queries each, widths of 16 to 256, in float32, bfloat16, float16 and
e4m3 with a power-of-two scale for each token and head.

Sizes follow from the case alone; values, the order of the sequences and of the pages follow from the
seed.
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}
_E4M3 = torch.float8_e4m3fn


def _bias(name, tokens, degree, heads, buckets, max_distance, dtype, *, bidirectional=True, shuffled=False,
          train=False):
    case = {"op": "bias", "tokens": tokens, "degree": degree, "heads": heads, "buckets": buckets,
            "max_distance": max_distance, "dtype": dtype, "bidirectional": bidirectional, "shuffled": shuffled,
            "train": train}
    return case if name is None else {"name": name, **case}


def _cache(name, op, sequences, length, heads, width, page, dtype, *, new=0, value_width=0, quantised=False,
           ragged=True):
    case = {"op": op, "sequences": sequences, "length": length, "new": new, "heads": heads, "width": width,
            "value_width": value_width or width, "page": page, "dtype": dtype, "quantised": quantised,
            "ragged": ragged}
    return case if name is None else {"name": name, **case}


def _decode(name, sequences, length, heads, group, width, page, dtype, *, value_width=0, quantised=False,
            ragged=True, window=0, buckets=0, max_distance=0):
    case = {"op": "decode", "sequences": sequences, "length": length, "heads": heads, "group": group,
            "width": width, "value_width": value_width or width, "page": page, "dtype": dtype,
            "quantised": quantised, "ragged": ragged, "window": window, "buckets": buckets,
            "max_distance": max_distance}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # inference over a text of 16k tokens with a local and a few far edges for each, eight heads
        _bias("bias f32", 16384, 64, 8, 32, 128, "f32"),
        # a training step of a causal model over a short text in 16 bits, an odd count of heads
        _bias("bias train bf16", 30000, 24, 5, 32, 256, "bf16", bidirectional=False, train=True),
        # a training step over a large graph whose nodes are numbered in another order than they stand in
        _bias("bias train shuffled 1M", 1000000, 16, 4, 64, 4096, "f32", shuffled=True, train=True),
        # the step between two tokens of a small batch: one key and one value a sequence
        _cache("write tokens bf16", "write", 24, 300, 8, 128, 16, "bf16", new=1),
        # prompts of up to 4,000 tokens into an empty cache, a width that is no multiple of 16
        _cache("write prompts f16", "write", 16, 0, 12, 72, 32, "f16", new=4000),
        # the next 512 tokens of eight long prompts into an 8-bit cache
        _cache("chunk e4m3 bf16", "chunk", 8, 8000, 8, 128, 64, "bf16", new=512, quantised=True),
        # a batch's whole cache of 8-bit numbers comes back in 16 bits
        _cache("read e4m3 f16", "read", 48, 4096, 8, 64, 16, "f16", quantised=True),
        # a few sequences come back from a cache with odd pages
        _cache("read f32", "read", 5, 900, 3, 40, 12, "f32"),
        # one sequence, just begun: the smallest call, where latency counts
        _decode("decode first tokens f16", 1, 17, 4, 1, 64, 16, "f16"),
        # a serving batch of ragged lengths with shared key heads
        _decode("decode batch bf16", 64, 8192, 8, 4, 128, 16, "bf16"),
        # two very long sequences from an 8-bit cache
        _decode("decode long e4m3", 2, 131072, 8, 8, 128, 64, "bf16", quantised=True, ragged=False),
        # a small float32 model with a position bias, odd widths and pages
        _decode("decode bias f32", 12, 1500, 6, 2, 40, 12, "f32", value_width=24, buckets=32, max_distance=128),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["bias", "bias", "write", "chunk", "read", "decode", "decode", "decode"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "bias":
        tokens, degree, heads = _log_int(rng, 1000, 1000000), _log_int(rng, 4, 64), _log_int(rng, 1, 16)
        while tokens * degree * (8 + 4 * heads) > 350_000_000:
            tokens = tokens * 2 // 3
        buckets = 2 * _log_int(rng, 4, 64)
        return _bias(None, tokens, degree, heads, buckets, buckets * _log_int(rng, 2, 64), dtype,
                     bidirectional=rng.random() < 0.6, shuffled=rng.random() < 0.3, train=rng.random() < 0.5)

    def width():
        w = _log_int(rng, 16, 256)
        return max(16, w // 8 * 8) if rng.random() < 0.7 else w

    page = rng.choice([1, 8, 12, 16, 16, 32, 64, 128, 256])
    sequences, length, heads = _log_int(rng, 1, 128), _log_int(rng, 1, 131072), _log_int(rng, 1, 16)
    group, widths = rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), (width(), width())
    if rng.random() < 0.7:
        widths = (widths[0], widths[0])
    while sequences * length * heads * (widths[0] + widths[1]) > 150_000_000:
        if length > sequences:
            length = length * 2 // 3
        else:
            sequences = sequences * 2 // 3
    quantised = op == "chunk" or (op != "write" and rng.random() < 0.4)
    ragged = sequences > 1 and rng.random() < 0.7
    if op == "decode":
        biased = rng.random() < 0.3
        return _decode(None, sequences, length, heads, group, widths[0], page, dtype, value_width=widths[1],
                       quantised=quantised, ragged=ragged,
                       window=_log_int(rng, 16, 4096) if rng.random() < 0.2 else 0,
                       buckets=32 if biased else 0, max_distance=_log_int(rng, 64, 4096) if biased else 0)
    new = 0 if op == "read" else rng.choice([1, 1, max(1, length // 8)])
    return _cache(None, op, sequences, length if op != "write" else min(length, 2000), heads, widths[0], page,
                  dtype, new=new, value_width=widths[1], quantised=quantised, ragged=ragged)


# ------------------------------------------------------------------------------------------------
# Sizes, which follow from the case alone


def _spread(total_of_one, sequences, ragged):
    """Lengths of the sequences: all alike, or from an eighth of the longest up to it."""
    if not ragged or sequences == 1 or total_of_one <= 1:
        return [total_of_one] * sequences
    low = max(1, total_of_one // 8)
    return [low + (total_of_one - low) * i // (sequences - 1) for i in range(sequences)]


def _lengths(case):
    """(tokens in the cache before the pass, new tokens) of every sequence."""
    before = _spread(case["length"], case["sequences"], case["ragged"]) if case["length"] else [0] * case["sequences"]
    new = _spread(case.get("new", 0), case["sequences"], case["ragged"]) if case.get("new", 0) else [0] * len(before)
    return before, new


def work(case):
    size = _SIZES[case["dtype"]]
    if case["op"] == "bias":
        edges = case["tokens"] * case["degree"]
        fixed = 8 * (case["tokens"] + 1) + (8 * case["tokens"] if case["shuffled"] else 0)
        table = case["buckets"] * case["heads"] * size
        passes = 2 if case["train"] else 1
        return {"bytes": fixed + 8 * edges + passes * (edges * case["heads"] * size + table),
                "flops": edges * case["heads"] if case["train"] else 0}
    before, new = _lengths(case)
    row = case["width"] + case["value_width"]
    held = row + 2 if case["quantised"] else row * size
    pages = sum(-(-(b + n) // case["page"]) for b, n in zip(before, new))
    lists = 8 * pages + 24 * case["sequences"]
    if case["op"] == "decode":
        seen = sum(min(b, case["window"]) if case["window"] else b for b in before)
        queries = case["sequences"] * case["heads"] * case["group"]
        return {"bytes": seen * case["heads"] * held + queries * row * size + lists,
                "flops": 2 * seen * case["heads"] * case["group"] * row}
    written = sum(new) * case["heads"] * (row * size + held)
    back = sum(b + n for b, n in zip(before, new)) * case["heads"] * (row * size + held)
    if case["op"] == "write":
        return {"bytes": written + lists, "flops": 0}
    if case["op"] == "read":
        return {"bytes": back + lists, "flops": 0}
    return {"bytes": written + back + lists, "flops": 0}


# ------------------------------------------------------------------------------------------------
# What a program has in hand before the call


def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _graph(case, gen):
    """Rows of ``degree`` edges: three quarters of them near (distances spread over their logarithm up
    to 64), the rest anywhere in the text; earlier nodes only where the model is causal."""
    n, degree = case["tokens"], case["degree"]
    rows = torch.arange(n, device="cuda").repeat_interleave(degree)
    u = torch.rand(rows.numel(), generator=gen, device="cuda")
    near = torch.arange(rows.numel(), device="cuda") % degree < (3 * degree + 3) // 4
    distance = torch.where(near, 65.0 ** u - 1.0, u * n).to(torch.long)
    if case["bidirectional"]:
        sign = torch.randint(0, 2, (rows.numel(),), generator=gen, device="cuda") * 2 - 1
        cols = (rows + sign * distance) % n
    else:
        cols = rows - distance % (rows + 1)
    positions = None
    if case["shuffled"]:
        positions = torch.randperm(n, generator=gen, device="cuda")
        node = torch.empty_like(positions)
        node[positions] = torch.arange(n, device="cuda")
        rows, cols = node[rows], node[cols]
    keys = torch.sort(rows * n + cols).values
    crow = torch.arange(n + 1, device="cuda") * degree
    return crow, keys % n, positions


def _prepare_bias(case, gen):
    crow, col, positions = _graph(case, gen)
    dtype = _DTYPES[case["dtype"]]
    table = (0.5 * torch.randn(case["buckets"], case["heads"], generator=gen, device="cuda")).to(dtype)
    grad = None
    if case["train"]:
        table.requires_grad_(True)
        grad = torch.randn(case["heads"], col.numel(), generator=gen, device="cuda").to(dtype)
    return {"crow": crow, "col": col, "positions": positions, "table": table, "grad": grad}


def _quantise(x):
    """(codes, exponents) of rows along the last dimension: the smallest power of two that brings the
    row's largest magnitude to 448 at most, and the numbers divided by it, rounded to e4m3."""
    x = x.float()
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    exponent = torch.where(mantissa == 0, -126, exponent - 9 + (mantissa > 0.875).to(torch.int32)).clamp_min(-126)
    return torch.ldexp(x, -exponent).to(_E4M3), exponent.squeeze(-1).to(torch.int8)


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
        held = torch.empty(pages, heads, page, width, dtype=_E4M3 if case["quantised"] else dtype, device="cuda")
        exponents = torch.empty(pages, heads, page, dtype=torch.int8, device="cuda") if case["quantised"] else None
        block = max(1, (1 << 26) // (heads * page * width))
        for at in range(0, pages, block):
            rows = _rows_of_tokens(gen, (min(block, pages - at), heads, page, width)).to(dtype)
            if case["quantised"]:
                codes, scale = _quantise(rows)
                held[at:at + block].view(torch.uint8).copy_(codes.view(torch.uint8))
                exponents[at:at + block] = scale
            else:
                held[at:at + block] = rows
        state[kind + "_pages"], state[kind + "_exponents"] = held, exponents
    if case["op"] == "decode":
        shape = (len(before), heads * case["group"], case["width"])
        state["query"] = torch.randn(*shape, generator=gen, device="cuda").to(dtype)
        state["table"] = None
        if case["buckets"]:
            state["table"] = (0.5 * torch.randn(case["buckets"], shape[1], generator=gen, device="cuda")).to(dtype)
        return state
    if sum(new):
        state["key"] = _rows_of_tokens(gen, (sum(new), heads, case["width"])).to(dtype)
        state["value"] = _rows_of_tokens(gen, (sum(new), heads, case["value_width"])).to(dtype)
        state["new_ptr"] = torch.tensor([0] + new, device="cuda").cumsum(0)
    if case["op"] != "write":
        after = [b + n for b, n in zip(before, new)]
        state["zero"] = torch.zeros(len(after), dtype=torch.long, device="cuda")
        state["all_ptr"] = torch.tensor([0] + after, device="cuda").cumsum(0)
        state["tokens"] = sum(after)
    return state


def prepare(case, seed):
    gen = _generator(seed)
    state = _prepare_bias(case, gen) if case["op"] == "bias" else _prepare_cache(case, gen)
    state["case"] = case
    return state


# ------------------------------------------------------------------------------------------------
# One pass


def run(state):
    case = state["case"]
    calls = _OWN if own else _PLAIN
    return calls[case["op"]](case, state)


# ---- through the framework


def _own_bias(case, state):
    import autosage_amd

    bias = autosage_amd.csr_position_bias(state["crow"], state["col"], state["table"],
                                          max_distance=case["max_distance"], bidirectional=case["bidirectional"],
                                          positions=state["positions"])
    if not case["train"]:
        return bias
    return bias.detach(), torch.autograd.grad(bias, state["table"], state["grad"])[0]


def _own_write(case, state):
    import autosage_amd

    autosage_amd.paged_cache_write(state["key"], state["value"], state["key_pages"], state["value_pages"],
                                   state["page_ptr"], state["page_idx"], state["new_ptr"], state["before"],
                                   key_exponents=state["key_exponents"], value_exponents=state["value_exponents"])
    return state["key_pages"], state["value_pages"]


def _own_read(case, state):
    import autosage_amd

    return autosage_amd.paged_cache_read(state["key_pages"], state["value_pages"], state["page_ptr"],
                                         state["page_idx"], state["all_ptr"], state["zero"], state["tokens"],
                                         dtype=_DTYPES[case["dtype"]], key_exponents=state["key_exponents"],
                                         value_exponents=state["value_exponents"])


def _own_chunk(case, state):
    _own_write(case, state)
    return _own_read(case, state)


def _own_decode(case, state):
    import autosage_amd

    return autosage_amd.paged_attention(
        state["query"], state["key_pages"], state["value_pages"], state["page_ptr"], state["page_idx"],
        state["before"], scale=case["width"] ** -0.5, key_exponents=state["key_exponents"],
        value_exponents=state["value_exponents"], window=case["window"] or None, bias_table=state["table"],
        max_distance=case["max_distance"] or None, bidirectional=False, max_length=state["max_length"])


_OWN = {"bias": _own_bias, "write": _own_write, "read": _own_read, "chunk": _own_chunk, "decode": _own_decode}


# ---- in plain form


def _borders(buckets, max_distance):
    """The smallest distance of every bucket from 1 on.  Half of the buckets hold one distance each; of the
    others, number j begins where (distance / half) ** rest reaches (max_distance / half) ** j, in integers."""
    half = buckets // 2
    rest = buckets - half
    borders = list(range(1, half + 1))
    for j in range(1, rest):
        goal = half ** (rest - j) * max_distance ** j
        low, high = half, max_distance
        while low < high:
            middle = (low + high) // 2
            if middle ** rest >= goal:
                high = middle
            else:
                low = middle + 1
        borders.append(low)
    return borders


def _plain_buckets(relative, buckets, max_distance, bidirectional):
    one_side = buckets // 2 if bidirectional else buckets
    distance = relative.abs() if bidirectional else (-relative).clamp_min(0)
    bucket = torch.zeros_like(distance, dtype=torch.int32)
    for border in _borders(one_side, max_distance):
        bucket += distance >= border
    if bidirectional:
        bucket += (relative > 0).to(torch.int32) * one_side
    return bucket.long()


def _plain_bias(case, state):
    crow, col, table = state["crow"], state["col"], state["table"].detach()
    counts = crow[1:] - crow[:-1]
    rows = torch.repeat_interleave(torch.arange(counts.numel(), device=col.device), counts, output_size=col.numel())
    positions = state["positions"]
    relative = col - rows if positions is None else positions[col] - positions[rows]
    bucket = _plain_buckets(relative, case["buckets"], case["max_distance"], case["bidirectional"])
    bias = table.t()[:, bucket]
    if not case["train"]:
        return bias
    # sums of 1,024 edges in 32 bits, as products with each edge's bucket, and their sum in 64
    total = torch.zeros(case["heads"], case["buckets"], dtype=torch.float64, device=col.device)
    numbers = torch.arange(case["buckets"], device=col.device)
    for at in range(0, col.numel(), 1 << 22):
        grad = state["grad"][:, at:at + (1 << 22)].float()
        rest = -grad.size(1) % 1024
        member = torch.nn.functional.pad(bucket[at:at + (1 << 22)], (0, rest), value=-1).view(-1, 1024, 1) == numbers
        grad = torch.nn.functional.pad(grad, (0, rest)).view(grad.size(0), -1, 1024).transpose(0, 1).contiguous()
        total += (grad @ member.float()).sum(0, dtype=torch.float64)
    return bias, total.t().to(table.dtype)


def _plain_places(page_ptr, page_idx, token_ptr, start, tokens, page):
    """(page, place in it) of every token, sequence after sequence from its start on."""
    counts = token_ptr[1:] - token_ptr[:-1]
    sequence = torch.repeat_interleave(torch.arange(counts.numel(), device=start.device), counts, output_size=tokens)
    position = start[sequence] + torch.arange(tokens, device=start.device) - token_ptr[sequence]
    return page_idx[page_ptr[sequence] + position // page], position % page


def _plain_write(case, state):
    where, place = _plain_places(state["page_ptr"], state["page_idx"], state["new_ptr"], state["before"],
                                 state["key"].size(0), case["page"])
    for kind in ("key", "value"):
        if case["quantised"]:
            codes, exponents = _quantise(state[kind])
            state[kind + "_pages"].view(torch.uint8)[where, :, place] = codes.view(torch.uint8)
            state[kind + "_exponents"][where, :, place] = exponents
        else:
            state[kind + "_pages"][where, :, place] = state[kind]
    return state["key_pages"], state["value_pages"]


def _plain_read(case, state):
    where, place = _plain_places(state["page_ptr"], state["page_idx"], state["all_ptr"], state["zero"],
                                 state["tokens"], case["page"])
    found = []
    for kind in ("key", "value"):
        if case["quantised"]:
            codes = state[kind + "_pages"].view(torch.uint8)[where, :, place].view(_E4M3).float()
            exponents = state[kind + "_exponents"][where, :, place].to(torch.int32)
            found.append(torch.ldexp(codes, exponents[..., None]).to(_DTYPES[case["dtype"]]))
        else:
            found.append(state[kind + "_pages"][where, :, place])
    return tuple(found)


def _plain_chunk(case, state):
    _plain_write(case, state)
    return _plain_read(case, state)


def _plain_decode(case, state):
    """Blocks of sequences, each padded to the longest: scores, softmax and sum in 32 bits."""
    heads, group, page = case["heads"], case["group"], case["page"]
    lengths, longest = state["before"], state["max_length"]
    time = torch.arange(longest, device=lengths.device)
    query = state["query"].float()
    out = []
    block = max(1, (1 << 28) // max(1, longest * heads * (case["width"] + case["value_width"])))
    for at in range(0, case["sequences"], block):
        length = lengths[at:at + block, None]
        seen = time < length
        if case["window"]:
            seen = seen & (time >= length - case["window"])
        first, last = state["page_ptr"][:-1][at:at + block, None], state["page_ptr"][1:][at:at + block, None]
        where = state["page_idx"][torch.minimum(first + time // page, last - 1)]
        place = (time % page).expand_as(where)
        held = []
        for kind in ("key", "value"):
            if case["quantised"]:
                rows = state[kind + "_pages"].view(torch.uint8)[where, :, place].view(_E4M3).float()
                rows = torch.ldexp(rows, state[kind + "_exponents"][where, :, place].to(torch.int32)[..., None])
            else:
                rows = state[kind + "_pages"][where, :, place].float()
            held.append(rows.transpose(1, 2).contiguous())
        keys, values = held
        q = query[at:at + block].view(-1, heads, group, case["width"])
        scores = (q @ keys.transpose(2, 3).contiguous()) * case["width"] ** -0.5
        if state["table"] is not None:
            bucket = _plain_buckets(time - (length - 1), case["buckets"], case["max_distance"], False)
            bias = state["table"].float()[bucket].permute(0, 2, 1)
            scores = scores + bias.reshape(-1, heads, group, longest)
        scores = torch.where(seen[:, None, None], scores, float("-inf"))
        weights = (scores - scores.amax(-1, keepdim=True)).exp()
        values = torch.where(seen[:, None, :, None], values, 0.0)
        rows = (weights @ values) / weights.sum(-1, keepdim=True)
        out.append(rows.reshape(-1, heads * group, case["value_width"]))
    return torch.cat(out).to(_DTYPES[case["dtype"]])


_PLAIN = {"bias": _plain_bias, "write": _plain_write, "read": _plain_read, "chunk": _plain_chunk,
          "decode": _plain_decode}


# ------------------------------------------------------------------------------------------------
# From the definition, in 64 bits, one sequence (or one edge's distance) after another


def _bucket_of_distance(distance, buckets, max_distance):
    """A distance's bucket in integers: the number of j with distance ** rest >= half ** (rest - j) * max ** j."""
    half = buckets // 2
    if distance < half:
        return distance
    if distance >= max_distance:
        return buckets - 1
    rest, j = buckets - half, 0
    power = distance ** rest
    while j + 1 < rest and power >= half ** (rest - j - 1) * max_distance ** (j + 1):
        j += 1
    return half + j


def _distance_table(buckets, max_distance):
    """Buckets of the distances 0 .. max_distance."""
    return torch.tensor([_bucket_of_distance(d, buckets, max_distance) for d in range(max_distance + 1)],
                        device="cuda")


def _exact_bias(case, state):
    n, degree, furthest = case["tokens"], case["degree"], case["max_distance"]
    position = state["positions"] if state["positions"] is not None else torch.arange(n, device="cuda")
    rel = (position[state["col"]].view(n, degree) - position[:, None]).view(-1)
    if case["bidirectional"]:
        side = case["buckets"] // 2
        bucket = _distance_table(side, furthest)[rel.abs().clamp_max(furthest)] + side * (rel > 0)
    else:
        bucket = _distance_table(case["buckets"], furthest)[rel.neg().clamp(0, furthest)]
    table = state["table"].detach().double()
    bias = torch.stack([table[:, h][bucket] for h in range(case["heads"])])
    if not case["train"]:
        return bias
    grads = [torch.stack([state["grad"][:, bucket == b].double().sum(1)]) for b in range(case["buckets"])]
    return bias, torch.cat(grads)


def _exact_rows(x):
    """The numbers that an 8-bit cache holds for ``x``: per row of the last dimension a step of powers of two, three
    bits behind the leading one."""
    x = x.double()
    largest = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(largest.clamp_min(2.0 ** -140) / 448.0)).clamp_min(-126))
    scale = torch.where(largest > 448.0 * scale, 2 * scale, scale)
    scaled = x / scale
    leading = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp_min(2.0 ** -6))))
    step = leading / 8
    return torch.round(scaled / step) * step * scale


def _exact_cache(case, state):
    before = state["before"].tolist()
    pages, ptr, size = state["page_idx"].tolist(), state["page_ptr"].tolist(), case["page"]
    new = [0] * (len(before) + 1) if "new_ptr" not in state else state["new_ptr"].tolist()
    results = []
    for kind in ("key", "value"):
        held = state[kind + "_pages"].double()
        if case["quantised"]:
            held *= torch.exp2(state[kind + "_exponents"].double())[..., None]
        back = []
        for b, length in enumerate(before):
            mine = torch.tensor(pages[ptr[b]:ptr[b + 1]], dtype=torch.long, device="cuda")
            rows = held[mine].transpose(1, 2).reshape(-1, case["heads"], held.size(-1))
            count = new[b + 1] - new[b]
            if count:
                fresh = state[kind][new[b]:new[b + 1]]
                rows[length:length + count] = _exact_rows(fresh) if case["quantised"] else fresh.double()
            if case["op"] == "write":
                held[mine] = rows.view(-1, size, case["heads"], held.size(-1)).transpose(1, 2)
            else:
                back.append(rows[:length + count])
        results.append(held if case["op"] == "write" else torch.cat(back))
    return tuple(results)


def _exact_decode(case, state):
    heads, group, size = case["heads"], case["group"], case["page"]
    pages, ptr = state["page_idx"].tolist(), state["page_ptr"].tolist()
    out = torch.zeros(case["sequences"], heads * group, case["value_width"], dtype=torch.float64, device="cuda")
    nearest = None
    if case["buckets"]:
        nearest = _distance_table(case["buckets"], case["max_distance"])
    for b, length in enumerate(state["before"].tolist()):
        first = max(0, length - case["window"]) if case["window"] else 0
        mine = torch.tensor(pages[ptr[b] + first // size:ptr[b + 1]], dtype=torch.long, device="cuda")
        skip = first % size
        for h in range(heads):
            rows = []
            for kind in ("key", "value"):
                held = state[kind + "_pages"][mine, h].double()
                if case["quantised"]:
                    held = held * torch.exp2(state[kind + "_exponents"][mine, h].double())[..., None]
                rows.append(held.reshape(-1, held.size(-1))[skip:skip + length - first])
            for g in range(h * group, (h + 1) * group):
                score = (rows[0] * state["query"][b, g].double()).sum(1) / math.sqrt(case["width"])
                if nearest is not None:
                    away = torch.arange(length - 1 - first, -1, -1, device="cuda").clamp_max(case["max_distance"])
                    score = score + state["table"][:, g].double()[nearest[away]]
                weight = torch.softmax(score, 0)
                out[b, g] = (weight[:, None] * rows[1]).sum(0)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "bias":
        return _exact_bias(case, state)
    if case["op"] == "decode":
        return _exact_decode(case, state)
    return _exact_cache(case, state)
