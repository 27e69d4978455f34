"""Attention over a cache of 4 bits an element: what is measured of the operators that fill, read and attend one.

A cached key or value vector of a token and kv head is kept in blocks of 32 consecutive elements, each a number of the 4-bit
floating type e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times a power of two of the block's own, 2^(byte - 127)
(the MXFP4 format of the Open Compute Project's Microscaling specification).  The block's power is the smallest whose sevenfold
is not below the block's largest magnitude, so that no element is off by more than one unit of it; elements are rounded to
the nearest number, ties to the even code; a block with a NaN or an infinity in it gets byte 255 and stands for NaN.  A cache is four
byte tensors, P being the tokens of a page:

  key codes     [pages, kv_heads, dim / 32, P, 16]          element 2 i of a block in the low half of byte i, 2 i + 1 in the high one
  key powers    [pages, kv_heads, P, dim / 32]
  value codes   [pages, kv_heads, P / 4, dim / 8, 4, 4]     runs of 4 tokens: 8 neighbouring elements of each, packed as the keys'
  value powers  [pages, kv_heads, P / 4, dim / 32, 4]

Cases of three kinds.  "append": a step's fused projection becomes queries (norm of every head, rotation) and cached keys and
values; what the cache then holds of the step's rows is read back.  "decode": single tokens of many requests attend
their cached keys.  "prompt": portions of prompts attend what is cached before them and themselves.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
ENGINE_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _append(name, rows, q_heads, kv_heads, dim, *, entries=1, longest=1024, dtype="bfloat16", planes=0, norm=True, rotary=0,
            pairing="half_split", page=64):
    """``planes`` 0: the projection comes in the engine's type; else as so many float32 planes whose sum is meant."""
    case = {"kind": "append", "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "entries": entries, "longest": longest,
            "dtype": dtype, "planes": planes, "norm": norm, "rotary": rotary or dim, "pairing": pairing, "page": page}
    return {"name": name, **case} if name else case


def _decode(name, batch, q_heads, kv_heads, dim, shortest, longest, *, dtype="bfloat16", window=0, page=64):
    case = {"kind": "decode", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "shortest": shortest,
            "longest": longest, "dtype": dtype, "window": window, "page": page}
    return {"name": name, **case} if name else case


def _prompt(name, batch, q_heads, kv_heads, dim, portion, start, *, window=0, page=64):
    case = {"kind": "prompt", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "portion": portion, "start": start,
            "dtype": "bfloat16", "window": window, "page": page}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user's chat: the new token of a decode step
        _append("append 1", 1, 32, 8, 128, longest=2048),
        # a full serving batch's decode step, its projection cut along the inner size
        _append("append 64 planes", 64, 64, 8, 128, entries=64, longest=8192, planes=2),
        # the benchmark's prompt of 2,048 tokens
        _append("append prompt 2048", 2048, 32, 8, 128, longest=2048),
        # the 32-bit engine, three prompts of odd lengths, half a head rotated in neighbouring pairs
        _append("append float32", 777, 16, 4, 64, entries=3, longest=900, dtype="float32", rotary=32, pairing="adjacent"),
        # a short question to a small model, where launches and latency are what is waited for
        _decode("decode short", 2, 16, 8, 128, 77, 120),
        # the benchmark's headline: eight requests at a context of 8,192
        _decode("decode 8 at 8192", 8, 32, 8, 128, 8176, 8176),
        # one request far into a long document
        _decode("decode 1 at 32768", 1, 64, 8, 128, 32768, 32768),
        # a full serving batch whose requests have come to different lengths
        _decode("decode 64 ragged", 64, 40, 8, 128, 300, 8191),
        # the 32-bit engine's decode step
        _decode("decode float32", 4, 16, 4, 128, 501, 777, dtype="float32"),
        # three prompts arriving together at a model of small heads with a sliding window
        _prompt("prompts windowed", 3, 16, 4, 64, 901, 0, window=512),
        # a late portion of a long prompt beside other work: few rows, many keys
        _prompt("portion 128 at 30720", 1, 64, 8, 128, 128, 30720),
        # a full prompt portion in the middle of a document
        _prompt("portion 2048 at 8192", 1, 32, 8, 128, 2048, 8192),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt"])
    page = rng.choice([16, 32, 64, 64, 64, 128])
    if kind == "append":
        rows = _log(rng, 1, 2048)
        heads = rng.choice([(16, 8), (16, 4), (32, 8), (40, 8), (64, 8), (8, 1)])
        dim = rng.choice([64, 128, 128, 128])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        planes = rng.choice([0, 0, 1, 2]) if dtype == "bfloat16" and rows <= 512 else 0
        return _append(None, rows, *heads, dim, entries=min(rows, rng.choice([1, 2, 5, rows])), longest=rng.randint(rows, rows + 8192),
                       dtype=dtype, planes=planes, norm=rng.random() < 0.8, rotary=rng.choice([dim, dim, dim // 2]),
                       pairing=rng.choice(["half_split", "half_split", "adjacent"]), page=page)
    if kind == "decode":
        if rng.random() < 0.2:
            longest = _log(rng, 1, 2048)
            return _decode(None, _log(rng, 1, 12), *rng.choice([(16, 8), (16, 4), (32, 8)]), rng.choice([64, 128]),
                           rng.randint(max(1, longest // 4), longest), longest, dtype="float32", page=page)
        batch = _log(rng, 1, 64)
        dim = rng.choice([64, 128, 128, 128, 256])
        longest = _log(rng, 1, min(32768, 33554432 // dim // batch))
        heads = rng.choice([(16, 8), (32, 8), (40, 8), (64, 8), (8, 8), (16, 1), (40, 2)])
        return _decode(None, batch, *heads, dim, rng.randint(max(1, longest // 8), longest), longest,
                       window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), page=page)
    portion = _log(rng, 17, 2048)
    batch = rng.choice([1, 1, 2, 3]) if portion <= 600 else 1
    start = rng.choice([0, _log(rng, 1, 8192 if portion > 512 else 16384)]) if batch == 1 else rng.choice([0, _log(rng, 1, 4096)])
    return _prompt(None, batch, *rng.choice([(16, 8), (32, 8), (16, 4), (32, 4)]), rng.choice([64, 128, 128]), portion, start,
                   window=rng.choice([0, 0, 0, _log(rng, 64, 4096)]), page=page)


def _spread(low, high, n):
    """``n`` lengths between ``low`` and ``high``, the longest first."""
    return [high - int(round((high - low) * ((i * 0.6180339887) % 1.0))) for i in range(n)]


def _rows_of(case):
    """(tokens cached before, rows brought) of every request of a case."""
    if case["kind"] == "decode":
        return [(n - 1, 1) for n in _spread(case["shortest"], case["longest"], case["batch"])]
    if case["kind"] == "prompt":
        return list(zip(_spread(case["start"] // 2, case["start"], case["batch"]), _spread(max(17, case["portion"] // 3), case["portion"], case["batch"])))
    each, rest = divmod(case["rows"], case["entries"])
    counts = [each + (i < rest) for i in range(case["entries"])]
    return [(n - c, c) for n, c in zip(_spread(max(counts[0], case["longest"] // 3), max(counts[0], case["longest"]), case["entries"]), counts)]


def _visible(case):
    """Keys that the rows of a case see, over all rows."""
    total = 0
    for start, count in _rows_of(case):
        last, w = start + count, case["window"] or 1 << 30
        full = max(0, last - max(start, w - 1))                      # rows whose window is filled
        grow = count - full
        total += full * w if full else 0
        total += grow * start + grow * (grow + 1) // 2
    return total


# ---- the format ------------------------------------------------------------------------------------------------------------
def _encode(x):
    """x ``[..., dim]`` (float32 or float64) -> (codes uint8 ``[..., dim]``, powers uint8 ``[..., dim / 32]``)."""
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    top = blocks.abs().amax(dim=-1)
    fine = torch.isfinite(top)
    part, power = torch.frexp(torch.where(fine, top, torch.zeros_like(top)))
    power = torch.where(part > 0.875, power - 2, power - 3)
    power = torch.where(top > 0, power, -126).clamp(-126, 127)
    a = torch.ldexp(blocks, -power.unsqueeze(-1)).abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * torch.signbit(blocks)
    return code.reshape(x.shape).to(torch.uint8), torch.where(fine, power + 127, 255).to(torch.uint8)


def _level(codes, powers, dtype=torch.float32):
    """The values that codes ``[..., dim]`` and powers ``[..., dim / 32]`` stand for."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=dtype, device=codes.device)
    blocks = levels.index_select(0, codes.reshape(-1).int()).reshape(*codes.shape[:-1], -1, 32)
    power = torch.ldexp(torch.ones((), dtype=dtype, device=codes.device), powers.int() - 127)
    return (blocks * torch.where(powers == 255, math.nan, power).unsqueeze(-1)).reshape(codes.shape)


def _pack(codes):
    """Two codes a byte, the first in the low half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=-1).reshape(*packed.shape[:-1], -1)


def _pools(k, v, page):
    """Pages of vectors ``[pages, kv_heads, page, dim]`` in the cache's layout."""
    pages, heads, _, dim = k.shape
    codes, k_powers = _encode(k)
    k_codes = _pack(codes).reshape(pages, heads, page, dim // 32, 16).transpose(2, 3).contiguous()
    codes, powers = _encode(v)
    v_codes = _pack(codes).reshape(pages, heads, page // 4, 4, dim // 8, 4).transpose(3, 4).contiguous()
    v_powers = powers.reshape(pages, heads, page // 4, 4, dim // 32).transpose(3, 4).contiguous()
    return k_codes, k_powers.contiguous(), v_codes, v_powers


def _cached(pools, table):
    """Keys and values (float32) ``[requests, kv_heads, tokens, dim]`` of the pages that ``table`` ``[requests, blocks]`` names; a place
    without a page (-1) gives the first page's."""
    at = table.clamp(min=0).long()
    n, blocks = at.shape
    k_codes, k_powers, v_codes, v_powers = (pool[at] for pool in pools)
    heads, groups, page = k_codes.shape[2:5]
    k = _level(_unpack(k_codes).transpose(3, 4).reshape(n, blocks, heads, page, groups * 32), k_powers)
    v = _level(_unpack(v_codes).transpose(4, 5).reshape(n, blocks, heads, page, groups * 32),
               v_powers.transpose(4, 5).reshape(n, blocks, heads, page, groups))
    return (t.transpose(1, 2).reshape(n, heads, blocks * page, groups * 32) for t in (k, v))


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    normal = lambda *shape, dtype=torch.float32: torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)  # noqa: E731
    kind, dim, page, heads = case["kind"], case["dim"], case["page"], case["kv_heads"]
    dtype = ENGINE_TYPES[case["dtype"]]
    requests = _rows_of(case)
    rows = sum(count for _, count in requests)
    positions = torch.cat([torch.arange(start, start + count, dtype=torch.int32) for start, count in requests]).to(DEVICE)
    row_entry = torch.cat([torch.full((count,), i, dtype=torch.int32) for i, (_, count) in enumerate(requests)]).to(DEVICE)
    # pages handed out in no order; places of the table behind a request's last page hold none
    blocks = [-(-(start + count) // page) for start, count in requests]
    pages = sum(blocks) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(requests), max(blocks)), -1, dtype=torch.int32, device=DEVICE)
    taken = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[taken:taken + n]
        taken += n
    state = {"case": case, "positions": positions, "row_entry": row_entry, "table": table, "longest": max(start + count for start, count in requests)}
    channels = torch.exp(0.4 * normal(dim))                      # some elements of a head are larger than others, of all tokens
    if kind == "append":
        width = (case["q_heads"] + 2 * heads) * dim
        state["pools"] = tuple(torch.zeros(shape, dtype=torch.uint8, device=DEVICE) for shape in (
            (pages, heads, dim // 32, page, 16), (pages, heads, page, dim // 32), (pages, heads, page // 4, dim // 8, 4, 4),
            (pages, heads, page // 4, dim // 32, 4)))
        shape = (case["planes"], rows, width) if case["planes"] else (rows, width)
        state["qkv"] = (normal(*shape) * channels.repeat(width // dim)).to(torch.float32 if case["planes"] else dtype)
        state["gains"] = ((1.0 + 0.1 * normal(dim)).to(dtype), (1.0 + 0.1 * normal(dim)).to(dtype)) if case["norm"] else (None, None)
        angles = torch.outer(torch.arange(state["longest"], dtype=torch.float64, device=DEVICE),
                             1e6 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=DEVICE) / case["rotary"]))
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        return state
    state["pools"] = _pools(normal(pages, heads, page, dim) * channels, normal(pages, heads, page, dim) * channels, page)
    state["q"] = (1.5 * normal(rows, case["q_heads"], dim) / channels).reshape(rows, -1).to(dtype)
    if kind == "prompt":
        # the step's plan: tiles (request, first row, rows) of at most 32 rows, four to a group
        tiles, first = [], 0
        for i, (_, count) in enumerate(requests):
            mine = [(i, first + at, min(32, count - at)) for at in range(0, count, 32)]
            tiles += mine + [(i, first, 0)] * (-len(mine) % 4)
            first += count
        state["tiles"] = torch.tensor(tiles, dtype=torch.int32, device=DEVICE)
        state["mean_keys"] = max(1, sum(start * count + count * (count + 1) // 2 for start, count in requests) // rows)
        # where each request's rows lie, filled up to the longest portion, and where each row lies among those
        counts = torch.tensor([count for _, count in requests], device=DEVICE)
        firsts = counts.cumsum(0) - counts
        state["padded"] = (firsts[:, None] + torch.arange(int(counts.max()), device=DEVICE)[None, :]).clamp(max=rows - 1)
        state["place"] = torch.arange(rows, device=DEVICE) - firsts[row_entry.long()]
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        from leone_amd import ops
        if case["kind"] == "append":
            q = ops.qk_norm_rope_write_4bit(state["qkv"], case["q_heads"], case["kv_heads"], case["dim"], *state["gains"], 1e-6, state["cos"],
                                            state["sin"], state["positions"], state["row_entry"], state["table"], state["pools"],
                                            out_dtype=ENGINE_TYPES[case["dtype"]], pairing=case["pairing"])
            k, v = ops.cache_rows_4bit(state["pools"], state["positions"], state["row_entry"], state["table"])
            return {"q": q, "k": k, "v": v}
        scale = case["dim"] ** -0.5
        where = (state["positions"], state["row_entry"], state["table"], case["q_heads"], scale, case["window"])
        if case["dtype"] == "float32":
            return ops.attention_rows_4bit(state["q"], state["pools"], *where)
        if case["kind"] == "decode":
            return ops.attention_decode_4bit(state["q"], state["pools"], *where, max_context=state["longest"])
        out = torch.empty_like(state["q"])
        return ops.attention_prefill_4bit(state["q"], out, state["pools"], state["positions"], state["tiles"], state["table"],
                                          case["q_heads"], scale, case["window"], mean_keys=state["mean_keys"])
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[case["kind"]](state)


def _rotated(x, cos, sin, pairing):
    """Heads ``[rows, heads, dim]`` whose first elements are turned in pairs by the rows' angles."""
    half = cos.shape[1]
    cos, sin = cos[:, None, :], sin[:, None, :]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if pairing == "half_split":
        a, b = turned[..., :half], turned[..., half:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], dim=-1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2), rest], dim=-1)


def _plain_append(state):
    case = state["case"]
    dim, q_heads, kv_heads = case["dim"], case["q_heads"], case["kv_heads"]
    # in 64 bits: a key next to the border between two codes falls on its own side of it
    rows = state["qkv"].double()
    rows = (rows.sum(dim=0) if case["planes"] else rows).reshape(-1, q_heads + 2 * kv_heads, dim)
    q, k, v = rows[:, :q_heads], rows[:, q_heads:q_heads + kv_heads], rows[:, q_heads + kv_heads:]
    if case["norm"]:
        q, k = (x * gain.double() / (x.square().mean(dim=-1, keepdim=True) + 1e-6).sqrt() for x, gain in zip((q, k), state["gains"]))
    at = state["positions"].long()
    q, k = (_rotated(x, state["cos"][at].double(), state["sin"][at].double(), case["pairing"]) for x in (q, k))
    k, v = (_level(*_encode(x)).to(torch.bfloat16).reshape(x.shape[0], -1) for x in (k, v))
    return {"q": q.to(ENGINE_TYPES[case["dtype"]]).reshape(q.shape[0], -1), "k": k, "v": v}


def _weighted(scores, sees, values):
    scores = scores.masked_fill(~sees, -math.inf)
    weights = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    return (weights @ values) / weights.sum(dim=-1, keepdim=True)


def _sees(positions, keys, window):
    sees = keys <= positions
    return sees & (keys > positions - window) if window else sees


def _plain_decode(state):
    case = state["case"]
    batch, dim, kv_heads = case["batch"], case["dim"], case["kv_heads"]
    k, v = _cached(state["pools"], state["table"])
    q = state["q"].float().reshape(batch, kv_heads, -1, dim) * dim ** -0.5
    sees = _sees(state["positions"].long()[:, None], torch.arange(k.shape[2], device=k.device)[None, :], case["window"])
    return _weighted(q @ k.transpose(-1, -2), sees[:, None, None, :], v).reshape(batch, -1).to(state["q"].dtype)


def _plain_prompt(state):
    case = state["case"]
    dim, kv_heads, padded = case["dim"], case["kv_heads"], state["padded"]
    n, longest = padded.shape
    k, v = _cached(state["pools"], state["table"])
    q = state["q"].float().reshape(-1, case["q_heads"], dim)[padded] * dim ** -0.5
    q = q.reshape(n, longest, kv_heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, -1, dim)
    at = state["positions"].long()[padded]
    sees = _sees(at[:, :, None], torch.arange(k.shape[2], device=k.device), case["window"])
    group = case["q_heads"] // kv_heads
    out = _weighted(q @ k.transpose(-1, -2), sees[:, None, None].expand(-1, -1, group, -1, -1).reshape(n, 1, -1, k.shape[2]), v)
    out = out.reshape(n, case["q_heads"], longest, dim).transpose(1, 2)
    return out[state["row_entry"].long(), state["place"]].reshape(-1, case["q_heads"] * dim).to(torch.bfloat16)


# ---- what a pass cannot do without, and what it should give -----------------------------------------------------------------
def work(case):
    dim, heads, size = case["dim"], case["kv_heads"], 4 if case["dtype"] == "float32" else 2
    requests = _rows_of(case)
    rows = sum(count for _, count in requests)
    token = heads * (dim + dim // 16)                                # a cached token: codes and powers of key and value
    if case["kind"] == "append":
        width = (case["q_heads"] + 2 * heads) * dim
        read = rows * (width * (4 * case["planes"] if case["planes"] else size) + 4 * case["rotary"] + 12)
        return {"bytes": read + rows * (case["q_heads"] * dim * size + token + 2 * 2 * heads * dim), "flops": 8 * rows * width}
    held = sum(min(start + count, (case["window"] or 1 << 30) + count - 1) for start, count in requests)
    return {"bytes": held * (token + 4 / case["page"]) + rows * (2 * case["q_heads"] * dim * size + 8),
            "flops": 4 * case["q_heads"] * dim * _visible(case)}


def exact(case, seed):
    state = prepare(case, seed)
    dim, q_heads, kv_heads = case["dim"], case["q_heads"], case["kv_heads"]
    group = q_heads // kv_heads
    if case["kind"] == "append":
        x = state["qkv"].to(torch.float64)
        x = x[0] + x[1] if case["planes"] == 2 else x.reshape(-1, x.shape[-1])
        at = state["positions"].long()
        cos, sin = state["cos"].double()[at], state["sin"].double()[at]
        turned = case["rotary"]
        first = torch.arange(turned // 2, device=x.device)
        second = first + turned // 2
        if case["pairing"] == "adjacent":
            first, second = 2 * first, 2 * first + 1
        heads = []
        for h in range(q_heads + 2 * kv_heads):
            y = x[:, h * dim:(h + 1) * dim].clone()
            if h < q_heads + kv_heads:
                if case["norm"]:
                    y = y / torch.sqrt((y * y).sum(dim=1, keepdim=True) / dim + 1e-6) * state["gains"][h >= q_heads].double()
                a, b = y[:, first].clone(), y[:, second].clone()
                y[:, first], y[:, second] = a * cos - b * sin, b * cos + a * sin
            if h >= q_heads:
                levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
                for d in range(0, dim, 32):
                    block = y[:, d:d + 32]
                    unit = 2.0 ** torch.ceil(torch.log2((block.abs().amax(dim=1, keepdim=True) / 7.0).clamp(min=2.0 ** -126)))
                    off = (block.abs()[..., None] / unit[..., None] - levels).abs()
                    off[..., 1::2] += 1e-14                          # of two levels equally far the even code
                    y[:, d:d + 32] = torch.copysign(levels[off.argmin(dim=-1)] * unit, block)
            heads.append(y)
        return {"q": torch.cat(heads[:q_heads], dim=1), "k": torch.cat(heads[q_heads:q_heads + kv_heads], dim=1),
                "v": torch.cat(heads[q_heads + kv_heads:], dim=1)}
    k_codes, k_powers, v_codes, v_powers = state["pools"]
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=DEVICE)
    e = torch.arange(dim, device=DEVICE)
    q, positions, table = state["q"].double().reshape(-1, q_heads, dim), state["positions"].long(), state["table"].long()
    out, row = torch.zeros_like(q), 0
    for entry, (start, count) in enumerate(_rows_of(case)):
        keys = torch.arange(max(0, start - case["window"] + 1) if case["window"] else 0, start + count, device=DEVICE)
        page, token = table[entry, keys // case["page"]][:, None], (keys % case["page"])[:, None]
        sees = keys[None, :] <= positions[row:row + count, None]
        if case["window"]:
            sees &= positions[row:row + count, None] - keys[None, :] < case["window"]
        for h in range(kv_heads):
            shift = 4 * (e % 2)
            k = levels[(k_codes[page, h, e // 32, token, e % 32 // 2].long() >> shift) & 15] * 2.0 ** (k_powers[page, h, token, e // 32].double() - 127)
            v = levels[(v_codes[page, h, token // 4, e // 8, token % 4, e % 8 // 2].long() >> shift) & 15] \
                * 2.0 ** (v_powers[page, h, token // 4, e // 32, token % 4].double() - 127)
            for g in range(h * group, (h + 1) * group):
                scores = (q[row:row + count, g] @ k.T) / math.sqrt(dim)
                scores[~sees] = -math.inf
                out[row:row + count, g] = torch.softmax(scores, dim=1) @ v
        row += count
    return out.reshape(row, -1)
