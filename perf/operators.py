"""The operators of a paged cache held in 4 bits, as cases that can be timed and checked: writing a step's keys and values to
their pages, reading tokens back, and attention over the pages for single tokens and for runs of positions.

A case is a plain dict:

  op        "store" | "read" | "decode" | "prefill"
  heads, kv_heads, head_dim, page, dtype ("bfloat16" | "float32")
  requests  sequences of one call
  context   the median of their lengths (store, read, decode: with the tokens of the call; prefill: without its runs)
  spread    lengths lie between context * exp(-spread) and context * exp(spread)
  run       tokens of each sequence in the call, the median of them (decode: 1)
  window    0: every key; else the last ``window`` keys of a row
  rotate    store: the rows come as the projection leaves them, with a table of angles

What 4 bits hold, for each token and kv head and for its key and its value x of head_dim entries:

  low = bf16(min x)    step = bf16((max x - low) / 15)    code = round((x - low) / step) in 0..15    value = low + step * code

A page is a row of tiles of 16 tokens: [pages, kv_heads, page / 16, 16 * (head_dim + 8)] bytes.  A tile holds the keys' codes
(token by token, the even entry of a byte in its low half), the keys' 16 pairs (step, low), the values' codes in the order of
``_value_places`` and the values' 16 pairs.
"""
import math
import random

import numpy as np
import torch

own = False      # True: run() calls the framework's operators, else their plain form

_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_TILE = 16


def listed():
    def case(name, op, heads, kv_heads, head_dim, requests, context, run=1, spread=0.0, dtype="bfloat16", page=16, window=0, rotate=True):
        return dict(name=name, op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, requests=requests,
                    context=context, spread=spread, run=run, window=window, rotate=rotate)
    return [
        # TinyLlama-1.1B, one user chats: a single token's key and value, where the launch is what counts
        case("store one token", "store", 32, 4, 64, 1, 400),
        # Llama-3-8B sizes, 64 requests decode together: a row each, pages all over the pool
        case("store a decode step of 64", "store", 32, 8, 128, 64, 700, spread=0.7),
        # Llama-3-8B sizes, a prompt of 2,048 tokens enters in one step
        case("store a prompt of 2048", "store", 32, 8, 128, 1, 2048, run=2048),
        # the 32-bit path that answers are checked against, a ragged batch of small sequences
        case("store ragged runs in 32 bits", "store", 32, 4, 64, 5, 150, run=101, spread=0.6, dtype="float32", page=32),
        # one short sequence is looked at
        case("read one short sequence", "read", 32, 4, 64, 1, 37),
        # a long sequence leaves the pages (Llama-3-8B sizes)
        case("read a sequence of 8192", "read", 32, 8, 128, 1, 8192),
        # TinyLlama-1.1B, one user chats, 512 tokens in: launches and the walk over the keys
        case("decode one row", "decode", 32, 4, 64, 1, 529),
        # Llama-2-7B sizes (no shared heads), a batch of ragged lengths
        case("decode 24 ragged rows no shared heads", "decode", 32, 32, 128, 24, 601, spread=0.8),
        # Llama-3-8B sizes, eight requests with long contexts: bound by the bytes of the cache
        case("decode eight rows of 32768", "decode", 32, 8, 128, 8, 32768),
        # the 32-bit path, ragged contexts, larger pages, a sliding window
        case("decode in 32 bits with a window", "decode", 32, 4, 64, 7, 901, spread=0.7, dtype="float32", page=64, window=512),
        # TinyLlama-1.1B: one prompt of 2,048 tokens (bench.py's prompt step)
        case("one prompt of 2048", "prefill", 32, 4, 64, 1, 0, run=2048),
        # Llama-3-8B sizes: portions of prompts behind long ragged contexts
        case("ragged portions behind long contexts", "prefill", 32, 8, 128, 3, 4999, run=701, spread=0.5),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    heads, kv_heads, head_dim = rng.choice([(32, 4, 64), (32, 8, 128), (32, 32, 128), (32, 4, 64), (3, 1, 32), (16, 2, 256), (24, 8, 64)])
    c = dict(op=rng.choice(["store", "store", "read", "decode", "decode", "decode", "prefill", "prefill"]), heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, page=rng.choice([16, 16, 32, 64]), dtype=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]), requests=1,
             context=0, spread=round(rng.uniform(0.0, 0.9), 2), run=1, window=0, rotate=True)
    token = kv_heads * head_dim      # sizes are held to a budget of tokens times this
    if c["op"] == "store":
        c["requests"] = _log_int(rng, 1, 64)
        c["run"] = _log_int(rng, 1, max(1, min(2048, (1 << 20) // (token * c["requests"]))))
        c["context"] = c["run"] + rng.randint(0, 300)
        c["rotate"] = rng.random() < 0.7
    elif c["op"] == "read":
        c["requests"] = _log_int(rng, 1, 16)
        c["context"] = _log_int(rng, 1, max(1, min(8192, (3 << 20) // (token * c["requests"]))))
    elif c["op"] == "decode":
        c["requests"] = _log_int(rng, 1, 64)
        c["context"] = _log_int(rng, 1, max(1, min(32768, (80 << 20) // (token * c["requests"]))))
        c["window"] = rng.choice([0, 0, 0, rng.randint(1, 2048)])
    else:
        c["requests"] = _log_int(rng, 1, 8)
        c["run"] = _log_int(rng, 2, max(2, 2048 // c["requests"]))
        c["context"] = rng.choice([0, _log_int(rng, 1, max(1, 8192 // c["requests"]))])
        c["window"] = rng.choice([0, 0, 0, rng.randint(1, 2048)])
    return c


def _spread_out(median, spread, n):
    """n whole numbers of at least 1 whose logarithms lie evenly around the median's."""
    return [max(1, int(round(median * math.exp(spread * ((2 * i + 1) / n - 1.0))))) for i in range(n)]


def _lengths(case):
    """-> (tokens in the call, tokens before them) of each sequence, by the case alone."""
    n, order = case["requests"], random.Random(case["requests"])
    if case["op"] == "prefill":
        runs = _spread_out(case["run"], case["spread"], n)
        before = _spread_out(case["context"], case["spread"], n) if case["context"] else [0] * n
        order.shuffle(before)
        return runs, before
    total = _spread_out(case["context"], case["spread"], n)
    order.shuffle(total)
    if case["op"] == "read":
        return total, [0] * n
    runs = _spread_out(case["run"], case["spread"] if case["run"] > 1 else 0.0, n)
    runs = [min(r, t) for r, t in zip(runs, total)]
    return runs, [t - r for t, r in zip(total, runs)]


def _seen(case):
    """(row, key) pairs of the call."""
    pairs, w = 0, case["window"]
    for run, before in zip(*_lengths(case)):
        p = np.arange(before + 1, before + run + 1)
        pairs += int((np.minimum(p, w) if w else p).sum())
    return pairs


def work(case):
    runs, before = _lengths(case)
    nh, nkv, hd, e = case["heads"], case["kv_heads"], case["head_dim"], 2 if case["dtype"] == "bfloat16" else 4
    rows, held = sum(runs), nkv * (hd + 8)      # bytes of a token's keys and values in the cache
    if case["op"] == "store":
        table = 4 * rows * hd + 2 * rows * nh * hd * e if case["rotate"] else 0      # the angles, and the queries once in and once out
        return {"bytes": 2 * rows * nkv * hd * e + table + 4 * rows + rows * held + 2 * rows * nkv * hd * e,
                "flops": rows * hd * (8 * nkv + (3 * (nh + nkv) if case["rotate"] else 0))}
    if case["op"] == "read":
        return {"bytes": rows * held + 4 * rows + 2 * rows * nkv * hd * e, "flops": 4 * rows * nkv * hd}
    w = case["window"]
    tokens = sum(min(b + r, w + r - 1) if w else b + r for r, b in zip(runs, before))
    return {"bytes": tokens * held + 2 * rows * nh * hd * e, "flops": 4 * hd * nh * _seen(case)}


# ------------------------------------------------------------------------------------------------ the format
def _value_places(hd):
    """The place, among a tile's 16 * hd halves of bytes, of entry d of token t's value: [16, hd].  Sixteen chunks of hd / 16 entries;
    of each, four tokens lie together, 4 entries of two tokens (2 entries of four where a chunk has 2) to a word of 32 bits."""
    t, d = torch.arange(_TILE).view(-1, 1), torch.arange(hd).view(1, -1)
    chunk = hd // 16
    four, pair, odd = t // 4, t // 2 % 2, t % 2
    word = (four * 16 + d // chunk) * (chunk // 2)
    if chunk == 2:
        return 8 * word + 2 * (2 * odd + pair) + d % 2
    return 8 * (word + pair * (chunk // 4) + d % chunk // 4) + 4 * odd + d % 4


def _codes(x):
    """x [..., hd] -> (codes, step, low) in x's type; step and low are bfloat16 values."""
    low = x.amin(-1, keepdim=True).bfloat16().to(x.dtype)
    step = ((x.amax(-1, keepdim=True) - low) / 15).bfloat16().to(x.dtype)
    code = ((x - low) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
    return torch.where(step > 0, code, torch.zeros_like(code)), step, low


def _tiles(x, values):
    """Tokens x [tiles, 16, hd] as the half of a tile that holds them: bytes [tiles, 8 * hd + 64]."""
    n, _, hd = x.shape
    code, step, low = _codes(x)
    code = code.to(torch.uint8).view(n, _TILE * hd)
    if values:
        halves = torch.empty_like(code)
        halves[:, _value_places(hd).view(-1).to(x.device)] = code
    else:
        halves = code
    halves = halves.view(n, 8 * hd, 2)
    pairs = torch.cat([step, low], -1).bfloat16().view(torch.uint8).reshape(n, 4 * _TILE)
    return torch.cat([halves[:, :, 0] | halves[:, :, 1] << 4, pairs], 1)


def _untiled(cache, hd, places=None, dtype=torch.float32):
    """The cache's keys (or, with the places of their codes, its values) as numbers, [pages * page, kv_heads, hd]."""
    pages, nkv, tiles, _ = cache.shape
    half = cache[..., :8 * hd + 64] if places is None else cache[..., 8 * hd + 64:]
    codes = torch.stack([half[..., :8 * hd] & 15, half[..., :8 * hd] >> 4], -1).flatten(-2)
    if places is not None:
        codes = codes[..., places]
    pairs = half[..., 8 * hd:].contiguous().view(torch.bfloat16).view(pages, nkv, tiles, _TILE, 2).to(dtype)
    x = pairs[..., 1:] + pairs[..., :1] * codes.view(pages, nkv, tiles, _TILE, hd).to(dtype)
    return x.permute(0, 2, 3, 1, 4).reshape(pages * tiles * _TILE, nkv, hd)


# ------------------------------------------------------------------------------------------------ states
def _random_tokens(shape, gen, dev):
    """Keys or values as a model has them: normal entries, of which some places of every head stand out on one side."""
    x = torch.randn(shape, generator=gen, device=dev)
    away = torch.randn(shape[-2:], generator=gen, device=dev)
    return x + 2.0 * away * (away.abs() > 1.2)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    nh, nkv, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    dtype = _TYPES[case["dtype"]]
    runs, before = _lengths(case)
    shuffled = random.Random(int(seed)).sample(range(len(runs)), len(runs))      # another seed: the lengths in another order
    runs, before = [runs[i] for i in shuffled], [before[i] for i in shuffled]
    n, rows = len(runs), sum(runs)
    need = [-(-(r + b) // page) for r, b in zip(runs, before)]
    stride, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    tables = torch.zeros(n, stride, dtype=torch.int32, device=dev)
    at = 0
    for i, k in enumerate(need):
        tables[i, :k] = order[at:at + k]
        at += k

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    run_start = ints(np.concatenate([[0], np.cumsum(runs)]).tolist())
    row_seq = torch.repeat_interleave(torch.arange(n, device=dev), ints(runs).long()).to(torch.int32)
    positions = ints(before)[row_seq] + torch.arange(rows, device=dev, dtype=torch.int32) - run_start[row_seq]
    slots = (tables[row_seq, (positions // page).long()] * page + positions % page).to(torch.int32)
    s = dict(case=dict(case), tables=tables.view(-1), stride=stride, run_start=run_start, seq_start=ints(before), row_seq=row_seq,
             ctx_lens=(positions + 1).to(torch.int32), slots=slots, max_run=max(runs), max_context=max(r + b for r, b in zip(runs, before)),
             places=_value_places(hd).view(-1).to(dev))
    if case["op"] == "store":
        s["cache"] = torch.zeros(pages, nkv, page // _TILE, _TILE * (hd + 8), dtype=torch.uint8, device=dev)
        s["plain_codes"] = torch.zeros(pages * page, 2 * nkv, hd, dtype=torch.uint8, device=dev)      # the plain form's cache, a code a byte
        s["plain_pairs"] = torch.zeros(pages * page, 2 * nkv, 2, dtype=torch.bfloat16, device=dev)
    else:
        tiles = pages * nkv * (page // _TILE)
        half = [_tiles(_random_tokens((pages, page // _TILE, _TILE, nkv, hd), gen, dev).permute(0, 3, 1, 2, 4).reshape(tiles, _TILE, hd), v)
                for v in (False, True)]
        s["cache"] = torch.cat(half, 1).view(pages, nkv, page // _TILE, _TILE * (hd + 8)).contiguous()
    if case["op"] != "read":
        s["qkv"] = torch.cat([torch.randn(rows, nh * hd, generator=gen, device=dev), _random_tokens((rows, nkv, hd), gen, dev).view(rows, -1),
                              _random_tokens((rows, nkv, hd), gen, dev).view(rows, -1)], 1).to(dtype)
    if case["op"] in ("decode", "prefill"):
        s["out"] = torch.empty(rows, nh * hd, dtype=dtype, device=dev)
    else:
        s["k"], s["v"] = (torch.empty(rows, nkv * hd, dtype=dtype, device=dev) for _ in range(2))
    if case["op"] == "store" and case["rotate"]:
        freq = 10000.0 ** (-torch.arange(hd // 2, device=dev, dtype=torch.float64) * 2 / hd)
        angle = positions.double().view(-1, 1) * freq
        s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        s["q"] = torch.empty(rows, nh * hd, dtype=dtype, device=dev)
    return s


# ------------------------------------------------------------------------------------------------ passes
def run(state):
    c = state["case"]
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if own:
        from kvcm_amd import ops
        if c["op"] == "store":
            ops.rope_cache4(state["qkv"], nh, nkv, hd, state["cache"], state["slots"], cos_sin=state.get("cos_sin"), q_out=state.get("q"))
            ops.cache4_rows(state["cache"], state["slots"], state["k"], state["v"])
            return {x: state[x] for x in "qkv" if x in state}
        if c["op"] == "read":
            ops.cache4_rows(state["cache"], state["slots"], state["k"], state["v"])
            return {"k": state["k"], "v": state["v"]}
        if c["op"] == "decode":
            ops.attention_decode4(state["qkv"], state["out"], state["cache"], state["tables"], state["stride"], state["row_seq"], state["ctx_lens"],
                                  nh, nkv, hd, hd ** -0.5, state["max_context"], window=c["window"])
        else:
            ops.attention_prefill4(state["qkv"], state["out"], state["cache"], state["tables"], state["stride"], state["run_start"],
                                   state["seq_start"], c["requests"], state["max_run"], nh, nkv, hd, hd ** -0.5,
                                   max_context=state["max_context"], window=c["window"])
        return state["out"]
    return _plain(state)


def _rotated(x, cos_sin):
    """Pairs (j, j + hd / 2) of x [rows, heads, hd] by the table's angles, in 64 bits (entries next to a code's border)."""
    a, b = x.double().chunk(2, -1)
    cs, sn = (cos_sin[:, None, :, i].double() for i in (0, 1))
    return torch.cat([a * cs - b * sn, b * cs + a * sn], -1)


def _plain(s):
    c = s["case"]
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    dtype = _TYPES[c["dtype"]]
    if c["op"] == "read":
        slots = s["slots"].long()
        return {x: _untiled(s["cache"], hd, s["places"] if x == "v" else None)[slots].flatten(1).to(dtype) for x in "kv"}
    if c["op"] == "store":
        return _plain_store(s, s["qkv"].shape[0], nh, nkv, hd, dtype)
    return _plain_attention(s, nh, nkv, hd, c["window"]).to(dtype)


def _plain_store(s, rows, nh, nkv, hd, dtype):
    x = s["qkv"].view(rows, nh + 2 * nkv, hd).float()
    out, kept = {}, x[:, nh:]
    if "cos_sin" in s:
        turned = _rotated(x[:, :nh + nkv], s["cos_sin"]).to(dtype)
        out["q"] = turned[:, :nh].flatten(1)
        kept = torch.cat([turned[:, nh:].float(), x[:, nh + nkv:]], 1)
    codes, pairs = s["plain_codes"], s["plain_pairs"]
    code, step, low = _codes(kept.double())
    slots = s["slots"].long()
    codes[slots] = code.to(torch.uint8)
    pairs[slots] = torch.cat([step, low], -1).bfloat16()
    held, pair = codes[slots].float(), pairs[slots].float()      # read back
    kept = (pair[..., 1:] + pair[..., :1] * held).to(dtype)
    return out | {"k": kept[:, :nkv].flatten(1), "v": kept[:, nkv:].flatten(1)}


def _plain_attention(s, nh, nkv, hd, window):
    dev, n, stride = s["tables"].device, s["run_start"].numel() - 1, s["stride"]
    page = s["cache"].shape[2] * _TILE
    k, v = _untiled(s["cache"], hd), _untiled(s["cache"], hd, s["places"])
    L, R = s["max_context"], s["max_run"]
    t = torch.arange(L, device=dev)
    slots = s["tables"].view(n, stride)[:, t // page].long() * page + t % page                     # [n, L]
    k, v = k[slots].permute(0, 2, 3, 1), v[slots].permute(0, 2, 1, 3)                              # [n, nkv, hd, L], [n, nkv, L, hd]
    r = torch.arange(R, device=dev)
    first, count = s["run_start"][:-1].long().view(-1, 1), s["run_start"].diff().view(-1, 1)
    row = first + torch.minimum(r, count - 1)                                                      # [n, R]: a run's rows, the last repeated
    at = s["seq_start"].view(-1, 1) + torch.minimum(r, count - 1)
    q = s["qkv"][:, :nh * hd].float()[row].view(n, R, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    x = (q @ k).view(n, nkv, nh // nkv, R, L) * hd ** -0.5
    seen = t <= at.unsqueeze(-1)
    if window:
        seen &= t > at.unsqueeze(-1) - window
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = (x.view(n, nkv, -1, L) @ v).view(n, nkv, nh // nkv, R, hd) / x.sum(-1, keepdim=True)
    x = x.permute(0, 3, 1, 2, 4).reshape(n, R, nh * hd)
    return x[s["row_seq"].long(), torch.arange(s["row_seq"].numel(), device=dev) - s["run_start"][s["row_seq"].long()]]


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] != "store":
        k, v = (_untiled(s["cache"], hd, places, torch.float64) for places in (None, s["places"]))
    if case["op"] == "read":
        return {"k": k[s["slots"].long()].flatten(1), "v": v[s["slots"].long()].flatten(1)}
    if case["op"] == "store":
        x = s["qkv"].double().view(-1, nh + 2 * nkv, hd)
        if "cos_sin" in s:
            z = torch.view_as_complex(s["cos_sin"].double().contiguous()).unsqueeze(1)
            turned = torch.complex(x[:, :nh + nkv, :hd // 2].contiguous(), x[:, :nh + nkv, hd // 2:].contiguous()) * z
            x = torch.cat([torch.cat([turned.real, turned.imag], -1), x[:, nh + nkv:]], 1)
        kept = x[:, nh:].to(_TYPES[case["dtype"]]).double()      # what the cache holds is made of the rows' own type
        low = kept.amin(-1, keepdim=True).bfloat16().double()
        step = ((kept.amax(-1, keepdim=True) - low) / 15).bfloat16().double()
        code = ((kept - low) / step).nan_to_num(0.0, 0.0, 0.0).round().clamp(0, 15)
        kept = low + step * code
        out = {"q": x[:, :nh].flatten(1)} if case["rotate"] else {}
        return out | {"k": kept[:, :nkv].flatten(1), "v": kept[:, nkv:].flatten(1)}
    page, out = case["page"], []
    starts, befores = s["run_start"].tolist(), s["seq_start"].tolist()
    for i, before in enumerate(befores):
        r0, r1 = starts[i], starts[i + 1]
        t = torch.arange(before + r1 - r0, device="cuda")
        slots = s["tables"].view(-1, s["stride"])[i, t // page].long() * page + t % page
        pos = before + torch.arange(r1 - r0, device="cuda").view(-1, 1)
        seen = (t <= pos) & ((t > pos - case["window"]) if case["window"] else True)
        q, of_heads = s["qkv"][r0:r1, :nh * hd].double().view(-1, nh, hd), []
        for h in range(nh):
            p = torch.softmax((q[:, h] @ k[slots, h * nkv // nh].T * hd ** -0.5).masked_fill(~seen, -math.inf), -1)
            of_heads.append(p @ v[slots, h * nkv // nh])
        out.append(torch.cat(of_heads, 1))
    return torch.cat(out)
