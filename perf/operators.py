"""What is measured of the operators that a decoder beside the packed image encoder needs: a key/value cache in pages, written and read
back in the ARCQ format, attention of new tokens over that cache, and attention to an encoder's states.

A cache page holds ``page`` tokens of every key/value head.  In 16 bits it is the values, [pages, kv_heads, page, 64]; in 2, 3 or 4 bits
the packed codes, [pages, kv_heads, page, 8 * bits] bytes, and an fp16 pair (center, scale) for each token and head: a head's 64 values
are one group of the ARCQ quantizer, x ~ center + scale * level[code].

Each function below takes plain torch operations where ``own`` is false and the framework's operators where it is true.
"""
import math

import torch

own = False

HEAD = 64
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    from __graft_entry__ import import_package
    return import_package().ops


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decoding step of 64 captions: a token each, written into a cache in 4 bits and read back
        {"name": "cache_step", "op": "cache", "write": True, "tokens": 64, "kv_heads": 6, "bits": 4, "page": 16, "dtype": "fp16"},
        # prompts of a batch written at once, as wide as DeiT-B
        {"name": "cache_prompts", "op": "cache", "write": True, "tokens": 16384, "kv_heads": 12, "bits": 4, "page": 64, "dtype": "bf16"},
        # a cache in 3 bits read back whole, an odd number of tokens: moved to another machine, say
        {"name": "cache_read_3bit", "op": "cache", "write": False, "tokens": 40009, "kv_heads": 3, "bits": 3, "page": 32, "dtype": "fp16"},
        # one caption, one new token, a short context: latency
        {"name": "paged_one", "op": "paged", "batch": 1, "heads": 6, "kv_heads": 6, "new": 1, "context": 333, "ragged": False, "bits": 4, "page": 16, "dtype": "fp16"},
        # a batch of captions, a token each, shared key heads
        {"name": "paged_batch", "op": "paged", "batch": 64, "heads": 12, "kv_heads": 4, "new": 1, "context": 4096, "ragged": True, "bits": 4, "page": 64, "dtype": "bf16"},
        # few sequences with long contexts: the work of a sequence has to be split
        {"name": "paged_long", "op": "paged", "batch": 2, "heads": 12, "kv_heads": 12, "new": 1, "context": 65521, "ragged": True, "bits": 3, "page": 128, "dtype": "fp16"},
        # prompts in pieces beside single tokens in one call, lengths of all kinds
        {"name": "paged_mixed", "op": "paged", "batch": 24, "heads": 12, "kv_heads": 6, "new": 197, "context": 2500, "ragged": True, "bits": 4, "page": 32, "dtype": "fp16"},
        # a long document in pieces of 2048 tokens, cache in 16 bits
        {"name": "paged_chunk_16bit", "op": "paged", "batch": 1, "heads": 12, "kv_heads": 12, "new": 2048, "context": 16384, "ragged": False, "bits": 16, "page": 64, "dtype": "bf16"},
        # the same over a cache in 4 bits, shared key heads
        {"name": "paged_chunk_4bit", "op": "paged", "batch": 1, "heads": 12, "kv_heads": 4, "new": 2048, "context": 16384, "ragged": False, "bits": 4, "page": 64, "dtype": "fp16"},
        # one caption token of each of 64 images against the 197 states of a DeiT encoder
        {"name": "cross_one", "op": "cross", "batch": 64, "heads": 6, "kv_heads": 6, "queries": 1, "states": 197, "mask": "none", "dtype": "fp16"},
        # captions of 40 tokens against 577 states (384 x 384 pixels in patches of 16), some of them dropped
        {"name": "cross_masked", "op": "cross", "batch": 32, "heads": 12, "kv_heads": 12, "queries": 40, "states": 577, "mask": "mask", "dtype": "fp16"},
        # texts of 1024 tokens against the states of several images, padded to the longest
        {"name": "cross_long", "op": "cross", "batch": 16, "heads": 12, "kv_heads": 12, "queries": 1024, "states": 2309, "mask": "lengths", "dtype": "bf16"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["cache", "paged", "paged", "cross"])
    kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    dtype = rng.choice(["fp16", "bf16"])
    most = 2048 * 15300 * 12               # pairs of a query and a key: those of the listed chunks
    if op == "cache":
        return {"op": op, "write": rng.random() < 0.7, "tokens": min(_log_uniform(rng, 1, 60000), 200000 // kv_heads), "kv_heads": kv_heads,
                "bits": rng.choice([2, 3, 4, 4, 16]), "page": page, "dtype": dtype}
    if op == "paged":
        new = 1 if rng.random() < 0.5 else _log_uniform(rng, 2, 2048)
        context = max(new, _log_uniform(rng, 1, 40000))
        batch = _log_uniform(rng, 1, 96)
        # at most the cached tokens of a few long sequences
        context = max(new, min(context, most // (new * heads)))
        batch = max(1, min(batch, 12 * 131072 // (context * kv_heads), most // (new * context * heads)))
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "new": new, "context": context, "ragged": rng.random() < 0.7,
                "bits": rng.choice([2, 3, 4, 4, 16]), "page": page, "dtype": dtype}
    queries = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 1500)
    states = _log_uniform(rng, 1, 2500)
    batch = max(1, min(_log_uniform(rng, 1, 128), most // (heads * queries * states), 16 * 12 * 2309 // (kv_heads * states)))
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "queries": queries, "states": states,
            "mask": rng.choice(["none", "lengths", "mask"]), "dtype": dtype}


def _sequence_lengths(case):
    """Tokens of every sequence after the new ones, and how many of them are new; of the case alone, so that its work is known."""
    B, n, L = case["batch"], case["new"], case["context"]
    if not case["ragged"]:
        return [L] * B, [n] * B
    new = [n if i % 3 == 0 else max(1, n * (i * 7 % 11) // 11) for i in range(B)]
    return [max(m, L - (L * (i * 5 % 16)) // 20) for i, m in enumerate(new)], new


def _state_lengths(case):
    B, S = case["batch"], case["states"]
    return [S - (S * (i * 3 % 8)) // 10 for i in range(B)] if case["mask"] == "lengths" else [S] * B


def _row_bytes(bits):
    """Of a token and head in the cache, keys or values alone."""
    return 2 * HEAD if bits == 16 else 8 * bits + 4


def work(case):
    if case["op"] == "cache":
        values = 2 * case["tokens"] * case["kv_heads"] * HEAD          # keys and values
        cached = 2 * case["tokens"] * case["kv_heads"] * _row_bytes(case["bits"])
        passes = 2 if case["write"] else 1                             # written (values in, cache out), read (cache in, values out)
        return {"bytes": passes * (2 * values + cached + 8 * case["tokens"]), "flops": passes * 8 * values}
    if case["op"] == "paged":
        lengths, new = _sequence_lengths(case)
        seen = sum(n * (L - n) + n * (n + 1) // 2 for L, n in zip(lengths, new))
        return {"bytes": 2 * 2 * sum(new) * case["heads"] * HEAD + 2 * sum(lengths) * case["kv_heads"] * _row_bytes(case["bits"]),
                "flops": 4 * HEAD * case["heads"] * seen}
    states = sum(_state_lengths(case))
    return {"bytes": 2 * 2 * case["batch"] * case["queries"] * case["heads"] * HEAD + 2 * 2 * states * case["kv_heads"] * HEAD,
            "flops": 4 * HEAD * case["heads"] * case["queries"] * states}


# ---------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1009 + 17)


def _values(gen, shape, dtype, spread=1.0):
    """Projections as a layer gives them: every channel of a head with a spread and an offset of its own."""
    channels = torch.randn(shape[-2:], generator=gen, device="cuda")
    offsets = torch.randn(shape[-2:], generator=gen, device="cuda")
    x = torch.randn(shape, generator=gen, device="cuda")
    return (spread * (x * (0.6 + 0.4 * channels.abs()) + 0.3 * offsets)).to(dtype)


def _levels(bits):
    """Codebooks of keys and of values [2, 2^bits], and the thresholds between their levels: quantiles of a normal distribution."""
    at = (torch.arange(2 ** bits, dtype=torch.float64) + 0.5) / 2 ** bits
    levels = torch.special.ndtri(at)
    levels = levels / levels.square().mean().sqrt()
    levels = torch.stack([levels, 1.04 * levels + 0.01]).float()
    return levels.cuda(), ((levels[:, :-1].double() + levels[:, 1:].double()) / 2).float().cuda()


def _cache(case, pages, gen, filled):
    """Empty pages, or pages of `filled` keys and values [pages, kv_heads, page, 64] each."""
    H, page, bits = case["kv_heads"], case["page"], case["bits"]
    c = {"bits": bits}
    if bits == 16:
        c["k_pages"], c["v_pages"] = filled or [torch.zeros(pages, H, page, HEAD, dtype=DTYPES[case["dtype"]], device="cuda") for _ in range(2)]
        c["k_stats"] = c["v_stats"] = c["codebooks"] = c["thresholds"] = None
        return c
    c["codebooks"], c["thresholds"] = _levels(bits)
    for i, name in enumerate("kv"):
        if filled is None:
            c[name + "_pages"] = torch.zeros(pages, H, page, 8 * bits, dtype=torch.uint8, device="cuda")
            c[name + "_stats"] = torch.zeros(pages, H, page, 2, dtype=torch.float16, device="cuda")
        else:
            codes, c[name + "_stats"] = _quantise(filled[i], c["thresholds"][i], c["codebooks"][i])
            c[name + "_pages"] = _pack(codes, bits)
    return c


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "cache":
        T, H, page = case["tokens"], case["kv_heads"], case["page"]
        pages = -(-T // page) + 3
        filled = None if case["write"] else [_values(gen, (pages, page, H, HEAD), dtype).transpose(1, 2).contiguous() for _ in range(2)]
        state["cache"] = _cache(case, pages, gen, filled)
        # tokens of many sequences, wherever their pages are; every 50th is padding and has no slot
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:T]
        slots[torch.arange(T, device="cuda") % 50 == 49] = -1
        state["slots"] = slots
        if case["write"]:
            qkv = _values(gen, (T, 3 * H, HEAD), dtype)          # the projection's output, queries first: keys and values are views
            state["k"], state["v"] = qkv[:, H:2 * H], qkv[:, 2 * H:]
        state["pages"] = pages
    elif case["op"] == "paged":
        lengths, new = _sequence_lengths(case)
        B, page = case["batch"], case["page"]
        widest = -(-max(lengths) // page)
        pages = sum(-(-L // page) for L in lengths) + 2
        filled = [_values(gen, (pages, page, case["kv_heads"], HEAD), dtype).transpose(1, 2).contiguous() for _ in range(2)]
        state["cache"] = _cache(case, pages, gen, filled)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        used = torch.tensor([-(-L // page) for L in lengths])
        first = torch.cumsum(used, 0) - used
        at = (first[:, None] + torch.arange(widest)[None, :]).clamp(max=pages - 1)
        table = order[at.cuda()]
        table[(torch.arange(widest)[None, :] >= used[:, None]).cuda()] = -1          # no page there
        state["table"] = table
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        state["starts"] = torch.cumsum(torch.tensor([0] + new), 0).to(torch.int32).cuda()
        state["q"] = _values(gen, (sum(new), case["heads"], HEAD), dtype, 1.3)
    else:
        B, S, H = case["batch"], case["states"], case["kv_heads"]
        state["q"] = _values(gen, (B, case["queries"], case["heads"], HEAD), dtype, 1.3)
        kv = _values(gen, (B, S, 2 * H, HEAD), dtype)                            # one projection of the states
        state["k"], state["v"] = kv[:, :, :H], kv[:, :, H:]
        state["lengths"] = state["mask_of"] = None
        if case["mask"] == "lengths":
            state["lengths"] = torch.tensor(_state_lengths(case), dtype=torch.int32, device="cuda")
        if case["mask"] == "mask":
            state["mask_of"] = torch.rand(B, S, generator=gen, device="cuda") < 0.8
    return state


# ---------------------------------------------------------------- plain forms
def _quantise(x, thresholds, levels):
    """Codes and (center, scale) of groups of 64, statistics and comparisons in 64 bits."""
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    r = x - mean
    scale = (r.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    codes = torch.bucketize(r / scale, thresholds.double())
    center = mean - scale * levels.double()[codes].mean(-1, keepdim=True)
    return codes, torch.cat([center, scale], -1).half()


def _pack(codes, bits):
    """Codes [..., 64] as a little-endian bit stream [..., 8 * bits] of bytes."""
    one = (codes.to(torch.uint8).unsqueeze(-1) >> torch.arange(bits, dtype=torch.uint8, device=codes.device)) & 1
    one = one.reshape(*codes.shape[:-1], 8 * bits, 8) << torch.arange(8, dtype=torch.uint8, device=codes.device)
    return one.sum(-1, dtype=torch.uint8)


def _unpack(packed, bits):
    one = (packed.unsqueeze(-1) >> torch.arange(8, dtype=torch.uint8, device=packed.device)) & 1
    one = one.reshape(*packed.shape[:-1], HEAD, bits) << torch.arange(bits, dtype=torch.uint8, device=packed.device)
    return one.sum(-1, dtype=torch.uint8).int()


def _restored(packed, stats, levels, bits):
    """Cached keys or values in 32 bits."""
    if bits == 16:
        return packed.float()
    return stats[..., :1].float() + stats[..., 1:].float() * levels[_unpack(packed, bits)]


def _write_plain(s):
    c, page = s["cache"], s["page"]
    real = s["slots"] >= 0
    slots = s["slots"][real]
    at = (slots // page, slice(None), slots % page)
    for i, name in enumerate("kv"):
        x = s[name][real]
        if c["bits"] == 16:
            c[name + "_pages"][at] = x
        else:
            codes, stats = _quantise(x, c["thresholds"][i], c["codebooks"][i])
            c[name + "_pages"][at] = _pack(codes, c["bits"])
            c[name + "_stats"][at] = stats


def _read_plain(s):
    c, page = s["cache"], s["page"]
    slots = s["slots"].clamp(min=0)
    at = (slots // page, slice(None), slots % page)
    out = []
    for i, name in enumerate("kv"):
        packed = c[name + "_pages"][at]
        x = packed.float() if c["bits"] == 16 else _restored(packed, c[name + "_stats"][at], c["codebooks"][i], c["bits"])
        out.append((x * (s["slots"] >= 0)[:, None, None]).to(DTYPES[s["dtype"]]))
    return out


def _attend_plain(q, k, v, seen):
    """q [B, n, H, 64], k and v [B, S, kv_heads, 64], seen [B, n, S]; 32 bits.  A query that sees nothing gets zeros."""
    B, n, H, _ = q.shape
    groups = H // k.shape[2]
    q = q.transpose(1, 2).reshape(B, k.shape[2], groups * n, HEAD)
    scores = (q @ k.permute(0, 2, 3, 1) * 0.125).reshape(B, H, n, -1)
    scores = scores.masked_fill(~seen[:, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == float("-inf"), 0.0))
    total = p.sum(-1, keepdim=True)
    out = p.reshape(B, k.shape[2], groups * n, -1) @ v.transpose(1, 2)
    return (out.reshape(B, H, n, HEAD) / total.masked_fill(total == 0, 1.0)).transpose(1, 2)


def _paged_plain(s):
    c, page = s["cache"], s["page"]
    B, widest = s["table"].shape
    keys = torch.arange(widest * page, device="cuda")
    there = keys < s["lengths"][:, None]                                        # [B, S]
    kv = []
    for i, name in enumerate("kv"):
        at = s["table"].clamp(min=0)
        x = _restored(c[name + "_pages"][at], None if c["bits"] == 16 else c[name + "_stats"][at], None if c["bits"] == 16 else c["codebooks"][i], c["bits"])
        x = x.transpose(2, 3).reshape(B, widest * page, s["kv_heads"], HEAD)
        kv.append(x.masked_fill(~there[:, :, None, None], 0.0))
    new = s["starts"][1:] - s["starts"][:-1]
    rows = torch.arange(s["new"], device="cuda")
    real = rows < new[:, None]                                                  # [B, n]
    at = (s["starts"][:-1, None] + rows).clamp(max=s["q"].shape[0] - 1)
    last = s["lengths"][:, None] - new[:, None] + rows                          # the newest key that a query sees
    out = _attend_plain(s["q"][at].float(), kv[0], kv[1], there[:, None] & (keys <= last[:, :, None]))
    return out[real].to(DTYPES[s["dtype"]])


def _cross_plain(s):
    B, S = s["batch"], s["states"]
    there = torch.ones(B, S, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        there = torch.arange(S, device="cuda") < s["lengths"][:, None]
    if s["mask_of"] is not None:
        there = s["mask_of"]
    k, v = (s[x].float().masked_fill(~there[:, :, None, None], 0.0) for x in "kv")
    return _attend_plain(s["q"].float(), k, v, there[:, None].expand(B, s["queries"], S)).to(DTYPES[s["dtype"]])


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    if own:
        ops = _ops()
        if s["op"] == "cross":
            return ops.cross_attention(s["q"], s["k"], s["v"], lengths=s["lengths"], mask=s["mask_of"])
        c = s["cache"]
        if s["op"] == "paged":
            return ops.paged_attention(s["q"], c["k_pages"], c["v_pages"], s["table"], s["lengths"], s["starts"], s["new"],
                                       k_stats=c["k_stats"], v_stats=c["v_stats"], codebooks=c["codebooks"])
        if s["write"]:
            ops.kv_cache_write(s["k"], s["v"], s["slots"], c["k_pages"], c["v_pages"], k_stats=c["k_stats"], v_stats=c["v_stats"],
                               thresholds=c["thresholds"], codebooks=c["codebooks"])
        return ops.kv_cache_read(s["slots"], c["k_pages"], c["v_pages"], k_stats=c["k_stats"], v_stats=c["v_stats"],
                                 codebooks=c["codebooks"], out_dtype=DTYPES[s["dtype"]])
    if s["op"] == "cross":
        return _cross_plain(s)
    if s["op"] == "paged":
        return _paged_plain(s)
    if s["write"]:
        _write_plain(s)
    return _read_plain(s)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_codes(packed, bits):
    """The code of value i is in bits [i * bits, (i + 1) * bits) of the row's bit stream."""
    b = packed.long()
    b = torch.cat([b, torch.zeros_like(b[..., :1])], -1)
    first = torch.arange(HEAD, device=packed.device) * bits
    return ((b[..., first // 8] + 256 * b[..., first // 8 + 1]) >> (first % 8)) & (2 ** bits - 1)


def _exact_token(c, name, i, page, offset):
    """Cached keys or values of tokens [n] in 64 bits, [n, kv_heads, 64]."""
    rows = c[name + "_pages"][page, :, offset]
    if c["bits"] == 16:
        return rows.double()
    stats = c[name + "_stats"][page, :, offset].double()
    return stats[..., :1] + stats[..., 1:] * c["codebooks"][i].double()[_exact_codes(rows, c["bits"])]


def _exact_attention(q, k, v, seen):
    """One sequence: q [n, H, 64], k and v [S, kv_heads, 64], seen [n, S], a head at a time."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        w = torch.einsum("nd,sd->ns", q[:, h].double(), k[:, h // group]) / math.sqrt(HEAD)
        w = torch.where(seen, w, torch.full_like(w, float("-inf")))
        some = seen.any(-1)
        if bool(some.any()):
            out[some, h] = torch.einsum("ns,sd->nd", torch.softmax(w[some], -1), v[:, h // group])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "cache":
        c, out = s["cache"], []
        for i, name in enumerate("kv"):
            if s["write"] and c["bits"] == 16:
                x = s[name].double()
            elif s["write"]:
                x = s[name].double()
                mean = x.sum(-1) / HEAD
                scale = torch.sqrt(((x - mean[..., None]) ** 2).sum(-1) / HEAD + 1e-6)
                t = (x - mean[..., None]) / scale[..., None]
                code = torch.zeros(t.shape, dtype=torch.long, device=t.device)
                for th in c["thresholds"][i].double():
                    code += t > th
                level = c["codebooks"][i].double()[code]
                center = mean - scale * level.sum(-1) / HEAD
                x = center.half().double()[..., None] + scale.half().double()[..., None] * level
            else:
                slots = s["slots"].clamp(min=0)
                x = _exact_token(c, name, i, slots // s["page"], slots % s["page"])
            out.append(torch.where((s["slots"] >= 0)[:, None, None], x, torch.zeros_like(x)))
        return out
    if s["op"] == "paged":
        lengths, new = _sequence_lengths(case)
        out = []
        for b, (L, n) in enumerate(zip(lengths, new)):
            j = torch.arange(L, device="cuda")
            pages = s["table"][b].long()[j // s["page"]]
            k, v = (_exact_token(s["cache"], name, i, pages, j % s["page"]) for i, name in enumerate("kv"))
            first = int(s["starts"][b])
            seen = j[None, :] <= (L - n + torch.arange(n, device="cuda"))[:, None]
            out.append(_exact_attention(s["q"][first:first + n], k, v, seen))
        return torch.cat(out)
    lengths = _state_lengths(case)
    out = []
    for b in range(s["batch"]):
        at = torch.arange(lengths[b], device="cuda") if s["mask_of"] is None else s["mask_of"][b].nonzero()[:, 0]
        seen = torch.ones(s["queries"], at.numel(), dtype=torch.bool, device="cuda")
        out.append(_exact_attention(s["q"][b], s["k"][b, at].double(), s["v"][b, at].double(), seen))
    return torch.stack(out)
