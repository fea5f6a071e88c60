"""Measured cases of the low-bit decode operators: the 8-bit paged K/V cache (append, read-back,
attention), linear layers with 4-bit weights, and log probabilities of given tokens.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges, ``prepare`` makes a
case's inputs on the GPU, ``run`` is one pass: in plain torch operations, or through
``vflorence_b200.paged_ops`` when ``own`` is set. ``exact`` is the definition in 64 bits.
"""

import functools
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
ELEM = {"float32": 4, "bfloat16": 2}
TINY = 2.0 ** -100  # smaller scales are taken as zero


# ------------------------------------------------------------------------------------- cases

def listed():
    return [
        # float32 greedy decoding of a few requests: one token a request, where only latency counts
        append_case("append 4 tokens f32", "float32", 16, 64, 16, 4, (1, 63), (1, 1)),
        # a full decode batch: one token a request into partly filled blocks
        append_case("append 256 tokens bf16", "bfloat16", 16, 64, 16, 256, (1, 1023), (1, 1)),
        # encoder pages of 64 requests of about 580-590 tokens, written once
        append_case("encoder pages 64x585 bf16", "bfloat16", 12, 64, 16, 64, (0, 0), (580, 590)),
        # one request's cross-attention over 577 image tokens
        attention_case("attend 1x577 bf16", "bfloat16", 16, 16, 64, 16, 1, (577, 577), (1, 1), False),
        # three beams a request over shared encoder pages
        attention_case("attend 64x3 beams x585 bf16", "bfloat16", 12, 12, 64, 16, 64, (580, 590), (3, 3), False),
        # a full decode batch over long contexts of every length
        attention_case("attend 256x4096 bf16", "bfloat16", 16, 16, 64, 16, 256, (1, 4096), (1, 1), False),
        # grouped heads, float32 queries, a few causal rows a request, larger blocks
        attention_case("attend 8x4 causal grouped f32", "float32", 32, 8, 128, 32, 8, (200, 1000), (2, 5), True),
        # greedy decoding of a few requests: the step's tokens with five alternatives
        logprobs_case("logprobs 4x50265 f32", "float32", 4, 50265, 7, 5),
        # scoring given texts: odd row length, so rows start at any alignment
        logprobs_case("logprobs 1024x51289 bf16", "bfloat16", 1024, 51289, 0, 20),
        # one row through a projection of the decoder
        linear_case("linear 1x1024x1024 bf16", "bfloat16", 1, 1024, 1024, 64, True, False),
        # a small float32 batch through the feed-forward layer with its activation
        linear_case("linear 16x4096x1024 f32", "float32", 16, 4096, 1024, 128, True, True),
        # a large layer, where the weights' bytes decide
        linear_case("linear 8x16384x8192 bf16", "bfloat16", 8, 16384, 8192, 128, False, False),
    ]


def append_case(name, dtype, heads, dim, block, requests, past, new):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "dim": dim, "block": block,
            "requests": requests, "past_lo": past[0], "past_hi": past[1], "new_lo": new[0], "new_hi": new[1]}


def attention_case(name, dtype, heads, kv_heads, dim, block, requests, length, rows, causal):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "block": block, "requests": requests, "len_lo": length[0], "len_hi": length[1], "rows_lo": rows[0],
            "rows_hi": rows[1], "causal": causal}


def logprobs_case(name, dtype, rows, vocab, pad, k):
    return {"name": name, "op": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "pad": pad, "k": k}


def linear_case(name, dtype, rows, n, k, group, bias, gelu):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "n": n, "k": k, "group": group,
            "bias": bias, "gelu": gelu}


def log_int(rng, lo, hi):
    """An integer in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "logprobs", "linear"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "append":
        heads, dim, block = rng.choice([4, 8, 12, 16]), rng.choice([32, 64, 64, 80, 128]), rng.choice([16, 16, 32])
        if rng.random() < 0.5:
            case = append_case("", dtype, heads, dim, block, log_int(rng, 1, 512), (0, log_int(rng, 16, 1023)), (1, 1))
        else:
            length = log_int(rng, 3, 1024)
            requests = log_int(rng, 1, max(1, min(64, 64 * 585 // length)))
            case = append_case("", dtype, heads, dim, block, requests, (0, rng.choice([0, 40])), (max(1, length - 10), length))
    elif op == "attention":
        dim = rng.choice([32, 64, 64, 64, 96, 128, 256])
        kv_heads, group = rng.choice([2, 4, 8, 12, 16]), rng.choice([1, 1, 1, 2, 4, 7])
        block = rng.choice([16, 16, 32, 64])
        hi = log_int(rng, 17, 4096)
        lo = rng.choice([1, max(1, hi * 3 // 4), hi])
        rows = rng.choice([(1, 1), (1, 1), (3, 4), (0, 9)])
        most = 256 * 2048 * 16 * 64 // (kv_heads * dim * ((lo + hi + 1) // 2) * max(1, group * rows[1] // 16))
        requests = log_int(rng, 1, max(1, min(512, most)))
        case = attention_case("", dtype, kv_heads * group, kv_heads, dim, block, requests, (lo, hi), rows,
                              rows[1] > 1 and rng.random() < 0.5)
    elif op == "logprobs":
        vocab = log_int(rng, 500, 60000)
        rows = log_int(rng, 1, max(1, min(2048, 1024 * 51289 // vocab)))
        case = logprobs_case("", dtype, rows, vocab, rng.choice([0, 0, -vocab % 64, 3]), rng.choice([0, 1, 5, 20, 40]))
    else:
        group = rng.choice([32, 64, 128])
        k = group * log_int(rng, 256 // group, 8192 // group)
        n = log_int(rng, 100, 16384)
        case = linear_case("", dtype, log_int(rng, 1, 16), n, k, group, rng.random() < 0.5, rng.random() < 0.3)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------ inputs

def spread(lo, hi, count):
    """``count`` whole numbers evenly spread over [lo, hi]."""
    if count == 1:
        return [(lo + hi) // 2]
    return [lo + (hi - lo) * i // (count - 1) for i in range(count)]


def ceil_div(a, b):
    return -(-a // b)


def shuffled(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def paged_pool(case, heads, blocks, gen):
    """Random codes and scales of ``blocks`` cache blocks for K and V."""
    shape = (blocks, heads, case["block"], case["dim"])

    def codes():
        x = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
        y = torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda", generator=gen)
        return (x >> 1) + (y >> 1)  # bell-shaped, within [-128, 126]

    def scales():
        return (1.8 + torch.rand(shape[:2], device="cuda", generator=gen)) / 127.0

    return codes().clamp_(min=-127), codes().clamp_(min=-127), scales(), scales()


def tables(counts, seed):
    """Distinct random pool blocks for each request: (int32 [requests, widest], pool size)."""
    total = sum(counts)
    pool = total + total // 8 + 2
    order = list(range(pool))
    random.Random(seed).shuffle(order)
    width = max(max(counts), 1)
    rows, at = [], 0
    for c in counts:
        rows.append(order[at:at + c] + [0] * (width - c))
        at += c
    return torch.tensor(rows, dtype=torch.int32), pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = {"append": prepare_append, "attention": prepare_attention, "logprobs": prepare_logprobs,
            "linear": prepare_linear}
    return {"case": case, **make[case["op"]](case, seed, gen)}


def append_sizes(case):
    """(tokens already cached, new tokens) of each request, before they are shuffled."""
    return (spread(case["past_lo"], case["past_hi"], case["requests"]),
            spread(case["new_lo"], case["new_hi"], case["requests"]))


def prepare_append(case, seed, gen):
    both = shuffled(zip(*append_sizes(case)), seed)
    past, new = [x for x, _ in both], [x for _, x in both]
    bs, dtype = case["block"], DTYPES[case["dtype"]]
    table, pool = tables([ceil_div(p + n, bs) for p, n in both], seed + 1)
    k_cache, v_cache, k_scale, v_scale = paged_pool(case, case["heads"], pool, gen)

    def slots(first):
        """Slots of each request's positions from ``first(past)`` on."""
        req = torch.tensor([i for i, (p, n) in enumerate(zip(past, new)) for _ in range(first(p), p + n)])
        pos = torch.tensor([t for p, n in zip(past, new) for t in range(first(p), p + n)])
        return (table[req, pos // bs].long() * bs + pos % bs).cuda()

    write = slots(lambda p: p)
    rows = (write.numel(), case["heads"], case["dim"])
    size = 0.5 + torch.rand(rows[1:], device="cuda", generator=gen)  # channels differ in size
    key = (torch.randn(rows, device="cuda", generator=gen) * size).to(dtype)
    value = torch.randn(rows, device="cuda", generator=gen).to(dtype)
    return {"key": key, "value": value, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale,
            "v_scale": v_scale, "slots": write, "live": slots(lambda p: p // bs * bs)}


def attention_sizes(case):
    """(cached tokens, query rows) of each request, before they are shuffled."""
    return (spread(case["len_lo"], case["len_hi"], case["requests"]),
            spread(case["rows_lo"], case["rows_hi"], case["requests"]))


def prepare_attention(case, seed, gen):
    lens, rows = attention_sizes(case)
    both = shuffled(zip(lens, rows), seed)
    lens, rows = [x for x, _ in both], [x for _, x in both]
    table, pool = tables([ceil_div(n, case["block"]) for n in lens], seed + 1)
    k_cache, v_cache, k_scale, v_scale = paged_pool(case, case["kv_heads"], pool, gen)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    dtype = DTYPES[case["dtype"]]
    query = torch.randn((starts[-1], case["heads"], case["dim"]), device="cuda", generator=gen).to(dtype)
    lens_t, starts_t = torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32)
    state = {"query": query, "k_cache": k_cache, "v_cache": v_cache, "k_scale": k_scale, "v_scale": v_scale,
             "lens": lens_t.cuda(), "starts": starts_t.cuda(), "table": table.cuda(), "most_rows": max(rows),
             "scale": case["dim"] ** -0.5, "output": torch.empty_like(query)}
    if own:  # the launch plan that a decode loop keeps for its step
        state["plan"] = ops().get_scheduler_metadata_int8(
            case["requests"], case["heads"], case["kv_heads"], case["dim"], lens_t, dtype, starts_t, case["causal"],
            case["block"])
    return state


def prepare_logprobs(case, seed, gen):
    rows, vocab = case["rows"], case["vocab"]
    x = torch.randn((rows, vocab + case["pad"]), device="cuda", generator=gen)
    x = x.mul_(2.5).to(DTYPES[case["dtype"]])
    banned = torch.randint(0, vocab, (rows, 4), device="cuda", generator=gen)
    x.scatter_(1, banned, -math.inf)  # tokens that a decoding rule forbids
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen, dtype=torch.int32)
    return {"logits": x[:, :vocab], "targets": targets}


def prepare_linear(case, seed, gen):
    n, k, dtype = case["n"], case["k"], DTYPES[case["dtype"]]
    codes = torch.randint(0, 256, (n, k // 2), device="cuda", generator=gen, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((n, k // case["group"]), device="cuda", generator=gen)) * 0.01).to(dtype)
    x = torch.randn((case["rows"], k), device="cuda", generator=gen).to(dtype)
    bias = torch.randn(n, device="cuda", generator=gen).to(dtype) if case["bias"] else None
    return {"x": x, "codes": codes, "scales": scales, "bias": bias}


# ------------------------------------------------------------------------------------ passes

@functools.cache
def ops():
    """The framework's operators (only where ``own`` is set)."""
    from vflorence_b200 import paged_ops

    return paged_ops


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": own_append, "attention": own_attention, "logprobs": own_logprobs,
                "linear": own_linear}[op](state)
    return {"append": plain_append, "attention": plain_attention, "logprobs": plain_logprobs,
            "linear": plain_linear}[op](state)


def own_append(s):
    """Quantise and store the new tokens, then read the touched blocks' tokens back."""
    cache = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    ops().reshape_and_cache_int8(s["key"], s["value"], *cache, s["slots"])
    key, value = ops().gather_kv_int8(*cache, s["live"], s["key"].dtype)
    return {"key": key, "value": value, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def own_attention(s):
    ops().attention_with_kv_cache_int8(s["query"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"],
                                           s["output"], s["starts"], s["lens"], s["scale"], s["case"]["causal"],
                                           s["table"], s["plan"])
    return s["output"]


def own_logprobs(s):
    logprobs, entropy, values, indices = ops().token_logprobs(s["logits"], s["targets"], s["case"]["k"])
    return {"logprobs": logprobs, "entropy": entropy, "values": values, "indices": indices}


def own_linear(s):
    return ops().linear_int4(s["x"], s["codes"], s["scales"], s["bias"], "gelu" if s["case"]["gelu"] else None)


def plain_append(s):
    k, k_scale = plain_append_one(s["key"], s["k_cache"], s["k_scale"], s["slots"], s["live"])
    v, v_scale = plain_append_one(s["value"], s["v_cache"], s["v_scale"], s["slots"], s["live"])
    return {"key": k, "value": v, "k_scale": k_scale, "v_scale": v_scale}


def plain_append_one(rows, cache, scale, slots, live):
    bs = cache.shape[2]
    block, offset = slots // bs, slots % bs
    x = rows.float()
    largest = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    wanted = torch.zeros_like(scale).index_reduce_(0, block, largest, "amax") * (1.0 / 127.0)
    wanted = torch.where(wanted < TINY, 0.0, wanted)
    fresh = torch.zeros(scale.shape[0], dtype=torch.bool, device=x.device)
    fresh[block[offset == 0]] = True
    old = torch.where(fresh[:, None], 0.0, scale)
    new = torch.maximum(old, wanted)
    touched = torch.unique(block)
    inverse = torch.where(new > 0, 1.0 / new, 0.0)
    ratio = torch.where(fresh[:, None] | (new <= old), 1.0, old * inverse)[touched]
    cache[touched] = (cache[touched].float() * ratio[:, :, None, None]).round().to(torch.int8)
    codes = (x * inverse[block][:, :, None]).nan_to_num(0.0, math.inf, -math.inf).round().clamp(-127, 127)
    cache[block, :, offset] = codes.to(torch.int8)
    scale[touched] = new[touched]
    block, offset = live // bs, live % bs
    return (cache[block, :, offset].float() * scale[block][:, :, None]).to(rows.dtype), scale


def plain_attention(s):
    case = s["case"]
    bs, d, hkv = case["block"], case["dim"], case["kv_heads"]
    group, most = case["heads"] // hkv, s["most_rows"]
    table, lens = s["table"].long(), s["lens"].long()
    b, span = table.shape[0], table.shape[1] * bs

    def pages(cache, scale):
        x = cache[table].float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(b, hkv, span, d)

    row = torch.arange(most, device=table.device)
    starts = s["starts"].long()
    count = starts[1:] - starts[:-1]
    real = row[None] < count[:, None]
    at = (starts[:-1, None] + row[None]).clamp(max=s["query"].shape[0] - 1)
    q = s["query"][at].float().reshape(b, most, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    scores = (q @ pages(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * s["scale"]
    seen = lens[:, None] - (count[:, None] - 1 - row[None] if case["causal"] else 0)
    seen = seen.expand(b, most).repeat(1, group)
    mask = torch.arange(span, device=table.device)[None, None] < seen[:, :, None]
    scores = scores.masked_fill(~mask[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = pages(s["v_cache"], s["v_scale"])
    v = v.masked_fill((torch.arange(span, device=table.device)[None] >= lens[:, None])[:, None, :, None], 0.0)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    out = out.reshape(b, hkv, group, most, d).permute(0, 3, 1, 2, 4).reshape(b, most, hkv * group, d)
    return out[real].to(s["query"].dtype)


def plain_logprobs(s):
    k = s["case"]["k"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    chosen = x.gather(1, s["targets"].long()[:, None]) - lse
    logp = x - lse
    entropy = -(torch.where(e > 0, logp, 0.0) * (e / total)).sum(-1)
    values, indices = torch.sort(x, dim=-1, descending=True, stable=True)
    return {"logprobs": chosen[:, 0], "entropy": entropy, "values": values[:, :k] - lse,
            "indices": indices[:, :k].to(torch.int32)}


def plain_linear(s):
    case = s["case"]
    w = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).float() - 8.0
    w = w.reshape(case["n"], -1, case["group"]) * s["scales"].float()[..., None]
    y = s["x"].float() @ w.reshape(case["n"], case["k"]).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["gelu"]:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------------- bytes and operations

def work(case):
    es = ELEM[case["dtype"]]
    if case["op"] == "append":
        past, new = append_sizes(case)
        bs, row = case["block"], case["heads"] * case["dim"]
        tokens = sum(new)
        older = sum(p % bs for p in past)  # what the first touched blocks hold already
        # new tokens in, codes out, then the blocks' live tokens: codes in, values out
        moved = 2 * row * (tokens * (es + 1) + (tokens + older) * (1 + es)) + 8 * (2 * tokens + older)
        blocks = sum(ceil_div(p + n, bs) - p // bs for p, n in zip(past, new))
        return {"bytes": moved + 4 * 8 * case["heads"] * blocks, "flops": 4 * row * (2 * tokens + older)}
    if case["op"] == "attention":
        lens, rows = attention_sizes(case)
        blocks = sum(ceil_div(n, case["block"]) for n, r in zip(lens, rows) if r)
        tokens = sum(n for n, r in zip(lens, rows) if r)
        seen = sum(max(0, n - (r - 1 - i if case["causal"] else 0)) for n, r in zip(lens, rows) for i in range(r))
        cache = 2 * case["kv_heads"] * (tokens * case["dim"] + 4 * blocks) + 4 * blocks
        return {"bytes": cache + 2 * sum(rows) * case["heads"] * case["dim"] * es + 8 * case["requests"],
                "flops": 4 * seen * case["heads"] * case["dim"]}
    if case["op"] == "logprobs":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * es + case["rows"] * (12 + 8 * case["k"]), "flops": 6 * cells}
    n, k, rows = case["n"], case["k"], case["rows"]
    moved = n * k // 2 + n * (k // case["group"]) * es + rows * (k + n) * es + (n * es if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * rows * n * k}


# ------------------------------------------------------------------------------ 64-bit definition

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": exact_append, "attention": exact_attention, "logprobs": exact_logprobs,
            "linear": exact_linear}[case["op"]](s)


def exact_append(s):
    out = {}
    for name, cache, scale in (("key", s["k_cache"], s["k_scale"]), ("value", s["v_cache"], s["v_scale"])):
        bs = cache.shape[2]
        slots = s["slots"]
        x = s[name].double()
        steps = scale.double()
        steps.index_fill_(0, slots[slots % bs == 0] // bs, 0.0)  # blocks that start anew
        before = steps.clone()
        need = x.abs().amax(-1) / 127.0
        steps.scatter_reduce_(0, (slots // bs)[:, None].expand_as(need), need, "amax")
        grown = (before / steps.clamp(min=1e-300))[:, :, None, None]
        live = s["live"]
        kept = cache[live // bs, :, live % bs].double()
        kept = torch.round(kept * grown[live // bs, :, 0]) * steps[live // bs][:, :, None]
        # the new tokens' values replace those of their slots
        where = {int(t): i for i, t in enumerate(slots.tolist())}
        pick = torch.tensor([where.get(int(t), -1) for t in live.tolist()], device=x.device)
        step = steps[slots // bs][:, :, None]
        fresh = (torch.round(x / step.clamp(min=1e-300)) * step)[pick.clamp(min=0)]
        out[name] = torch.where((pick >= 0)[:, None, None], fresh, kept)
        out["k_scale" if name == "key" else "v_scale"] = steps
    return out


def exact_attention(s):
    case = s["case"]
    bs, hkv = case["block"], case["kv_heads"]
    group = case["heads"] // hkv
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for r, n in enumerate(lens):
        q0, q1 = starts[r], starts[r + 1]
        if q1 == q0 or n == 0:
            continue
        blocks = s["table"][r, : ceil_div(n, bs)].long()
        k, v = ((c[blocks].double() * z[blocks].double()[..., None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :n]
                for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        q = s["query"][q0:q1].double().transpose(0, 1)
        logits = torch.einsum("hqd,htd->hqt", q, k) * s["scale"]
        if case["causal"]:
            last = n - (q1 - q0 - 1 - torch.arange(q1 - q0, device="cuda"))
            hidden = torch.arange(n, device="cuda")[None] >= last[:, None]
            logits = logits.masked_fill(hidden[None], -math.inf)
        out[q0:q1] = torch.einsum("hqt,htd->qhd", logits.softmax(-1).nan_to_num(0.0), v)
    return out


def exact_logprobs(s):
    k = s["case"]["k"]
    logp = torch.cat([torch.log_softmax(part.double(), -1) for part in s["logits"].split(64)])
    p = logp.exp()
    return {"logprobs": logp.gather(1, s["targets"].long()[:, None])[:, 0],
            "entropy": torch.special.entr(p).sum(-1), "values": logp.topk(k, -1).values, "indices": None}


def exact_linear(s):
    case = s["case"]
    out = []
    x = s["x"].double()
    for codes, scales in zip(s["codes"].split(2048), s["scales"].split(2048)):
        w = torch.empty((codes.shape[0], case["k"]), dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
        w *= scales.double().repeat_interleave(case["group"], 1)
        out.append(x @ w.T)
    y = torch.cat(out, 1)
    if s["bias"] is not None:
        y = y + s["bias"].double()
    return torch.nn.functional.gelu(y) if case["gelu"] else y
