"""Cases and plain forms of the decoding-step operators, for timing and for comparison.

Four operators stand around the linear layers of one decoding step:

* ``rotate``: RMS norm of every query and key head with the position rotation, and the new keys
  and values put into a paged cache (``qk_norm_rope``, ``qk_norm_rope_append``);
* ``attend``: attention of one new token per sequence over the paged cache, with grouped heads,
  an optional window and first tokens that stay visible (``paged_attention``);
* ``int4``: linear layer for a few tokens with 4-bit weights and group scales (``int4_linear``);
* ``route``: scores, top-k and weights of a mixture-of-experts router (``route_experts``).

``own`` chooses between the elementary torch form of each (false) and the calls a user makes of
this package (true). ``exact`` holds each operator's definition in 64 bits.
"""

import math
import random

import torch

own = False

TABLE_POSITIONS = 131072


# ---- cases -----------------------------------------------------------------------------------

def listed():
    """The cases that are timed every time, smallest to largest within each operator."""
    return [
        # one user's decoding step: 64 query and 8 key heads of 128, one token into a cache of 16-token pages
        dict(name="rotate_one_token", op="rotate", tokens=1, heads=64, kv_heads=8, depth=128, rotary=128,
             interleaved=False, cache="bf16", page=16, pages=64),
        # a busy server's step: some rows are padding (no slot), 8-bit cache with pages of one token,
        # a quarter-odd head layout and a rotation of part of the depth in adjacent pairs
        dict(name="rotate_batch_fp8", op="rotate", tokens=203, heads=28, kv_heads=4, depth=80, rotary=32,
             interleaved=True, cache="e4m3", page=1, pages=4001),
        # prefill of a long prompt, queries and keys as slices of the packed projection
        dict(name="rotate_prefill", op="rotate", tokens=8192, heads=64, kv_heads=8, depth=128, rotary=128,
             interleaved=False, cache="none", page=0, pages=0),
        # one user, a short chat
        dict(name="attend_one_short", op="attend", batch=1, heads=64, kv_heads=8, depth=128, longest=300,
             page=16, cache="bf16", window=0, sinks=0),
        # a server's batch, lengths from nothing to 8191
        dict(name="attend_ragged_batch", op="attend", batch=48, heads=64, kv_heads=8, depth=128, longest=8191,
             page=16, cache="bf16", window=0, sinks=0),
        # one user with a book in the context
        dict(name="attend_one_long", op="attend", batch=1, heads=64, kv_heads=8, depth=128, longest=130977,
             page=64, cache="bf16", window=0, sinks=0),
        # streaming: a window of 1000 tokens behind four first ones, five query heads to a key head, 8-bit cache
        dict(name="attend_window_fp8", op="attend", batch=128, heads=40, kv_heads=8, depth=64, longest=4096,
             page=1, cache="e4m3", window=1000, sinks=4),
        # one token through a shard's key projection
        dict(name="int4_one_token_small", op="int4", rows=1, outputs=1280, inner=4096, group=128, zeros=False),
        # one token through the down projection 28672 -> 8192
        dict(name="int4_one_token_down", op="int4", rows=1, outputs=8192, inner=28672, group=128, zeros=False),
        # a small batch, fine groups with zero points, an odd number of outputs
        dict(name="int4_batch_zeros", op="int4", rows=37, outputs=5003, inner=7168, group=32, zeros=True),
        # one token's choice among 256 experts in eight groups
        dict(name="route_one_token", op="route", tokens=1, experts=256, choices=8, scoring="sigmoid", biased=True,
             groups=8, kept=4, renormalise=True, dtype="fp32"),
        # a prefill batch, softmax scores over bf16 logits, where equal scores are common
        dict(name="route_prefill", op="route", tokens=16384, experts=128, choices=8, scoring="softmax", biased=False,
             groups=1, kept=1, renormalise=True, dtype="bf16"),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(("rotate", "attend", "attend", "int4", "route"))
    if op == "rotate":
        depth = rng.choice((64, 80, 96, 128, 192, 256))
        kv_heads = rng.choice((1, 2, 4, 8))
        cache = rng.choice(("none", "bf16", "e4m3"))
        tokens = _log_int(rng, 1, 4096)
        page = rng.choice((1, 8, 16, 48, 64)) if cache != "none" else 0
        return dict(op=op, tokens=tokens, heads=kv_heads * rng.choice((1, 3, 4, 5, 8)), kv_heads=kv_heads, depth=depth,
                    rotary=rng.choice((depth, depth // 2)), interleaved=rng.random() < 0.5, cache=cache, page=page,
                    pages=-(-2 * tokens // page) + rng.randrange(1, 9) if page else 0)
    if op == "attend":
        batch = _log_int(rng, 1, 96)
        kv_heads = rng.choice((1, 2, 4, 8))
        depth = rng.choice((64, 96, 128, 128, 256))
        longest = _log_int(rng, 1, max(1, min(65536, (1 << 27) // (batch * kv_heads * depth))))
        window = rng.choice((0, 0, _log_int(rng, 1, 4096)))
        return dict(op=op, batch=batch, heads=kv_heads * rng.choice((1, 2, 4, 5, 8, 16)), kv_heads=kv_heads,
                    depth=depth, longest=longest, page=rng.choice((1, 5, 16, 64)),
                    cache=rng.choice(("bf16", "bf16", "e4m3")), window=window,
                    sinks=rng.choice((0, 1, 4, 37)) if window else 0)
    if op == "int4":
        group = rng.choice((32, 64, 128))
        return dict(op=op, rows=rng.choice((1, _log_int(rng, 1, 64))), outputs=_log_int(rng, 100, 16384),
                    inner=group * _log_int(rng, 512 // group, 16384 // group), group=group, zeros=rng.random() < 0.5)
    groups = rng.choice((1, 1, 4, 8))
    experts = groups * _log_int(rng, 8, 512 // groups)
    kept = rng.randrange(1, groups + 1)
    return dict(op=op, tokens=_log_int(rng, 1, 16384), experts=experts,
                choices=rng.randrange(1, min(16, kept * (experts // groups)) + 1),
                scoring=rng.choice(("softmax", "sigmoid")), biased=rng.random() < 0.5, groups=groups, kept=kept,
                renormalise=rng.random() < 0.5, dtype=rng.choice(("fp32", "bf16")))


def _lengths(case):
    """Visible lengths of an ``attend`` case: the longest, nothing where there are eight sequences
    or more, and lengths spread over the logarithm between."""
    rng = random.Random(case["batch"] * 1000003 + case["longest"])
    lengths = [_log_int(rng, 1, case["longest"]) for _ in range(case["batch"])]
    if case["batch"] >= 8:
        lengths[3] = 0
    lengths[case["batch"] // 2] = case["longest"]
    return lengths


def _seen(case, length):
    window, sinks = case["window"], case["sinks"]
    if not window or length <= window:
        return length
    return window + min(sinks, length - window)


# ---- inputs ----------------------------------------------------------------------------------

def _rotation(positions, rotary, base=500000.0):
    inverse = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inverse[None, :]
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def _to_cache(values, kind):
    return values.to(torch.float8_e4m3fn) if kind == "e4m3" else values.bfloat16()


def prepare(case, seed):
    """Inputs of one case on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def integers(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "rotate":
        tokens, heads, kv_heads, depth = case["tokens"], case["heads"], case["kv_heads"], case["depth"]
        packed = normal(tokens, heads + 2 * kv_heads, depth).bfloat16()
        state["q"], state["k"], state["v"] = packed.split((heads, kv_heads, kv_heads), dim=1)
        state["q_weight"] = (1 + 0.2 * normal(depth)).bfloat16()
        state["k_weight"] = (1 + 0.2 * normal(depth)).bfloat16()
        state["table"] = _rotation(TABLE_POSITIONS, case["rotary"])
        if case["cache"] == "none":
            start = TABLE_POSITIONS - tokens
            state["positions"] = torch.arange(start, start + tokens, device="cuda")
        else:
            state["positions"] = integers(0, TABLE_POSITIONS, tokens)
            shape = (case["pages"], case["page"], kv_heads, depth)
            state["key_cache"] = _to_cache(normal(*shape), case["cache"])
            state["value_cache"] = _to_cache(normal(*shape), case["cache"])
            slots = torch.randperm(case["pages"] * case["page"], generator=g, device="cuda")[:tokens]
            if tokens >= 16:  # padding rows of a fixed-size step
                slots[tokens - tokens // 16:] = -1
            state["slots"] = slots
            state["scales"] = (0.03125, 0.046875) if case["cache"] == "e4m3" else (1.0, 1.0)
    elif case["op"] == "attend":
        lengths, page = _lengths(case), case["page"]
        need = [-(-length // page) for length in lengths]
        width = max(1, max(need))
        total = sum(need) + 3
        order = torch.randperm(total, generator=g, device="cuda").int()
        column = torch.arange(width, device="cuda")
        counts = torch.tensor(need, device="cuda")
        first = counts.cumsum(0) - counts
        place = (first[:, None] + column[None, :]).clamp(max=total - 1)
        state["table"] = torch.where(column[None, :] < counts[:, None], order[place], -1).int().contiguous()
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        shape = (total, page, case["kv_heads"], case["depth"])
        state["scales"] = (0.5, 0.75) if case["cache"] == "e4m3" else (1.0, 1.0)
        state["key_cache"] = _to_cache(normal(*shape) / state["scales"][0], case["cache"])
        state["value_cache"] = _to_cache(normal(*shape) / state["scales"][1], case["cache"])
        state["q"] = (2 * normal(case["batch"], case["heads"], case["depth"])).bfloat16()
    elif case["op"] == "int4":
        outputs, inner, groups = case["outputs"], case["inner"], case["inner"] // case["group"]
        codes = integers(0, 256, outputs, inner // 2).to(torch.uint8)
        scale = (0.02 * (0.5 + torch.rand(outputs, groups, generator=g, device="cuda"))).bfloat16()
        zero = integers(0, 16, outputs, groups).to(torch.uint8) if case["zeros"] else None
        state["x"] = normal(case["rows"], inner).bfloat16()
        if own:
            from camblas_b200 import _kernels as cb

            state["weight"] = cb.Int4Weight(codes, scale, zero)  # laid out once, at load time
        else:
            state["codes"], state["scale"], state["zero"] = codes, scale, zero
    else:
        logits = 1.5 * normal(case["tokens"], case["experts"])
        state["logits"] = logits if case["dtype"] == "fp32" else logits.bfloat16()
        state["bias"] = 0.1 * normal(case["experts"]) if case["biased"] else None
    return state


# ---- one pass --------------------------------------------------------------------------------

def run(state):
    """One pass through the operator of the case, with the plain form or with this package."""
    if own:
        return _run_own(state)
    return {"rotate": _plain_rotate, "attend": _plain_attend, "int4": _plain_int4,
            "route": _plain_route}[state["op"]](state)


def _run_own(s):
    from camblas_b200 import _kernels as cb

    if s["op"] == "rotate":
        if s["cache"] == "none":
            return cb.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], 1e-6, s["positions"], s["table"],
                                   interleaved=s["interleaved"])
        q = cb.qk_norm_rope_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], 1e-6, s["positions"],
                                   s["table"], s["key_cache"], s["value_cache"], s["slots"],
                                   key_scale=s["scales"][0], value_scale=s["scales"][1],
                                   interleaved=s["interleaved"])
        return q, s["key_cache"], s["value_cache"]
    if s["op"] == "attend":
        return cb.paged_attention(s["q"], s["key_cache"], s["value_cache"], s["table"], s["lengths"],
                                  window=s["window"], sinks=s["sinks"], key_scale=s["scales"][0],
                                  value_scale=s["scales"][1])
    if s["op"] == "int4":
        return cb.int4_linear(s["x"], s["weight"])
    return cb.route_experts(s["logits"], s["choices"], bias=s["bias"], scoring=s["scoring"], groups=s["groups"],
                            kept_groups=s["kept"], renormalise=s["renormalise"], scale=2.5)


def _plain_head(x, weight, cos, sin, rotary, interleaved):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    turned, rest = x[..., :rotary], x[..., rotary:]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _plain_store(cache, values, slots, scale):
    rows = cache.view(-1, cache.shape[2], cache.shape[3])
    if cache.dtype == torch.float8_e4m3fn:
        values = (values / scale).clamp(-448, 448)
    kept = slots >= 0
    rows.view(torch.uint8 if cache.dtype == torch.float8_e4m3fn else cache.dtype)[slots[kept]] = (
        values[kept].to(cache.dtype).view(torch.uint8) if cache.dtype == torch.float8_e4m3fn
        else values[kept].to(cache.dtype))


def _plain_rotate(s):
    rotary = s["rotary"]
    angles = s["table"][s["positions"]]
    cos, sin = angles[:, :rotary // 2], angles[:, rotary // 2:]
    q = _plain_head(s["q"], s["q_weight"], cos, sin, rotary, s["interleaved"]).bfloat16()
    k = _plain_head(s["k"], s["k_weight"], cos, sin, rotary, s["interleaved"])
    if s["cache"] == "none":
        return q, k.bfloat16()
    _plain_store(s["key_cache"], k, s["slots"], s["scales"][0])
    _plain_store(s["value_cache"], s["v"].float(), s["slots"], s["scales"][1])
    return q, s["key_cache"], s["value_cache"]


def _plain_gather(cache, table, tokens):
    page = cache.shape[1]
    at = table[:, tokens // page].long().clamp(min=0) * page + tokens % page
    if cache.dtype == torch.float8_e4m3fn:
        return cache.view(torch.uint8).flatten(0, 1)[at].view(cache.dtype).float()
    return cache.flatten(0, 1)[at].float()


def _plain_attend(s):
    batch, heads, depth = s["q"].shape
    kv_heads = s["key_cache"].shape[2]
    tokens = torch.arange(s["table"].shape[1] * s["page"], device="cuda")
    length = s["lengths"][:, None]
    seen = tokens[None, :] < length
    if s["window"]:
        seen &= (tokens[None, :] >= length - s["window"]) | (tokens[None, :] < s["sinks"])
    q = s["q"].float().view(batch, kv_heads, heads // kv_heads, depth)
    k = _plain_gather(s["key_cache"], s["table"], tokens).permute(0, 2, 3, 1)
    scores = (q @ k) * (s["scales"][0] * depth ** -0.5)
    del k
    scores = torch.where(seen[:, None, None, :], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.where(seen[:, None, None, :], torch.exp(scores - top), 0.0)
    total = p.sum(-1, keepdim=True)
    v = _plain_gather(s["value_cache"], s["table"], tokens).permute(0, 2, 1, 3)
    out = (p @ v) * s["scales"][1] / torch.where(total > 0, total, 1.0)
    return out.view(batch, heads, depth).bfloat16()


def _plain_int4(s):
    codes = s["codes"]
    w = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1).float().unflatten(1, (-1, s["group"]))
    zero = 8.0 if s["zero"] is None else s["zero"].float()[:, :, None]
    w = ((w - zero) * s["scale"].float()[:, :, None]).flatten(1)
    return (s["x"].float() @ w.t()).bfloat16()


def _plain_route(s):
    # the choice is made between scores that may lie next to each other, so they are held in 64 bits
    logits, experts = s["logits"].double(), s["experts"]
    if s["scoring"] == "softmax":
        score = torch.exp(logits - logits.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-logits))
    rank = score if s["bias"] is None else score + s["bias"].double()
    if s["groups"] > 1:
        best = rank.view(-1, s["groups"], experts // s["groups"]).sort(-1, descending=True).values[..., :2].sum(-1)
        order = best.sort(dim=-1, descending=True, stable=True).indices[:, :s["kept"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, True)
        rank = torch.where(keep.repeat_interleave(experts // s["groups"], 1), rank, -math.inf)
    chosen = rank.sort(dim=-1, descending=True, stable=True).indices[:, :s["choices"]]
    weights = score.gather(1, chosen)
    if s["renormalise"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return chosen, (weights * 2.5).float()


# ---- what a pass cannot do without -----------------------------------------------------------

def work(case):
    """Bytes read once and written once, and operations, of one pass."""
    if case["op"] == "rotate":
        tokens, heads, kv_heads, depth = case["tokens"], case["heads"], case["kv_heads"], case["depth"]
        values = tokens * (heads + kv_heads) * depth
        size = 2 * 2 * values + tokens * (4 * case["rotary"] + 8) + 4 * depth
        if case["cache"] != "none":
            kept = tokens - (tokens // 16 if tokens >= 16 else 0)
            cell = 1 if case["cache"] == "e4m3" else 2
            # keys go to the cache in place of an output; values are read for the kept rows and written there
            size += 8 * tokens - 2 * tokens * kv_heads * depth + kept * kv_heads * depth * (2 * cell + 2)
        return dict(bytes=size, flops=7 * values)
    if case["op"] == "attend":
        cell = 1 if case["cache"] == "e4m3" else 2
        seen = sum(_seen(case, length) for length in _lengths(case))
        pages = sum(-(-_seen(case, length) // case["page"]) for length in _lengths(case))
        size = (2 * cell * seen * case["kv_heads"] * case["depth"] + 4 * pages + 4 * case["batch"]
                + 4 * case["batch"] * case["heads"] * case["depth"])
        return dict(bytes=size, flops=4 * seen * case["heads"] * case["depth"])
    if case["op"] == "int4":
        rows, outputs, inner = case["rows"], case["outputs"], case["inner"]
        groups = inner // case["group"]
        size = outputs * inner // 2 + outputs * groups * (3 if case["zeros"] else 2) + 2 * rows * (inner + outputs)
        return dict(bytes=size, flops=2 * rows * outputs * inner)
    cell = 4 if case["dtype"] == "fp32" else 2
    size = case["tokens"] * (case["experts"] * cell + case["choices"] * 12)
    return dict(bytes=size + (4 * case["experts"] if case["biased"] else 0), flops=6 * case["tokens"] * case["experts"])


# ---- the definitions in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    """What ``run`` returns, from each operator's definition in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "int4":
        return _exact_int4(case, s)
    return _exact_route(s)


def _exact_rotate(s):
    tokens, rotary = s["tokens"], s["rotary"]
    half = rotary // 2
    row = s["table"].double()[s["positions"]]
    turn = torch.complex(row[:, :half], row[:, half:]).view(tokens, 1, half)
    pair = torch.arange(rotary, device="cuda")
    pair = pair.view(half, 2) if s["interleaved"] else pair.view(2, half).t()

    def head(x, weight):
        x = x.double()
        y = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * weight.double()
        z = torch.complex(y[..., pair[:, 0]], y[..., pair[:, 1]]) * turn
        y[..., pair[:, 0]], y[..., pair[:, 1]] = z.real, z.imag
        return y

    q, k = head(s["q"], s["q_weight"]), head(s["k"], s["k_weight"])
    if s["cache"] == "none":
        return q, k

    def stored(cache, values, scale):
        after = cache.double()
        slot = s["slots"].tolist()
        kept = [i for i in range(tokens) if slot[i] >= 0]
        places = torch.tensor([slot[i] for i in kept], device="cuda")
        new = values[torch.tensor(kept, device="cuda")] / scale
        after[places // s["page"], places % s["page"]] = new.clamp(-448, 448) if s["cache"] == "e4m3" else new
        return after

    return q, stored(s["key_cache"], k, s["scales"][0]), stored(s["value_cache"], s["v"].double(), s["scales"][1])


def _exact_attend(s):
    batch, heads, depth = s["q"].shape
    kv_heads, page = s["kv_heads"], s["page"]
    out = torch.zeros(batch, heads, depth, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        visible = [t for t in range(length) if not s["window"] or t >= length - s["window"] or t < s["sinks"]]
        if not visible:
            continue
        t = torch.tensor(visible, device="cuda")
        where = s["table"][b].long()[t // page], t % page
        for h in range(kv_heads):
            k = s["key_cache"][:, :, h].double()[where] if s["cache"] == "e4m3" else s["key_cache"][where][:, h].double()
            v = (s["value_cache"][:, :, h].double()[where] if s["cache"] == "e4m3"
                 else s["value_cache"][where][:, h].double())
            rows = slice(h * heads // kv_heads, (h + 1) * heads // kv_heads)
            a = torch.softmax(s["q"][b, rows].double() @ k.t() * (s["scales"][0] / math.sqrt(depth)), dim=-1)
            out[b, rows] = a @ v * s["scales"][1]
    return out


def _exact_int4(case, s):
    if own:
        return None
    outputs, inner, group = case["outputs"], case["inner"], case["group"]
    x = s["x"].double()
    out = torch.zeros(case["rows"], outputs, dtype=torch.float64, device="cuda")
    for start in range(0, inner, group):
        byte = s["codes"][:, start // 2:(start + group) // 2].int()
        part = (x[:, start:start + group:2] @ (byte % 16).double().t()
                + x[:, start + 1:start + group:2] @ (byte // 16).double().t())
        zero = s["zero"][:, start // group].double() if s["zero"] is not None else torch.full_like(out[0], 8)
        part -= x[:, start:start + group].sum(-1, keepdim=True) * zero
        out += part * s["scale"][:, start // group].double()
    return out


def _exact_route(s):
    # the chosen experts are whole numbers, held against the plain form; the weights follow from them
    logits = s["logits"].double()
    score = torch.softmax(logits, -1) if s["scoring"] == "softmax" else torch.sigmoid(logits)
    rank = score.clone() if s["bias"] is None else score + s["bias"].double()
    tokens, experts = rank.shape
    if s["groups"] > 1:
        member = rank.view(tokens, s["groups"], -1)
        best = member.topk(min(2, member.shape[-1]), dim=-1).values.sum(-1)
        cut = best.topk(s["kept"], dim=-1).values[:, -1:]
        member[best < cut] = -math.inf
    chosen = rank.argsort(dim=-1, descending=True, stable=True)[:, :s["choices"]]
    weights = torch.take_along_dim(score, chosen, 1)
    if s["renormalise"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return None, weights * 2.5
