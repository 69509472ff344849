"""The decoding-step operators in 64 bits, written from their formulas, on whatever device the inputs lie.

Each function returns the exact value and a bound on the rounding of a kernel that keeps 32-bit sums and
rounds where the operator's documentation says.
"""

import math

import torch

HALF_STEP = {dtype: torch.finfo(dtype).eps / 2
             for dtype in (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn)}
U32 = HALF_STEP[torch.float32]


def norm_rope(x, weight, epsilon, positions, table, interleaved):
    """``[tokens, heads, depth]`` in 64 bits and the FP32 part of its bound.

    FP32 steps behind an element: the sum of squares is a tree of at most 8 + 5 additions and a
    square each (half of that relative error survives the root), a division, an addition, a root of
    two units, two products: below 16 units of each of the two rotated elements; two products and an
    addition of the rotation: below 20 units of |a| + |b|, taken as 32 of twice the largest element.
    """
    x = x.double()
    depth, rotary = x.shape[-1], table.shape[1]
    y = x if weight is None else x * (x.square().mean(-1, keepdim=True) + epsilon).rsqrt() * weight.double()
    bound = 64 * U32 * y.abs().amax(-1, keepdim=True).expand_as(y)
    inside = (positions >= 0) & (positions < table.shape[0])
    row = table.double()[positions.clamp(0, max(0, table.shape[0] - 1))] if table.shape[0] else table.double().new_zeros(
        x.shape[0], rotary)
    cos, sin = row[:, None, :rotary // 2], row[:, None, rotary // 2:]
    out = y.clone()
    first = slice(0, rotary, 2) if interleaved else slice(0, rotary // 2)
    second = slice(1, rotary, 2) if interleaved else slice(rotary // 2, rotary)
    out[..., first] = y[..., first] * cos - y[..., second] * sin
    out[..., second] = y[..., second] * cos + y[..., first] * sin
    out[~inside] = 0
    return out, bound


def attention(q, key_cache, value_cache, table, lengths, scale, window, sinks, key_scale=1.0, value_scale=1.0):
    """``[batch, heads, depth]`` in 64 bits, and its bound before the last rounding.

    The scores' FP32 sums are off by at most (depth + 8) units of sum |q||k|, which the exponential turns
    into a relative error of each weight, as do its own few units; a weight is rounded to BF16 (over
    an 8-bit cache to FP16) for the second product; sums over n tokens add n units at most.
    """
    batch, heads, depth = q.shape
    pages, page, kv_heads, _ = key_cache.shape
    group = heads // kv_heads
    out = torch.zeros(batch, heads, depth, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    rounding = HALF_STEP[torch.bfloat16 if key_cache.dtype == torch.bfloat16 else torch.float16]
    room = table.shape[1] * page
    for b in range(batch):
        length = min(max(int(lengths[b]), 0), room)
        keys, values = [], []
        for t in range(length):
            if window and t < length - window and t >= sinks:
                continue
            number = int(table[b, t // page])
            if 0 <= number < pages:
                keys.append((number, t % page))
        if not keys:
            continue
        where = torch.tensor(keys, device=q.device)
        k = key_cache.double()[where[:, 0], where[:, 1]] * key_scale
        v = value_cache.double()[where[:, 0], where[:, 1]] * value_scale
        for h in range(heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[b, h].double()
            p = torch.softmax(scale * (kh @ qh), 0)
            out[b, h] = p @ vh
            score_error = abs(scale) * (depth + 8) * U32 * float((kh.abs() @ qh.abs()).max())
            relative = rounding + 2 * score_error + (len(keys) + 64) * U32
            bound[b, h] = relative * (p @ vh.abs())
    return out, bound


def int4(x, codes, scale, zero=None):
    """``x @ W.T`` in 64 bits and its bound before the last rounding.

    A term passes through at most group / 16 + 16 additions inside its group, one scaling, one addition
    for every eighth block of 64 inputs and eight at the end.
    """
    outputs, groups = scale.shape
    group = 2 * codes.shape[1] // groups
    w = torch.stack((codes % 16, codes // 16), -1).double().view(outputs, groups, group)
    w = (w - (8 if zero is None else zero.double()[:, :, None])) * scale.double()[:, :, None]
    w = w.view(outputs, -1)
    steps = group // 16 + 16 + 1 + codes.shape[1] // 128 + 2 + 16
    return x.double() @ w.t(), steps * U32 * (x.double().abs() @ w.abs().t())


def route(logits, choices, bias=None, scoring="softmax", groups=1, kept_groups=1, renormalise=True, scale=1.0):
    """Ids and weights in 64 bits, token by token; a NaN ranks last, equal ranks in order of index."""
    logits = logits.double().cpu()
    bias = None if bias is None else bias.double().cpu()
    tokens, experts = logits.shape
    ids, weights = [], []
    for row in logits:
        if scoring == "sigmoid":
            score = [1 / (1 + math.exp(-v)) if v > -700 else 0.0 if v == v else v for v in row.tolist()]
        else:
            top = max([v for v in row.tolist() if v == v], default=0.0)
            top = 0.0 if top == -math.inf else top
            e = torch.exp(row - top)
            total = float(e.sum())
            score = (e / total).tolist() if total != 0 else [0.0] * experts
        rank = [s + (0.0 if bias is None else float(bias[i])) for i, s in enumerate(score)]

        def order(value):
            return -math.inf if value != value else value

        size = experts // groups
        best = []
        for g in range(groups):
            part = sorted((order(r) for r in rank[g * size:(g + 1) * size]), reverse=True)
            best.append(sum(part[:2]))
        kept = sorted(range(groups), key=lambda g: (-best[g], g))[:kept_groups]
        candidates = [e for e in range(experts) if e // size in kept]
        # a NaN behind every number, -inf included
        chosen = sorted(candidates, key=lambda e: (rank[e] != rank[e], -order(rank[e]) if rank[e] == rank[e] else 0, e))
        chosen = chosen[:choices]
        w = [score[e] for e in chosen]
        if renormalise:
            total = sum(w)
            w = [v / total if total != 0 else 0.0 for v in w]
        ids.append(chosen)
        weights.append([v * scale for v in w])
    return (torch.tensor(ids, dtype=torch.int64).view(tokens, choices),
            torch.tensor(weights, dtype=torch.float64).view(tokens, choices))


def within(actual, exact, bound):
    """Whether a rounded result lies within its bound plus half a step of its own type."""
    half = HALF_STEP[actual.dtype]
    error = (actual.double() - exact).abs()
    return bool((error <= bound * (1 + half) + half * exact.abs() + 1e-38).all())
