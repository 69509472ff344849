"""Decoding-step operators where types run out: small softmax weights, scores that tie, sums that cancel.

Held against the 64-bit definitions and bounds of ``decode_oracle``.
"""

import ctypes as ct

import pytest
import torch

from camblas_b200 import _kernels, _native
from tests import decode_oracle as exact
from tests.helpers import error_text, pointer, raw
from tests.test_decode_step_gpu import gen, int4_case, integers, normal, paged  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("heads,depth", [(3, 64), (16, 128), (4, 256)])
@pytest.mark.parametrize("ahead", [9.0, 12.5, 17.0, 20.0])
def test_small_weights_beside_a_dominant_token(gen, kind, heads, depth, ahead):
    """A first token that takes the weight and has the value zero: the result is made of the others' weights,
    e^-ahead of it."""
    length = 1500
    keys, values, table, counts = paged(gen, (length,), 16, 1, depth, BF16)
    first = int(table[0, 0])
    keys *= 0.25
    keys[..., 0] = 0
    keys[first, 0] = 0
    keys[first, 0, 0, 0] = 8
    values += 1
    values[first, 0] = 0
    keys, values = keys.to(kind), values.to(kind)
    q = (0.25 * normal(gen, 1, heads, depth)).to(BF16)
    q[..., 0] = 8
    out = _kernels.paged_attention(q, keys, values, table, counts, scale=ahead / 64)
    want, bound = exact.attention(q, keys, values, table, counts, ahead / 64, 0, 0)
    assert exact.within(out, want, bound)


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("heads,depth,length", [(1, 64, 23), (8, 128, 64), (16, 128, 40), (2, 256, 17), (12, 16, 61)])
def test_weights_keep_more_bits_than_the_values(gen, kind, heads, depth, length):
    """Values that nearly cancel under the weights show the rounding of the weights, which the result's own
    rounding hides elsewhere: two parts of eight (eleven) bits leave at most 2^-16 (2^-22) of each."""
    keys, values, table, counts = paged(gen, (length,), 16, 1, depth, kind)
    q = (0.5 * normal(gen, 1, heads, depth)).to(BF16)
    scale = depth ** -0.5
    last = int(table[0, (length - 1) // 16]), (length - 1) % 16
    k = torch.stack([keys[int(table[0, t // 16]), t % 16, 0] for t in range(length)]).double()
    v = torch.stack([values[int(table[0, t // 16]), t % 16, 0] for t in range(length)]).double()
    p = torch.softmax(scale * (q[0].double() @ k.t()), -1)[0]  # of the first head
    values[last][0] = (-(p[:-1] @ v[:-1]) / p[-1]).clamp(-400, 400).to(kind)
    out = _kernels.paged_attention(q, keys, values, table, counts, scale=scale)
    want, bound = exact.attention(q, keys, values, table, counts, scale, 0, 0)
    # the oracle's bound holds one rounding of the weights to BF16 (FP16); in its place the second part's
    half = exact.HALF_STEP[BF16 if kind is BF16 else torch.float16]
    v[-1] = values[last][0].double()
    p = torch.softmax(scale * (q[0].double() @ k.t()), -1)
    bound = bound - (half - half * half) * (p @ v.abs())[None]
    assert exact.within(out, want, bound)


@pytest.mark.parametrize("heads,depth", [(1, 64), (16, 128), (3, 256)])
def test_infinite_values_stay_infinite(gen, heads, depth):
    """A visible infinity has a positive weight: its column is infinite in its sign, and the others are finite."""
    keys, values, table, counts = paged(gen, (1, 150, 700), 16, 1, depth)
    q = normal(gen, 3, heads, depth).to(BF16)
    q[2] = 0  # weights that are powers of two, which a first part holds whole
    for b, t in ((0, 0), (1, 149), (2, 333)):
        row = values[int(table[b, t // 16]), t % 16, 0]
        row[3], row[depth - 1] = float("inf"), -float("inf")
    out = _kernels.paged_attention(q, keys, values, table, counts)
    assert (out[..., 3] == float("inf")).all() and (out[..., depth - 1] == -float("inf")).all()
    rest = torch.ones(depth, dtype=torch.bool, device="cuda")
    rest[3] = rest[depth - 1] = False
    assert out[..., rest].isfinite().all()


def attention_by_c(gen, batch=2, offset=0):
    """Status, message and output of a small call through the C ABI, the output `offset` elements into its buffer."""
    keys, values, table, counts = paged(gen, (30, 20), 16, 2, 64)
    q = normal(gen, 2, 4, 64).to(BF16)
    strides = (ct.c_longlong * 9)(q.stride(0), q.stride(1), *keys.stride()[:3], *values.stride()[:3], table.stride(0))
    size = _native.context(0).workspace_bytes("paged_attention", 2, 4, 2, 64, 2, 16, table.shape[1], 0, 0)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    buffer = torch.zeros(q.numel() + 4, dtype=BF16, device="cuda")
    out = buffer[offset:offset + q.numel()].view(q.shape)
    status, context = raw("paged_attention", batch, 4, 2, 64, 0.125, pointer(q), 2, pointer(keys), pointer(values),
                          strides, keys.shape[0], 16, 1.0, 1.0, pointer(table), table.shape[1], pointer(counts), 0, 0,
                          pointer(workspace), size, pointer(out))
    if status:
        assert not buffer.any()
    else:
        assert torch.equal(out, _kernels.paged_attention(q, keys, values, table, counts))
    return status, error_text(context) if status else ""


def test_attention_refuses_an_output_off_its_pairs(gen):
    for offset in (1, 3):
        status, message = attention_by_c(gen, offset=offset)
        assert status < 0 and "operands" in message
    assert attention_by_c(gen)[0] == 0 and attention_by_c(gen, offset=2)[0] == 0


def test_attention_counts_its_sequences_in_32_bits(gen):
    """The scans of the lengths step past the last sequence by up to 31."""
    sizes = 4, 2, 64, 2, 16, 2, 0, 0
    assert _native.context(0).workspace_bytes("paged_attention", 2 ** 29 - 1, *sizes) == 0
    assert _native.context(0).workspace_bytes("paged_attention", 2 ** 29 - 16, *sizes) >= 8 * (2 ** 29 - 16)
    status, message = attention_by_c(gen, batch=2 ** 29 - 1)
    assert status < 0 and "dimensions" in message
    status, message = attention_by_c(gen, batch=2 ** 29 - 16)  # a size that is taken, with too small a workspace
    assert status < 0 and "workspace" in message


def test_router_at_the_largest_number_of_tokens():
    """The step of the last warps passes 2^31."""
    tokens = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 45 * 2 ** 30:
        pytest.skip("needs 45 GB")
    logits = torch.zeros(tokens, 1, dtype=BF16, device="cuda")
    ids, weights = _kernels.route_experts(logits, 1, scoring="sigmoid", renormalise=False)
    del logits
    for start in range(0, tokens, 2 ** 28):
        assert not ids[start:start + 2 ** 28].any()
        assert (weights[start:start + 2 ** 28] == 0.5).all()
    del ids, weights
    torch.cuda.empty_cache()


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_groups_whose_ranks_cancel(gen, scoring):
    """Large biases of opposite sign in a group: the sum of its two ranks is small beside their rounding to FP32."""
    logits = torch.tensor([[1.503, 0.286, 1.711, 0.170]], device="cuda")
    bias = torch.tensor([1e4, -1e4, 1e4, -1e4], device="cuda")
    options = dict(bias=bias, scoring=scoring, groups=2, kept_groups=1)
    assert torch.equal(_kernels.route_experts(logits, 2, **options)[0].cpu(), exact.route(logits, 2, **options)[0])
    for experts, groups, kept in ((64, 32, 5), (96, 8, 3), (512, 4, 1)):
        logits = 1.5 * normal(gen, 60, experts)
        for size in (1e2, 1e4, 3e6, 3e38):
            bias = torch.where(torch.arange(experts, device="cuda") % 2 == 0, size, -size)
            bias[experts // 2] = 0.25
            options = dict(bias=bias, scoring=scoring, groups=groups, kept_groups=kept)
            ids, weights = _kernels.route_experts(logits, 4, **options)
            want_ids, want = exact.route(logits, 4, **options)
            assert torch.equal(ids.cpu(), want_ids)
            assert ((weights.cpu().double() - want).abs() <= (exact.U32 * 1.001 + 1e-12) * want.abs()).all()


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_cache_scales_mean_the_same_to_the_writer_and_the_reader(gen, kind):
    """value = entry * scale for either type of cache: what was appended under scales is attended over under them."""
    tokens, page, kv_heads, depth = 9, 4, 2, 64
    q, k, v = (normal(gen, tokens, n, depth).to(BF16) for n in (4, kv_heads, kv_heads))
    w = (1 + 0.3 * normal(gen, depth)).to(BF16)
    positions, slots = torch.arange(tokens, device="cuda"), torch.randperm(12, generator=gen, device="cuda")[:tokens]
    table = _kernels.rotary_table(16, depth)
    keys, values = (torch.zeros(3, page, kv_heads, depth, device="cuda").to(kind) for _ in range(2))
    scales = dict(key_scale=0.037, value_scale=0.0625 / 3)
    _kernels.qk_norm_rope_append(q, k, v, w, w, 1e-5, positions, table, keys, values, slots, **scales)
    new, bound = exact.norm_rope(k, w, 1e-5, positions, table, False)
    for cache, want, room, scale in ((keys, new, bound, scales["key_scale"]),
                                     (values, v.double(), torch.zeros_like(bound), scales["value_scale"])):
        entry = want / scale
        # the quotient adds a unit of FP32 and the scale's own rounding one; E4M3 has a fixed step below 2^-6
        room = room / scale + 3 * exact.U32 * entry.abs() + (2.0 ** -10 if kind == E4M3 else 0.0)
        got = cache.view(torch.uint8).flatten(0, 1)[slots].view(kind) if kind == E4M3 else cache.flatten(0, 1)[slots]
        assert exact.within(got, entry.clamp(-448, 448) if kind == E4M3 else entry, room)
    pages = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([12], dtype=torch.int32, device="cuda")
    out = _kernels.paged_attention(q[:1], keys, values, pages, counts, **scales)
    want, bound = exact.attention(q[:1], keys, values, pages, counts, depth ** -0.5, 0, 0, **scales)
    assert exact.within(out, want, bound + 4 * exact.U32 * want.abs())


def test_scales_of_one_change_no_bit_of_a_cache(gen):
    q, k, v = (normal(gen, 5, n, 80).to(BF16) for n in (2, 1, 1))
    positions = torch.arange(5, device="cuda")
    table = _kernels.rotary_table(8, 80)
    keys, values = (torch.zeros(2, 4, 1, 80, device="cuda", dtype=BF16) for _ in range(2))
    _kernels.qk_norm_rope_append(q, k, v, None, None, 0.0, positions, table, keys, values, positions)
    assert torch.equal(values.flatten(0, 1)[:5], v)
    assert torch.equal(keys.flatten(0, 1)[:5], _kernels.qk_norm_rope(q, k, None, None, 0.0, positions, table)[1])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_distinct_logits_of_equal_scores(gen, dtype):
    """Ranks are compared in FP64, where distinct logits can have one score: the lower index comes first, with a
    bias of zeros as without one."""
    inf = float("inf")
    sigmoid = [[40.0, 45.0, 1.0, 60.0], [1e-20, 2e-20, 0.0, -1.0], [-800.0, -750.0, -900.0, -710.0],
               [-inf, -800.0, -inf, 2.0], [15.0, 15.5, 16.0, 16.5], [39.0, 38.5, 38.0, 37.0]]
    softmax = [[0.0, -900.0, -800.0, -1.0], [0.0, 1e-20, -1e-20, 3e-20], [100.0, -640.0, -647.0, -800.0],
               [-inf, -800.0, 0.0, -750.0], [1000.0, 1.0, 2.0, 3.0], [5.0, 5.5, 6.0, 6.5]]
    for scoring, rows in (("sigmoid", sigmoid), ("softmax", softmax)):
        logits = torch.tensor(rows, device="cuda").to(dtype)
        for experts in (4, 40, 300):
            wide = torch.full((len(rows), experts), -inf, device="cuda", dtype=dtype)
            wide[:, torch.arange(4) * (experts // 4)] = logits
            for choices in (1, 2, 3, 4):
                ids, weights = _kernels.route_experts(wide, choices, scoring=scoring)
                want_ids, want = exact.route(wide, choices, scoring=scoring)
                assert torch.equal(ids.cpu(), want_ids)
                # below FP32's normal numbers the step is 2^-149, and a rounding off by up to half of it
                room = (exact.U32 * 1.001 + 1e-12) * want.abs() + 2.0 ** -150
                assert ((weights.cpu().double() - want).abs() <= room).all()
                zero = _kernels.route_experts(wide, choices, bias=torch.zeros(experts, device="cuda"), scoring=scoring)
                assert torch.equal(zero[0], ids) and torch.equal(zero[1], weights)


@pytest.mark.parametrize("scoring,spread", [("softmax", 400.0), ("sigmoid", 15.0), ("softmax", 1e-12)])
def test_saturated_scores_of_many_experts(gen, scoring, spread):
    logits = spread * normal(gen, 40, 128)
    for choices in (1, 8, 32):
        ids, _ = _kernels.route_experts(logits, choices, scoring=scoring)
        assert torch.equal(ids.cpu(), exact.route(logits, choices, scoring=scoring)[0])


@pytest.mark.parametrize("rows", [1, 8, 13, 40, 64, 70])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, True), (128, True), (128, False)])
def test_int4_codes_at_and_near_the_zero_point(gen, rows, group, zeros):
    """What the zero point takes away leaves no noise: rows of codes equal to it give zeros, rows within one of it
    keep the accuracy of their small weights, and a large input on a weight of zero leaves the others alone."""
    outputs, inner = 150, 512
    _, scale, zero = int4_case(gen, outputs, inner, group, True)
    if not zeros:
        zero = torch.full_like(zero, 8)
    whole = zero.int().repeat_interleave(group, 1)
    whole[50:100] = (whole[50:100] + integers(gen, -1, 2, 50, inner)).clamp(0, 15)
    whole[100:] = integers(gen, 0, 16, 50, inner).int()
    whole[100:, 77] = zero[100:, 77 // group].int()
    codes = (whole[:, ::2] + 16 * whole[:, 1::2]).to(torch.uint8)
    weight = _kernels.Int4Weight(codes, scale, zero if zeros else None)
    x = normal(gen, rows, inner).to(BF16)
    x[:, 77] = 2.0 ** 14
    out = _kernels.int4_linear(x, weight)
    assert not out[:, :50].any()
    assert exact.within(out, *exact.int4(x, codes, scale, zero))


@pytest.mark.parametrize("depth,rotary,interleaved", [(64, 64, False), (128, 64, True), (256, 256, False), (8, 8, True)])
def test_norm_of_heads_whose_squares_leave_the_range(gen, depth, rotary, interleaved):
    """Squares beyond FP32's largest number, and below its smallest ones where epsilon does not cover them."""
    sizes = (2.0 ** 62, 2.0 ** 90, 2.0 ** 125, 2.0 ** -66, 2.0 ** -90, 2.0 ** -118, 1.0)
    x = normal(gen, len(sizes), 3, depth)
    x = (x.clamp(-3, 3) * torch.tensor(sizes, device="cuda")[:, None, None]).to(BF16)
    x[2, 0] = torch.finfo(BF16).max
    w = (1 + 0.3 * normal(gen, depth)).to(BF16)
    table = _kernels.rotary_table(512, rotary)
    positions = integers(gen, 0, 512, len(sizes))
    for epsilon in (0.0, 1e-6):
        q_out, k_out = _kernels.qk_norm_rope(x, x[:, :1], w, w, epsilon, positions, table, interleaved=interleaved)
        want, bound = exact.norm_rope(x, w, epsilon, positions, table, interleaved)
        assert exact.within(q_out, want, bound)
        assert torch.equal(q_out[:, :1], k_out)
    zero = torch.zeros(1, 1, depth, device="cuda", dtype=BF16)
    assert not _kernels.qk_norm_rope(zero, zero, w, w, 1e-30, positions[:1], table)[0].any()
    zero[0, 0, 3] = float("inf")
    assert _kernels.qk_norm_rope(zero, zero, None, None, 1e-6, positions[:1] * 0, table)[0][0, 0, 3].isinf()


def test_scales_that_are_not_finite_are_refused(gen):
    keys, values, table, counts = paged(gen, (30,), 16, 2, 64)
    q = normal(gen, 1, 4, 64).to(BF16)
    for name in ("scale", "key_scale", "value_scale"):
        for value in (float("nan"), float("inf"), -float("inf")):
            with pytest.raises(ValueError):
                _kernels.paged_attention(q, keys, values, table, counts, **{name: value})
            with pytest.raises(ValueError):
                _kernels.route_experts(normal(gen, 2, 8), 2, scale=value)
