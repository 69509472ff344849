"""Head norm with rotation, paged attention, 4-bit linear and expert choice against 64-bit definitions.

Bounds are derived in ``decode_oracle`` from the number of FP32 steps and the roundings that the
operators document, each at most half a step of its type.
"""

import pytest
import torch

from camblas_b200 import _kernels, _native
from tests import decode_oracle as exact
from tests.helpers import error_text, pointer, raw

pytestmark = pytest.mark.gpu

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture
def gen():
    generator = torch.Generator(device="cuda")
    generator.manual_seed(20261208)
    return generator


def normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def integers(gen, low, high, *shape):
    return torch.randint(low, high, shape, generator=gen, device="cuda")


# ---- norm and rotation ----

@pytest.mark.parametrize("tokens,heads,kv_heads,depth,rotary,interleaved", [
    (1, 1, 1, 8, 8, False), (1, 64, 8, 128, 128, False), (7, 5, 1, 80, 32, True), (33, 6, 2, 64, 64, True),
    (129, 3, 3, 256, 256, False), (5, 4, 2, 96, 0, False), (3, 9, 3, 200, 104, False), (2, 2, 2, 128, 8, True)])
def test_norm_and_rotation(gen, tokens, heads, kv_heads, depth, rotary, interleaved):
    packed = normal(gen, tokens, heads + 2 * kv_heads, depth).to(BF16)
    q, k, _ = packed.split((heads, kv_heads, kv_heads), 1)
    qw, kw = (1 + 0.3 * normal(gen, depth)).to(BF16), (1 + 0.3 * normal(gen, depth)).to(BF16)
    table = _kernels.rotary_table(4097, rotary, base=500000.0)
    positions = integers(gen, 0, 4097, tokens)
    before = packed.clone()
    q_out, k_out = _kernels.qk_norm_rope(q, k, qw, kw, 1e-6, positions, table, interleaved=interleaved)
    assert q_out.is_contiguous() and k_out.is_contiguous() and torch.equal(packed, before)
    for out, x, w in ((q_out, q, qw), (k_out, k, kw)):
        assert exact.within(out, *exact.norm_rope(x, w, 1e-6, positions, table, interleaved))


def test_rotation_without_norm_keeps_lengths_and_padding_is_zero(gen):
    q, k = normal(gen, 6, 4, 64).to(BF16), normal(gen, 6, 2, 64).to(BF16)
    table = _kernels.rotary_table(100, 64)
    positions = torch.tensor([0, 99, 100, -1, 50, 2 ** 40], device="cuda")
    q_out, k_out = _kernels.qk_norm_rope(q, k, None, None, 0.0, positions, table)
    for out, x in ((q_out, q), (k_out, k)):
        assert exact.within(out, *exact.norm_rope(x, None, 0.0, positions, table, False))
        assert torch.equal(out[0], x[0])  # position 0 turns nothing
        assert not out[torch.tensor([2, 3, 5])].any()


def test_norm_of_zero_and_huge_heads(gen):
    q = torch.zeros(3, 2, 128, device="cuda", dtype=BF16)
    q[1] = 2.0 ** 60
    q[2] = 2.0 ** -70
    w = torch.ones(128, device="cuda", dtype=BF16)
    table = _kernels.rotary_table(4, 128)
    positions = torch.zeros(3, dtype=torch.int64, device="cuda")
    out, _ = _kernels.qk_norm_rope(q, q, w, w, 1e-6, positions, table)
    assert not out[0].any()
    assert torch.equal(out[1], torch.ones_like(out[1]))
    assert exact.within(out, *exact.norm_rope(q, w, 1e-6, positions, table, False))


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("page,heads_first,depth", [(1, False, 64), (16, False, 128), (5, True, 96), (64, True, 256)])
def test_append_writes_its_slots_and_nothing_else(gen, kind, page, heads_first, depth):
    tokens, heads, kv_heads, pages = 23, 6, 3, 40
    q, k, v = (normal(gen, tokens, n, depth).to(BF16) for n in (heads, kv_heads, kv_heads))
    v[3] *= 1000  # saturates an 8-bit cache
    w = (1 + 0.3 * normal(gen, depth)).to(BF16)
    table = _kernels.rotary_table(512, depth)
    positions = integers(gen, 0, 512, tokens)
    positions[5] = -3
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens]
    slots[7], slots[8] = -1, pages * page
    shape = (pages, kv_heads, page, depth) if heads_first else (pages, page, kv_heads, depth)
    caches = [normal(gen, *shape).to(kind) for _ in range(2)]
    if heads_first:
        caches = [cache.transpose(1, 2) for cache in caches]
    before = [cache.double() for cache in caches]
    scales = (0.05, 0.07) if kind == E4M3 else (1.0, 1.0)
    out = _kernels.qk_norm_rope_append(q, k, v, w, w, 1e-5, positions, table, *caches, slots,
                                       key_scale=scales[0], value_scale=scales[1])
    assert exact.within(out, *exact.norm_rope(q, w, 1e-5, positions, table, False))
    key, key_bound = exact.norm_rope(k, w, 1e-5, positions, table, False)
    for cache, old, new, bound, scale in ((caches[0], before[0], key, key_bound, scales[0]),
                                          (caches[1], before[1], v.double(), torch.zeros_like(key_bound), scales[1])):
        untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        for i in range(tokens):
            slot = int(slots[i])
            if not (0 <= slot < pages * page) or i == 5:
                continue
            untouched[slot // page, slot % page] = False
            got = cache[slot // page, slot % page]
            want = new[i] / scale
            if kind == E4M3:
                want = want.clamp(-448, 448)
                # below the smallest normal the step is fixed: half of 2^-9; the quotient adds a unit of FP32
                room = bound[i] / scale + 2 * exact.U32 * want.abs() + 2.0 ** -10
            else:
                room = bound[i]
            assert exact.within(got, want, room)
        assert torch.equal(cache.double()[untouched], old[untouched])


def test_rotation_refusals(gen):
    q, k = normal(gen, 4, 4, 64).to(BF16), normal(gen, 4, 2, 64).to(BF16)
    w, table = torch.ones(64, device="cuda", dtype=BF16), _kernels.rotary_table(8, 64)
    positions = torch.zeros(4, dtype=torch.int64, device="cuda")
    good = dict(q=q, k=k, q_weight=w, k_weight=w, epsilon=1e-6, positions=positions, table=table)
    for change in (dict(q=q.float()), dict(k=k[:3]), dict(k=k[..., :32]), dict(q=q[..., :60], k=k[..., :60]),
                   dict(q_weight=w[:32]), dict(k_weight=w.float()), dict(positions=positions.int()),
                   dict(positions=positions[:3]), dict(table=table.double()), dict(table=table[:, :12].contiguous()),
                   dict(table=torch.zeros(8, 72, device="cuda")), dict(epsilon=-1.0), dict(epsilon=float("nan")),
                   dict(q=q.clone().requires_grad_()), dict(q_weight=w.clone().requires_grad_())):
        with pytest.raises(ValueError):
            _kernels.qk_norm_rope(**{**good, **change})
    with torch.no_grad():
        _kernels.qk_norm_rope(**{**good, "q_weight": w.clone().requires_grad_()})
    cache = torch.zeros(3, 4, 2, 64, device="cuda", dtype=BF16)
    append = dict(good, v=k, key_cache=cache, value_cache=cache.clone(), slots=positions)
    for change in (dict(value_cache=cache), dict(value_cache=cache[:2].clone()), dict(value_cache=cache.to(E4M3)),
                   dict(key_cache=cache.half(), value_cache=cache.half()), dict(slots=positions.int()),
                   dict(v=k[:, :1]), dict(key_scale=0.0), dict(value_scale=float("inf")),
                   dict(key_cache=cache.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(ValueError):
            _kernels.qk_norm_rope_append(**{**append, **change})
    q_out, k_out = _kernels.qk_norm_rope(q[:0], k[:0], w, w, 1e-6, positions[:0], table)
    assert q_out.shape == (0, 4, 64) and k_out.shape == (0, 2, 64)


# ---- paged attention ----

def paged(gen, lengths, page, kv_heads, depth, kind=BF16, spare=3):
    """Caches, page table (-1 behind the last page of a sequence) and lengths for given sequences."""
    need = [-(-length // page) for length in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, count in enumerate(need):
        table[b, :count] = order[at:at + count]
        at += count
    caches = [normal(gen, pages, page, kv_heads, depth).to(kind) for _ in range(2)]
    return *caches, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("heads,kv_heads,depth,page,lengths,window,sinks", [
    (1, 1, 64, 1, (1,), 0, 0),
    (8, 1, 128, 16, (63, 64, 65, 0, 1, 300), 0, 0),
    (64, 8, 128, 16, (1000,), 0, 0),
    (12, 4, 96, 5, (17, 128, 0, 640), 0, 0),
    (10, 2, 64, 64, (700, 33, 257), 100, 3),
    (16, 1, 128, 7, (513, 2), 0, 0),
    (24, 1, 64, 16, (130, 129, 1), 64, 0),
    (40, 2, 256, 3, (200, 31), 0, 0),
    (9, 9, 80, 8, (65, 1, 0, 12), 5, 2),
    (4, 2, 16, 2, (40,), 39, 7),
    (2, 2, 208, 1, (90, 91), 1, 0),
    (3, 3, 72, 16, (33, 0, 70), 0, 0),
    (5, 1, 8, 4, (100,), 30, 2),
    (256, 1, 64, 1000, (400, 77), 0, 0),
    (33, 1, 128, 16, (260, 5), 0, 0),
    (36, 2, 192, 128, (150,), 2 ** 31 - 1, 2 ** 31 - 1),
])
def test_paged_attention(gen, kind, heads, kv_heads, depth, page, lengths, window, sinks):
    if kind == E4M3 and depth % 16:
        pytest.skip("an 8-bit depth is a multiple of 16")
    keys, values, table, counts = paged(gen, lengths, page, kv_heads, depth, kind)
    q = (2 * normal(gen, len(lengths), heads, depth)).to(BF16)
    scales = dict(key_scale=0.5, value_scale=1.5) if kind == E4M3 else {}
    out = _kernels.paged_attention(q, keys, values, table, counts, window=window, sinks=sinks, **scales)
    want, bound = exact.attention(q, keys, values, table, counts, depth ** -0.5, window, sinks, **scales)
    assert exact.within(out, want, bound)
    again = _kernels.paged_attention(q, keys, values, table, counts, window=window, sinks=sinks, **scales)
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_attention_never_reads_what_is_not_visible(gen, kind):
    """NaN and infinities behind the last token, outside the window and in other sequences' pages; bad page
    numbers inside the table take their tokens out; lengths beyond the table end with it."""
    lengths, page, kv_heads, depth = (37, 100, 70, 50, 90), 8, 2, 64
    keys, values, table, counts = paged(gen, lengths, page, kv_heads, depth, kind, spare=5)
    table[2, 1], table[2, 4] = -7, keys.shape[0]
    table[3, :] = 2 ** 31 - 1
    counts[4] = 10 ** 6  # 13 pages are listed, the last entries of its row are real
    table[4] = table[4].clamp(min=0)
    window, sinks = 40, 6
    q = normal(gen, len(lengths), 6, depth).to(BF16)
    seen = torch.zeros(keys.shape[:2], dtype=torch.bool, device="cuda")
    for b, length in enumerate(lengths):
        length = min(int(counts[b]), table.shape[1] * page)
        for t in range(length):
            number = int(table[b, t // page])
            if (t >= length - window or t < sinks) and 0 <= number < keys.shape[0]:
                seen[number, t % page] = True
    clean_keys, clean_values = keys.clone(), values.clone()
    for cache in (keys, values):
        cache.view(torch.uint8 if kind == E4M3 else torch.int16)[~seen] = 0x7f if kind == E4M3 else 0x7fc0
    out = _kernels.paged_attention(q, keys, values, table, counts, window=window, sinks=sinks)
    want, bound = exact.attention(q, clean_keys, clean_values, table, counts, depth ** -0.5, window, sinks)
    assert exact.within(out, want, bound)
    assert not out[3].any()


def test_attention_extreme_scores(gen):
    keys, values, table, counts = paged(gen, (200, 90, 1, 90), 16, 1, 128)
    q = normal(gen, 4, 8, 128).to(BF16)
    q[0] *= 100  # one token takes almost all weight
    q[1] = 0  # all weights equal
    out = _kernels.paged_attention(q, keys, values, table, counts, scale=1.0)
    want, bound = exact.attention(q, keys, values, table, counts, 1.0, 0, 0)
    assert exact.within(out, want, bound)
    keys[table[3, 0].long(), 3] = float("nan")  # a NaN that is seen reaches the result
    out = _kernels.paged_attention(q, keys, values, table, counts, scale=1.0)
    assert out[3].isnan().all() and not out[:3].isnan().any()


def test_eight_bit_attention_takes_queries_of_any_size(gen):
    """FP16 operands hold a BF16 query after a power of two is divided out per head."""
    keys, values, table, counts = paged(gen, (100,), 16, 1, 64, E4M3)
    q = normal(gen, 1, 4, 64).to(BF16)
    for factor, scale in ((2.0 ** 90, 2.0 ** -93), (2.0 ** -90, 2.0 ** 87)):
        out = _kernels.paged_attention((q.float() * factor).to(BF16), keys, values, table, counts, scale=scale)
        want, bound = exact.attention(q, keys, values, table, counts, 0.125, 0, 0)
        assert exact.within(out, want, bound)


def test_attention_over_strided_operands(gen):
    keys, values, table, counts = paged(gen, (77, 130), 16, 2, 64)
    heads_first = [cache.transpose(1, 2).contiguous().transpose(1, 2) for cache in (keys, values)]
    both = torch.stack((keys, values), dim=1)  # pages that hold keys and values side by side
    q = normal(gen, 2, 10, 64).to(BF16)
    wide = torch.empty(2, 13, 64, device="cuda", dtype=BF16)
    wide[:, 2:12] = q
    wide_table = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    expected = _kernels.paged_attention(q, keys, values, table, counts)
    for k, v in (heads_first, (both[:, 0], both[:, 1])):
        assert torch.equal(_kernels.paged_attention(wide[:, 2:12], k, v, wide_table[:, :table.shape[1]], counts),
                           expected)


def test_attention_offsets_beyond_32_bits(gen):
    """Two pages more than 2^31 elements apart."""
    apart = 2 ** 31 + 4096
    store = torch.empty(apart + 16 * 64, dtype=BF16, device="cuda")
    keys = store.as_strided((2, 16, 1, 64), (apart, 64, 64, 1))
    keys[:] = normal(gen, 2, 16, 1, 64).to(BF16)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    counts = torch.tensor([30], dtype=torch.int32, device="cuda")
    values = normal(gen, 2, 16, 1, 64).to(BF16)
    q = normal(gen, 1, 3, 64).to(BF16)
    out = _kernels.paged_attention(q, keys, values, table, counts)
    want, bound = exact.attention(q, keys.contiguous(), values, table, counts, 0.125, 0, 0)
    assert exact.within(out, want, bound)
    slots = torch.tensor([17], device="cuda")
    k = normal(gen, 1, 1, 64).to(BF16)
    _kernels.qk_norm_rope_append(q, k, k, None, None, 0.0, torch.zeros(1, dtype=torch.int64, device="cuda"),
                                 _kernels.rotary_table(1, 64), keys, values, slots)
    assert torch.equal(keys[1, 1], k[0]) and torch.equal(values[1, 1], k[0])


def test_many_sequences_of_all_lengths(gen):
    """More sequences than a warp scans at once, most of them shorter than a tile, some empty."""
    lengths = [int(v) for v in integers(gen, 0, 90, 77)]
    lengths[40] = 1500
    keys, values, table, counts = paged(gen, lengths, 4, 2, 64)
    q = normal(gen, 77, 4, 64).to(BF16)
    out = _kernels.paged_attention(q, keys, values, table, counts)
    want, bound = exact.attention(q, keys, values, table, counts, 0.125, 0, 0)
    assert exact.within(out, want, bound)


def test_a_large_batch_of_short_sequences(gen):
    """Several scans of 32 lengths, three key heads (one warp per team), sequences without tokens at both ends."""
    lengths = [0] + [int(v) for v in integers(gen, 0, 40, 698)] + [0]
    keys, values, table, counts = paged(gen, lengths, 8, 3, 32)
    q = normal(gen, 700, 3, 32).to(BF16)
    out = _kernels.paged_attention(q, keys, values, table, counts)
    want, bound = exact.attention(q, keys, values, table, counts, 32 ** -0.5, 0, 0)
    assert exact.within(out, want, bound)


def test_attention_in_graphs_follows_lengths(gen):
    """Two graphs of the same call on two streams, replayed side by side, with lengths that changed since."""
    keys, values, table, counts = paged(gen, (600, 600), 16, 2, 128)
    q = normal(gen, 2, 8, 128).to(BF16)
    graphs = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _kernels.paged_attention(q, keys, values, table, counts)  # creates the stream's context
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _kernels.paged_attention(q, keys, values, table, counts)
        graphs.append((stream, graph, out))
    for lengths in ((600, 600), (1, 599), (0, 65)):
        counts.copy_(torch.tensor(lengths, dtype=torch.int32))
        expected = _kernels.paged_attention(q, keys, values, table, counts)
        torch.cuda.synchronize()
        for _ in range(5):
            for stream, graph, _ in graphs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for _, _, out in graphs:
            assert torch.equal(out, expected)


def test_attention_refusals(gen):
    keys, values, table, counts = paged(gen, (30, 20), 16, 2, 64)
    q = normal(gen, 2, 4, 64).to(BF16)
    good = dict(q=q, key_cache=keys, value_cache=values, table=table, lengths=counts)
    offset = torch.empty(keys.numel() + 4, dtype=BF16, device="cuda")[4:].view(keys.shape)
    for change in (dict(q=q[:, :3]), dict(q=q.float()), dict(q=q[..., :32]), dict(table=table.long()),
                   dict(table=table[:1]), dict(lengths=counts.long()), dict(lengths=counts[:1]),
                   dict(window=-1), dict(sinks=-1), dict(value_cache=values.to(E4M3)), dict(key_cache=offset),
                   dict(value_cache=values[:1]), dict(q=q.clone().requires_grad_()),
                   dict(table=table.t().contiguous().t())):
        with pytest.raises(ValueError):
            _kernels.paged_attention(**{**good, **change})
    eight = torch.zeros(2, 16, 2, 72, device="cuda").to(E4M3)
    with pytest.raises(ValueError):
        _kernels.paged_attention(normal(gen, 2, 4, 72).to(BF16), eight, eight.clone(), table, counts)
    assert _kernels.paged_attention(q[:0], keys, values, table[:0], counts[:0]).shape == (0, 4, 64)
    empty = _kernels.paged_attention(q, keys[:0], values[:0], table, counts)  # a cache without pages
    assert not empty.any()
    assert not _kernels.paged_attention(q, keys, values, table[:, :0], counts).any()
    # through the C ABI: a workspace that is too small
    import ctypes as ct
    strides = (ct.c_longlong * 9)(q.stride(0), q.stride(1), *keys.stride()[:3], *values.stride()[:3], table.stride(0))
    out = torch.empty_like(q)
    status, context = raw("paged_attention", 2, 4, 2, 64, 0.125, pointer(q), 2, pointer(keys), pointer(values),
                          strides, keys.shape[0], 16, 1.0, 1.0, pointer(table), table.shape[1], pointer(counts), 0, 0,
                          pointer(out), 16, pointer(out))
    assert status < 0 and "workspace" in error_text(context)


# ---- 4-bit linear ----

def int4_case(gen, outputs, inner, group, zeros, scale_type=BF16):
    codes = integers(gen, 0, 256, outputs, inner // 2).to(torch.uint8)
    scale = (0.02 * (0.5 + torch.rand(outputs, inner // group, generator=gen, device="cuda"))).to(scale_type)
    zero = integers(gen, 0, 16, outputs, inner // group).to(torch.uint8) if zeros else None
    return codes, scale, zero


@pytest.mark.parametrize("rows,outputs,inner,group,zeros,scale_type", [
    (1, 1, 32, 32, False, BF16), (1, 16, 64, 64, True, BF16), (3, 17, 96, 32, True, torch.float32),
    (8, 1280, 4096, 128, False, BF16), (9, 100, 640, 128, True, torch.float32), (16, 33, 1024, 64, False, BF16),
    (17, 250, 224, 32, True, BF16), (32, 512, 2048, 128, False, torch.float32), (33, 48, 512, 64, True, BF16),
    (70, 1003, 1120, 32, False, BF16), (1, 4096, 14336, 128, True, BF16), (2, 64, 11008, 32, False, torch.float32),
    (3, 17000, 256, 64, True, BF16), (45, 130, 1536, 64, False, BF16), (130, 70, 416, 32, True, torch.float32)])
def test_int4_linear(gen, rows, outputs, inner, group, zeros, scale_type):
    codes, scale, zero = int4_case(gen, outputs, inner, group, zeros, scale_type)
    weight = _kernels.Int4Weight(codes, scale, zero)
    x = normal(gen, rows, inner).to(BF16)
    want, bound = exact.int4(x, codes, scale, zero)
    assert exact.within(_kernels.int4_linear(x, weight), want, bound)
    bias, residual = normal(gen, outputs).to(BF16), normal(gen, rows, outputs).to(BF16)
    # two additions more in FP32
    extra = bound + 2 * exact.U32 * (want.abs() + bias.double().abs() + residual.double().abs())
    assert exact.within(_kernels.int4_linear(x, weight, bias, residual),
                        want + bias.double() + residual.double(), extra)


@pytest.mark.parametrize("rows", [3, 40])
def test_int4_tokens_of_any_size(gen, rows):
    """Powers of two far beyond FP16's range and spread within a token keep the result's accuracy; what is not
    finite stays in its own token."""
    codes, scale, zero = int4_case(gen, 70, 256, 64, True)
    weight = _kernels.Int4Weight(codes, scale, zero)
    x = normal(gen, rows, 256).to(BF16)
    x[0] *= 2.0 ** 100
    x[1] *= 2.0 ** -120
    x[2, ::3] *= 2.0 ** -25
    want, bound = exact.int4(x, codes, scale, zero)
    assert exact.within(_kernels.int4_linear(x, weight), want, bound)
    clean = _kernels.int4_linear(x, weight)
    x[0, 17], x[1, 200] = float("inf"), float("nan")
    out = _kernels.int4_linear(x, weight)
    assert out[:2].isnan().all() and torch.equal(out[2:], clean[2:])


def test_int4_picks_single_weights(gen):
    """One-hot tokens read the matrix element by element: every code, place and scale is found."""
    outputs, inner, group = 40, 192, 64
    codes, scale, zero = int4_case(gen, outputs, inner, group, True)
    scale.fill_(1.0)
    x = torch.eye(inner, device="cuda").to(BF16)
    out = _kernels.int4_linear(x, _kernels.Int4Weight(codes, scale, zero))
    whole = torch.stack((codes % 16, codes // 16), -1).view(outputs, inner).int()
    whole = whole - zero.int().repeat_interleave(group, 1)
    assert torch.equal(out.t().int(), whole)


def test_int4_strided_and_shaped_operands(gen):
    codes, scale, zero = int4_case(gen, 96, 256, 128, False)
    weight = _kernels.Int4Weight(codes, scale)
    wide = normal(gen, 6, 520).to(BF16)
    expected = _kernels.int4_linear(wide[:, 8:264].contiguous(), weight)
    assert torch.equal(_kernels.int4_linear(wide[:, 8:264], weight), expected)
    assert torch.equal(_kernels.int4_linear(wide[:, 1:257], weight),  # 2-byte aligned rows are copied
                       _kernels.int4_linear(wide[:, 1:257].contiguous(), weight))
    assert torch.equal(_kernels.int4_linear(wide[:, 8:264].reshape(2, 3, 256), weight), expected.view(2, 3, 96))
    assert torch.equal(_kernels.int4_linear(wide[0, 8:264], weight), expected[0])
    residual = normal(gen, 6, 200).to(BF16)
    assert torch.equal(_kernels.int4_linear(wide[:, 8:264], weight, residual=residual[:, 4:100]),
                       _kernels.int4_linear(wide[:, 8:264], weight, residual=residual[:, 4:100].contiguous()))
    assert _kernels.int4_linear(wide[:0, 8:264], weight).shape == (0, 96)


@pytest.mark.parametrize("rows", [2, 20])
def test_int4_captured_beside_another_call(gen, rows):
    """A captured product keeps its own workspace: replays beside eager calls of other tokens give its own result."""
    codes, scale, zero = int4_case(gen, 300, 1024, 64, True)
    weight = _kernels.Int4Weight(codes, scale, zero)
    x, other = normal(gen, rows, 1024).to(BF16), normal(gen, rows, 1024).to(BF16)
    expected = [_kernels.int4_linear(value, weight) for value in (x, other)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _kernels.int4_linear(x, weight)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = _kernels.int4_linear(x, weight)
    for _ in range(20):
        with torch.cuda.stream(stream):
            graph.replay()
        assert torch.equal(_kernels.int4_linear(other, weight), expected[1])
        stream.synchronize()
        assert torch.equal(out, expected[0])


def test_int4_leaves_its_neighbours_alone(gen):
    """Rows and columns around a strided output, through the C ABI."""
    codes, scale, _ = int4_case(gen, 37, 128, 32, False)
    weight = _kernels.Int4Weight(codes, scale)
    x = normal(gen, 5, 128).to(BF16)
    out = torch.full((7, 50), float("nan"), device="cuda", dtype=BF16)
    size = _native.context(0).workspace_bytes("int4_linear", 5, 128, 32)
    workspace = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    workspace[size:] = 77
    status, context = raw("int4_linear", 5, 128, 37, 32, pointer(x), 128, pointer(weight.packed), 2, 0,
                          None, None, 0, pointer(workspace), size, pointer(out[1:, 3:]), 50)
    assert status == 0, error_text(context)
    assert torch.equal(out[1:6, 3:40], _kernels.int4_linear(x, weight))
    out[1:6, 3:40] = float("nan")
    assert out.isnan().all() and (workspace[size:] == 77).all()
    status, context = raw("int4_linear", 5, 128, 37, 32, pointer(x), 128, pointer(weight.packed), 2, 0,
                          None, None, 0, pointer(workspace), size - 1, pointer(out), 50)
    assert status < 0 and "workspace" in error_text(context)


def test_int4_refusals(gen):
    codes, scale, zero = int4_case(gen, 32, 128, 32, True)
    for arguments in ((codes.int(), scale), (codes, scale.half()), (codes, scale[:, :3]), (codes, scale[:16]),
                      (codes, scale, zero.int()), (codes, scale, zero[:, :2]), (codes, scale, zero + 16),
                      (codes[:, :8], scale[:, :1])):
        with pytest.raises(ValueError):
            _kernels.Int4Weight(*arguments)
    weight = _kernels.Int4Weight(codes, scale, zero)
    x = normal(gen, 2, 128).to(BF16)
    for change in (dict(x=x.float()), dict(x=x[:, :64]), dict(bias=torch.zeros(31, device="cuda", dtype=BF16)),
                   dict(residual=x), dict(x=x.clone().requires_grad_()), dict(weight=codes)):
        with pytest.raises(ValueError):
            _kernels.int4_linear(**{**dict(x=x, weight=weight), **change})


# ---- expert choice ----

@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,experts,choices,groups,kept,biased,dtype", [
    (1, 1, 1, 1, 1, False, torch.float32), (5, 8, 2, 1, 1, False, BF16), (33, 256, 8, 8, 4, True, torch.float32),
    (17, 65, 7, 1, 1, True, BF16), (9, 128, 8, 1, 1, False, BF16), (4, 512, 32, 4, 2, True, torch.float32),
    (3, 1024, 10, 32, 5, False, torch.float32), (6, 60, 6, 4, 2, True, BF16), (3, 16, 3, 16, 3, False, torch.float32),
    (2, 33, 32, 1, 1, True, torch.float32)])
def test_route_experts(gen, scoring, tokens, experts, choices, groups, kept, biased, dtype):
    logits = (1.5 * normal(gen, tokens, experts)).to(dtype)
    bias = 0.2 * normal(gen, experts) if biased else None
    for renormalise in (True, False):
        options = dict(bias=bias, scoring=scoring, groups=groups, kept_groups=kept, renormalise=renormalise, scale=2.5)
        ids, weights = _kernels.route_experts(logits, choices, **options)
        want_ids, want = exact.route(logits, choices, **options)
        assert torch.equal(ids.cpu(), want_ids)
        # FP64 inside (a float copy of scale), one rounding; 1e-12 for the exponentials and sums
        assert ((weights.cpu().double() - want).abs() <= (exact.U32 * 1.001 + 1e-12) * want.abs()).all()


def test_equal_ranks_go_to_the_lower_index(gen):
    logits = torch.zeros(3, 96, device="cuda")
    logits[1, 40:] = 1
    ids, weights = _kernels.route_experts(logits, 5)
    assert ids.tolist() == [[0, 1, 2, 3, 4], [40, 41, 42, 43, 44], [0, 1, 2, 3, 4]]
    assert torch.allclose(weights, torch.full_like(weights, 0.2))
    ids, _ = _kernels.route_experts(logits, 5, scoring="sigmoid", groups=8, kept_groups=2)
    # groups of twelve: in the middle row the first two with two large members are 36..47 and 48..59
    assert ids.tolist() == [[0, 1, 2, 3, 4], [40, 41, 42, 43, 44], [0, 1, 2, 3, 4]]
    # ranks that differ in the 40th bit only
    bias = torch.zeros(64, device="cuda")
    close = torch.zeros(1, 64, device="cuda")
    close[0, 50], close[0, 3] = 4.0, 4.0
    bias[50] = 2.0 ** -40
    ids, _ = _kernels.route_experts(close, 2, bias=bias, scoring="sigmoid")
    assert ids.tolist() == [[50, 3]]


def test_closed_and_broken_rows(gen):
    """Rows of -inf, of NaN and of mixtures give valid distinct ids; a closed expert has weight 0."""
    inf, nan = float("inf"), float("nan")
    logits = normal(gen, 6, 40)
    logits[0] = -inf
    logits[1] = nan
    logits[2, :38] = -inf
    logits[3, 7] = nan
    logits[4, 5] = inf
    logits[5] = torch.finfo(torch.float32).min
    for scoring in ("softmax", "sigmoid"):
        ids, weights = _kernels.route_experts(logits, 4, scoring=scoring)
        assert ((ids >= 0) & (ids < 40)).all()
        assert all(len(set(row)) == 4 for row in ids.tolist())
        assert ids[0].tolist() == [0, 1, 2, 3] and not weights[0].any()
        assert ids[1].tolist() == [0, 1, 2, 3]
        assert sorted(ids[2, :2].tolist()) == [38, 39] and ids[2, 2:].tolist() == [0, 1]
        assert not weights[2, 2:].any()
        assert abs(float(weights[2].sum()) - 1) < 1e-6
    ids, weights = _kernels.route_experts(logits, 4, scoring="sigmoid")
    assert 7 not in ids[3].tolist() and weights[3].isfinite().all()
    assert ids[4, 0] == 5


def test_more_tokens_than_a_grid_holds(gen):
    logits = normal(gen, 270001, 12)
    ids, weights = _kernels.route_experts(logits, 3, scoring="sigmoid", renormalise=False)
    ranked = logits.double().sort(dim=1, descending=True, stable=True)
    assert torch.equal(ids, ranked.indices[:, :3])
    want = torch.sigmoid(ranked.values[:, :3])
    assert ((weights.double() - want).abs() <= (exact.U32 * 1.001 + 1e-12) * want).all()


def test_route_strided_and_refusals(gen):
    wide = normal(gen, 6, 70)
    expected = _kernels.route_experts(wide[:, 3:35].contiguous(), 4)
    for view in (wide[:, 3:35], wide[:, 3:35].t().contiguous().t()):
        got = _kernels.route_experts(view, 4)
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
    logits = wide[:, :32].contiguous()
    for change in (dict(choices=0), dict(choices=33), dict(groups=5), dict(groups=0), dict(groups=4, kept_groups=5),
                   dict(groups=16, kept_groups=1), dict(scoring="relu"), dict(bias=torch.zeros(31, device="cuda")),
                   dict(bias=torch.zeros(32, device="cuda", dtype=BF16)), dict(logits=logits.double()),
                   dict(logits=logits[0]), dict(logits=logits.clone().requires_grad_()),
                   dict(logits=torch.zeros(1, 1025, device="cuda"))):
        with pytest.raises(ValueError):
            _kernels.route_experts(**{**dict(logits=logits, choices=4), **change})
    ids, weights = _kernels.route_experts(logits[:0], 4)
    assert ids.shape == (0, 4) and weights.dtype == torch.float32


# ---- together ----

def decode_step(x, layer, state):
    """One layer of a decoding step, as a serving loop would call it."""
    normed = _kernels.rms_norm(x, layer["norm"], 1e-6)
    q, k, v = _kernels.int4_linear(normed, layer["qkv"]).view(x.shape[0], -1, 64).split((8, 2, 2), 1)
    q = _kernels.qk_norm_rope_append(q, k, v, layer["q_norm"], layer["k_norm"], 1e-6, state["positions"],
                                     layer["table"], state["keys"], state["values"], state["slots"])
    mixed = _kernels.paged_attention(q, state["keys"], state["values"], state["pages"], state["lengths"])
    x = _kernels.int4_linear(mixed.flatten(1), layer["out"], residual=x)
    ids, weights = _kernels.route_experts(_kernels.linear(x, layer["router"]), 2, scoring="sigmoid",
                                          bias=layer["bias"])
    slots, reverse, counts = _kernels.route_groups(ids, layer["experts"], 0, 16)
    return x, ids, weights, slots, reverse, counts


def test_a_decoding_step_eager_and_captured(gen):
    batch, hidden, page = 4, 256, 16
    layer = dict(norm=torch.ones(hidden, device="cuda", dtype=BF16),
                 q_norm=(1 + 0.1 * normal(gen, 64)).to(BF16), k_norm=(1 + 0.1 * normal(gen, 64)).to(BF16),
                 table=_kernels.rotary_table(256, 64), router=(0.1 * normal(gen, 16, hidden)).to(BF16),
                 bias=0.05 * normal(gen, 16), experts=torch.arange(16, dtype=torch.int32, device="cuda"))
    raw_weights = {}
    for name, outputs, inner in (("qkv", 12 * 64, hidden), ("out", hidden, 8 * 64)):
        codes, scale, zero = int4_case(gen, outputs, inner, 64, True)
        raw_weights[name] = (codes, scale, zero)
        layer[name] = _kernels.Int4Weight(codes, scale, zero)
    pages = torch.randperm(batch * 4, generator=gen, device="cuda").int().view(batch, 4)
    state = dict(keys=torch.zeros(batch * 4, page, 2, 64, device="cuda", dtype=BF16),
                 values=torch.zeros(batch * 4, page, 2, 64, device="cuda", dtype=BF16), pages=pages,
                 positions=torch.zeros(batch, dtype=torch.int64, device="cuda"),
                 slots=torch.zeros(batch, dtype=torch.int64, device="cuda"),
                 lengths=torch.zeros(batch, dtype=torch.int32, device="cuda"))
    x = torch.zeros(batch, hidden, device="cuda", dtype=BF16)

    def place(step):
        state["positions"].fill_(step)
        state["lengths"].fill_(step + 1)
        state["slots"].copy_(pages[:, step // page].long() * page + step % page)

    inputs = [normal(gen, batch, hidden).to(BF16) for _ in range(40)]
    stream = torch.cuda.Stream()
    eager = []
    with torch.no_grad():
        for step, value in enumerate(inputs):
            place(step)
            x.copy_(value)
            eager.append([t.clone() for t in decode_step(x, layer, state)])
        keys_after = state["keys"].clone()
        # the last step against 64 bits, from the cache that it left
        normed = _kernels.rms_norm(x, layer["norm"], 1e-6)
        qkv = _kernels.int4_linear(normed, layer["qkv"])
        assert exact.within(qkv, *exact.int4(normed, *raw_weights["qkv"]))
        q = qkv.view(batch, -1, 64)[:, :8]
        q_new, bound = exact.norm_rope(q, layer["q_norm"], 1e-6, state["positions"], layer["table"], False)
        q_out, _ = _kernels.qk_norm_rope(q, qkv.view(batch, -1, 64)[:, 8:10], layer["q_norm"], layer["k_norm"], 1e-6,
                                         state["positions"], layer["table"])
        assert exact.within(q_out, q_new, bound)
        mixed = _kernels.paged_attention(q_out, state["keys"], state["values"], pages, state["lengths"])
        assert exact.within(mixed, *exact.attention(q_out, state["keys"], state["values"], pages, state["lengths"],
                                                    0.125, 0, 0))
        # the same steps from a graph
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            decode_step(x, layer, state)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured = decode_step(x, layer, state)
        state["keys"].zero_(), state["values"].zero_()
        for step, value in enumerate(inputs):
            place(step)
            x.copy_(value)
            graph.replay()
            for got, want in zip(captured, eager[step]):
                assert torch.equal(got, want)
        assert torch.equal(state["keys"], keys_after)
    assert _native.context(0).device_status() == 0


def test_calls_run_on_the_current_stream(gen):
    """Work queued on a side stream sees what that stream did before."""
    stream = torch.cuda.Stream()
    keys, values, table, counts = paged(gen, (100,), 16, 1, 64)
    q = normal(gen, 1, 4, 64).to(BF16)
    expected = _kernels.paged_attention(2 * q, keys, values, table, counts)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        later = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        later.copy_(2 * q)
        out = _kernels.paged_attention(later, keys, values, table, counts)
    stream.synchronize()
    assert torch.equal(out, expected)
