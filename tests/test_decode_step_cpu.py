"""Refusals and host logic of the decoding-step operators that need no GPU."""

import ctypes as ct

import pytest
import torch

from camblas_b200 import _kernels, _native


def bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_cpu_tensors_are_refused():
    q, k = bf16(2, 4, 64), bf16(2, 2, 64)
    w, table = bf16(64), torch.zeros(8, 64)
    positions = torch.zeros(2, dtype=torch.int64)
    cache = bf16(3, 4, 2, 64)
    with pytest.raises(ValueError):
        _kernels.qk_norm_rope(q, k, w, w, 1e-6, positions, table)
    with pytest.raises(ValueError):
        _kernels.qk_norm_rope_append(q, k, k, w, w, 1e-6, positions, table, cache, cache.clone(), positions)
    with pytest.raises(ValueError):
        _kernels.paged_attention(q, cache, cache.clone(), torch.zeros(2, 3, dtype=torch.int32),
                                 torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        _kernels.Int4Weight(torch.zeros(16, 32, dtype=torch.uint8), bf16(16, 1))
    with pytest.raises(ValueError):
        _kernels.int4_linear(q, q)
    with pytest.raises(ValueError):
        _kernels.route_experts(torch.zeros(2, 8), 2)


def test_null_context_is_a_status_not_a_crash():
    library = _native.library()
    null, strides = ct.c_void_p(), (ct.c_longlong * 12)()
    calls = (
        ("qk_norm_rope", (1, 1, 1, 64, 64, 0, 1e-6, null, null, null, strides, null, null, null, null, 1, null,
                          null, 0, null, null, 0, 1, 1.0, 1.0, null)),
        ("paged_attention", (1, 1, 1, 64, 1.0, null, 2, null, null, strides, 1, 1, 1.0, 1.0, null, 1, null, 0, 0,
                             null, 0, null)),
        ("int4_linear", (1, 32, 16, 32, null, 32, null, 2, 0, null, null, 0, null, 0, null, 16)),
        ("route_experts", (0, 1, 8, 2, 0, 1, 1, 1, 1.0, null, 8, null, null, null)),
    )
    for name, arguments in calls:
        assert getattr(library, "camblas_cuda_" + name)(None, *arguments) < 0
        assert b"missing context" in library.camblas_cuda_error(None)
    assert library.camblas_cuda_paged_attention_workspace(None, 1, 8, 8, 128, 2, 16, 4, 0, 0) == 0
    assert library.camblas_cuda_int4_linear_workspace(None, 1, 128, 64) == 0


def test_rotary_table_is_formed_in_64_bits():
    table = _kernels.rotary_table(200003, 64, base=10000.0, device="cpu")
    assert table.shape == (200003, 64) and table.dtype == torch.float32
    angle = 200002 * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    exact = torch.cat((angle.cos(), angle.sin()))
    # one rounding to FP32 of a value of at most 1, and the FP64 angle's own error (2e5 * 2^-52)
    assert (table[200002].double() - exact).abs().max() <= 2.0 ** -25 + 1e-9
    with pytest.raises(ValueError):
        _kernels.rotary_table(4, 7, device="cpu")
    assert _kernels.rotary_table(0, 8, device="cpu").shape == (0, 8)


@pytest.mark.parametrize("tiles,per,workers", [((1,), 1, 1), ((1, 1, 1), 8, 296), ((40, 1, 7), 3, 16),
                                               ((2047,), 8, 296), ((1, 300, 2, 5), 2, 148)])
def test_equal_ranges_cover_every_tile_once(tiles, per, workers):
    """The cut of the paged attention: ranges, their pieces' places, and the workers an item finds its pieces at."""
    def start(cta):
        return total // grid * cta + min(cta, total % grid)

    def owner(tile):
        each, longer = divmod(total, grid)
        return tile // (each + 1) if tile < longer * (each + 1) else longer + (tile - longer * (each + 1)) // each

    total = sum(tiles) * per
    grid = workers
    written, pieces = {}, {}
    for cta in range(grid):
        tile, end = start(cta), start(cta + 1)
        begin = tile
        while tile < end:
            sequence, first = 0, 0
            while first + tiles[sequence] * per <= tile:
                first += tiles[sequence] * per
                sequence += 1
            item = (tile - first) // tiles[sequence]
            at = first + item * tiles[sequence]
            upto = min(end - at, tiles[sequence])
            for j in range(tile - at, upto):
                assert (sequence, item, j) not in written
                written[sequence, item, j] = cta
            if (tile - at, upto) != (0, tiles[sequence]):
                place = 2 * cta + (0 if tile == begin else 1)
                assert place not in pieces
                pieces[place] = (sequence, item, tile - at, upto)
            tile = at + upto
    assert len(written) == total
    found = set()
    for sequence, count in enumerate(tiles):
        for item in range(per):
            first = sum(tiles[:sequence]) * per + item * count
            owners = sorted({written[sequence, item, j] for j in range(count)})
            assert owners == list(range(owner(first), owner(first + count - 1) + 1))
            if len(owners) == 1:
                continue
            reached = 0
            for cta in owners:
                place = 2 * cta + (1 if cta == owners[0] and start(cta) < first else 0)
                assert pieces[place][:3] == (sequence, item, reached)
                reached = pieces[place][3]
                found.add(place)
            assert reached == count
    assert found == set(pieces)
