"""Calls around the 4-bit cache that are refused, or decided on the host, where their first tests did not look."""

from __future__ import annotations

import weakref

import numpy as np
import pytest
import torch


@pytest.mark.parametrize("rot", [64, 32, 0])
@pytest.mark.parametrize("fp4", [True, False])
def test_backend_refuses_positions_behind_the_rotation_table(mlb, fp4, rot):
    """A key at such a position has no rotation: nothing may reach the cache, whichever launch would have made it."""
    shape, dtype = ((4, 2, 17, 32), torch.uint8) if fp4 else ((4, 16, 2, 64), torch.bfloat16)
    pools = [torch.full(shape, 7, dtype=dtype) for _ in range(2)]
    meta = mlb.AttentionMetadata.build([mlb.SeqStep(0, 2, [1]), mlb.SeqStep(19, 1, [0, 2])], 16, "cpu")
    q, k = torch.zeros(3, 8, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    backend = mlb.get_backend("b200")
    with pytest.raises(ValueError, match="position 19 .* 19 rows"):
        backend.forward(q, k, k, *pools, meta, rotary=mlb.Rotary(torch.zeros(19, rot)))
    assert all((p == 7).all() for p in pools)
    with pytest.raises(ValueError, match="CUDA"):  # the last position that has a row: on to the entry points' own checks
        backend.forward(q, k, k, *pools, meta, rotary=mlb.Rotary(torch.zeros(20, rot)))


def test_plan_knows_the_last_position_of_a_new_token(mlb):
    lens, width = [40, 900, 7], 57
    for qo, last in (([0, 3, 3, 4], 39), ([0, 0, 1, 1], 899), ([0, 0, 0, 0], -1)):  # rows without new tokens do not count
        assert mlb.plan_attention(qo, lens, width, 8, 2, "cpu").last_position == last


def test_attention_refuses_a_scale_that_overflows(mlb):
    """scale * log2(e) is what the kernels multiply by."""
    L = mlb.ops._lib

    def call(scale):
        f = 1 << 20  # a pointer that is never followed
        return L.lib().mlb_paged_attention_fp4(f, 512, 64, f, f, 2, 4, 8, 2, 64, scale, f, 1, f, f, 1, f, 0, None, 0, None,
                                               None, None, 0, f, 512, 64, None, None, None)

    assert call(2.3e38) == L.MLB_OK  # no units: nothing to do
    for scale in (2.5e38, 3.4e38, -2.5e38):
        assert call(scale) == L.MLB_EINVAL and "scale" in L.last_error()


def test_workspace_gives_back_large_buffers_that_it_has_outgrown(mlb):
    """Scratch of gigabytes (on the meta device: sizes without memory): one buffer at a time, no larger than asked."""
    ws, dev = mlb.Workspace(), torch.device("meta")
    first = [weakref.ref(t) for t in ws.get(1 << 17, 32, 128, dev)]
    assert all(r() is not None for r in first)
    o, lse = ws.get((1 << 17) + 1, 32, 128, dev)
    assert o.numel() == ((1 << 17) + 1) * 32 * 128 and lse.numel() == ((1 << 17) + 1) * 32
    assert all(r() is None for r in first)
    assert ws.get(5, 32, 128, dev)[0] is o  # smaller asks share it
    assert ws.get((1 << 16) + 2, 64, 64, dev)[0] is not o  # more row sums than it has
    assert ws.get(1, 32, 128, torch.device("cpu"))[0].numel() == 32 * 128
    assert ws.get((1 << 17) + 1, 32, 128, dev)[1].numel() == ((1 << 16) + 2) * 64


def test_workspace_releases_what_it_keeps(mlb):
    ws, dev = mlb.Workspace(), torch.device("cpu")
    first = [weakref.ref(t) for t in ws.get(4, 2, 64, dev)]
    last = ws.get(5, 2, 64, dev)
    assert all(r() is not None for r in first)
    ws.release()
    assert all(r() is None for r in first) and ws.get(5, 2, 64, dev)[0] is last[0]


def test_reduction_goes_by_pieces_and_by_rows(mlb):
    """A CTA per (token, head) is for few rows of many pieces: thousands of unsplit rows beside one long row would
    launch a CTA each that has nothing to do."""

    def plan(lens, new):  # with block tables, as the backend plans: long chunks become query tiles
        tables = np.arange(len(lens) * 8192, dtype=np.int32).reshape(len(lens), 8192)
        return mlb.plan_attention([sum(new[:i]) for i in range(len(new) + 1)], lens, 8192, 32, 8, "cpu",
                                  pool_dtype=torch.uint8, block_tables_host=tables)

    long_row, mixed = plan([32001], [1]), plan([32001, 8192], [1, 8192])
    assert long_row.max_pieces > 32 and mixed.max_pieces > 32
    assert mlb.ops.wide_reduction(long_row) and not mlb.ops.wide_reduction(mixed)
    assert mlb.ops.wide_reduction(plan([131072] * 4, [1] * 4))
    assert not mlb.ops.wide_reduction(plan([700] * 64, [1] * 64))


def test_error_words_are_checked(mlb):
    """Kernels write through the pointer: a tensor of another device or type must not get that far."""
    word = mlb.ops._err_adr
    assert word(None, 0, "x") == 0
    good = torch.zeros(1, dtype=torch.int32)
    assert word(good, -1, "x") == good.data_ptr()  # -1: the ordinal of CPU tensors
    for bad, dev in ((good, 0), (good.long(), -1), (good.float(), -1), (good[:0], -1)):
        with pytest.raises(ValueError, match="x: err"):
            word(bad, dev, "x")
