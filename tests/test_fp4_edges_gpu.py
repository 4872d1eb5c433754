"""The 4-bit operators where their first tests did not look: scales next to nothing, weights far below the
largest, query elements far below the row's."""

from __future__ import annotations

import math
import weakref

import pytest
import torch

from test_fp4_gpu import Step

pytestmark = pytest.mark.gpu


class Rows:
    """Rows of given keys, values and queries: key and value of position p are k[p], v[p] for every row and head.  The
    keys have to be values that the 4-bit format holds; `held` are the values that the cache has of v, by position."""

    def __init__(self, mlb, cuda, h, hkv, steps, k, v, q, dtype, how="plain"):
        dh = k.shape[1]
        need = [-(-(c + n) // 16) for c, n in steps]
        ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).tolist()
        self.seqs = [(c, n, [ids.pop() for _ in range(m)]) for (c, n), m in zip(steps, need)]
        self.pools = [torch.full((sum(need), hkv, 17, dh // 2), 0xFF, dtype=torch.uint8, device=cuda) for _ in range(2)]
        for c, n, blk in self.seqs:
            p = torch.arange(c + n)
            slots = (torch.tensor(blk)[p // 16] * 16 + p % 16).to(cuda)
            rows = [x[:c + n, None].expand(-1, hkv, -1).to(dtype).to(cuda) for x in (k, v)]
            mlb.kv_append_fp4(*self.pools, slots, *rows)
            keys, values = mlb.kv_read_fp4(*self.pools, slots, dtype)
            assert torch.equal(keys, rows[0])
            self.held = values[:, 0].cpu().double()
        n = sum(x for _, x in steps)
        wide = torch.zeros(n, h, dh + 3, dtype=dtype, device=cuda)  # "odd": rows off 16-byte alignment
        self.q = q.to(dtype).to(cuda).expand(n, h, dh).contiguous() if how == "plain" else wide[:, :, 1:dh + 1].copy_(q)
        self.meta = mlb.AttentionMetadata.build([mlb.SeqStep(*s) for s in self.seqs], 16, cuda)
        self.heads, self.seen = (h, hkv), [c + i + 1 for c, n in steps for i in range(n)]  # keys that each token sees

    def run(self, mlb, cuda, tables=True, pages=0, **kw):
        m = self.meta
        plan = mlb.plan_attention(m.query_start_loc, m.seq_lens, m.block_tables_i32.shape[1], *self.heads, cuda,
                                  pages_per_unit=pages, pool_dtype=torch.uint8,
                                  block_tables_host=m.block_tables_host if tables else None)
        return mlb.paged_attention_fp4(self.q, *self.pools, m.block_tables_i32, m.seq_lens_i32, m.qo_indptr, plan, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e-9, 1e-30, 1e-38])
def test_zero_queries_under_a_tiny_scale(mlb, cuda, dtype, scale):
    """Keys past a row's end stay masked however small the scale is: every key that is seen weighs the same."""
    for how in ("plain", "odd"):
        st = Step(mlb, cuda, 8, 2, 64, [(70, 1), (200, 1), (9, 20), (0, 1)], dtype, how=how)
        st.q[::2] = 0.0
        st.q_dev.copy_(st.q)
        for tables, pages in ((True, 0), (False, 0), (False, 2)):
            st.check(st.run(mlb, cuda, tables, pages, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tables,how", [(True, "plain"), (True, "odd"), (False, "plain")])
def test_a_long_tail_keeps_its_weight(mlb, cuda, dtype, tables, how):
    """One key weighs e^18 times each of the 40000 others; its value is 0, theirs 6, so what comes out is the others'
    weight.  A weight is 2^-25.97 of the largest: rounded on a grid of 2^-34 (fp16 at 2^10 times the weight) it is off
    by at most 2^-35 / 2^-25.97 = 2^-9.03; fp32 sums of 2500 pages and the merge, 2^-23 an addition, twice: 2^-10.7;
    the exponent's argument, 26 with 2 roundings of 2^-24, times ln 2 and twice: 2^-18; then the output's rounding."""
    length, dh = 40040, 64
    k, v = torch.zeros(length, dh), torch.full((length, dh), 6.0)
    k[0, 0], v[0] = 18.0, 0.0
    q = torch.zeros(dh)
    q[0] = 1.0
    st = Rows(mlb, cuda, 4, 1, [(40000, 1), (40000, 20)], k, v, q, dtype, how)
    rel = 2.0**-9.03 + 2.0**-10.7 + 2.0**-18 + torch.finfo(dtype).eps / 2
    assert torch.equal(st.held, v[:len(st.held)].double())
    for pages in (1 << 20, 0):
        got = st.run(mlb, cuda, tables, pages, scale=1.0).cpu().double()
        tail = (torch.tensor(st.seen, dtype=torch.float64) - 1) * math.exp(-18)
        want = (6 * tail / (1 + tail))[:, None, None]
        assert ((got - want).abs() <= rel * want).all(), ((got - want).abs() / want).max().item()


@pytest.mark.parametrize("tables,how", [(True, "plain"), (True, "odd"), (False, "plain")])
def test_a_small_query_element_meets_a_large_key(mlb, cuda, tables, how):
    """A bf16 query of 2048 and 1.5 * 2^-14, keys of 0 and 61440: the score is the small element's alone, 0.70.  Its one
    product is exact, the exponent's argument has 2 roundings of 2^-24; a weight is rounded to 2^-11, twice."""
    k, v = torch.zeros(120, 64), torch.zeros(120, 64)
    k[::2, 1], v[::2] = 61440.0, 1.0
    q = torch.zeros(64)
    q[0], q[1] = 2048.0, 1.5 * 2.0**-14
    st = Rows(mlb, cuda, 4, 1, [(50, 1), (100, 20)], k, v, q, torch.bfloat16, how)
    got = st.run(mlb, cuda, tables).cpu().double()
    seen = torch.tensor(st.seen, dtype=torch.float64)
    top = torch.ceil(seen / 2) * math.exp(1.5 * 2.0**-14 * 61440 / 8)
    want = (top / (top + torch.floor(seen / 2)))[:, None, None] * st.held[0]
    assert ((got - want).abs() <= (2.0**-8 + 2.0**-10) * want).all(), ((got - want).abs() / want).max().item()


def test_workspace_keeps_only_what_a_graph_holds(mlb, cuda):
    """Large buffers (above Workspace.SMALL_BYTES): dropped when outgrown, kept when a capture was given them."""
    ws, dev = mlb.Workspace(), torch.zeros(1, device=cuda).device
    rows = 1 << 13
    first = [weakref.ref(t) for t in ws.get(rows, 8, 128, dev)]
    assert 4 * first[0]().numel() > mlb.Workspace.SMALL_BYTES
    second = [weakref.ref(t) for t in ws.get(rows + 1, 8, 128, dev)]
    assert all(r() is None for r in first)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ws.get(rows, 8, 128, dev)[0].fill_(1.0)
    third = [weakref.ref(t) for t in ws.get(rows + 2, 8, 128, dev)]
    assert all(r() is not None for r in second) and third[0]().numel() == 3 * (rows + 1) * 8 * 128 // 2
    g.replay()
    torch.cuda.synchronize()
    assert (second[0]() == 1).all()
    del g
    ws.get(2 * rows, 8, 128, dev)
    assert all(r() is None for r in third)
    ws.release()
    assert all(r() is None for r in second)


def test_an_outgrown_buffer_waits_for_the_stream_that_uses_it(mlb, cuda):
    """Scratch of one stream, used on another and outgrown there: its memory is not given out before that stream is
    done with it."""
    ws, dev = mlb.Workspace(), torch.zeros(1, device=cuda).device
    rows = 1 << 13
    home = ws.get(rows, 8, 128, dev)[0].data_ptr()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = ws.get(rows, 8, 128, dev)[0]
        torch.cuda._sleep(50_000_000)  # some tens of milliseconds
        o.fill_(1.0)
        del o
        ws.get(4 * rows, 8, 128, dev)
    other = torch.full((rows * 8 * 128,), 2.0, device=cuda)  # on the home stream, which does not wait
    assert other.data_ptr() != home
    torch.cuda.synchronize()
    assert (other == 2).all()


@pytest.mark.parametrize("first", [True, False])
def test_one_long_row_beside_a_chunk(mlb, cuda, first):
    """A row of many pieces among unsplit ones: each is reduced, or left alone, for itself."""
    steps = [(9000, 1), (0, 600)] if first else [(0, 600), (9000, 1)]
    st = Step(mlb, cuda, 8, 2, 64, steps, torch.bfloat16)
    plan = st.plan(mlb, cuda)
    assert plan.max_pieces > mlb.ops.WIDE_REDUCE_PIECES and not mlb.ops.wide_reduction(plan)
    st.check(st.run(mlb, cuda))
    alone = Step(mlb, cuda, 8, 2, 64, [(9000, 1)], torch.bfloat16)
    assert mlb.ops.wide_reduction(alone.plan(mlb, cuda))
    alone.check(alone.run(mlb, cuda))


def test_error_words_of_another_device_or_type_are_refused(mlb, cuda):
    st = Step(mlb, cuda, 8, 2, 64, [(20, 1)], torch.bfloat16)
    m, pools = st.meta, (st.k_pool, st.v_pool)
    x, slots, table = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=cuda), m.slot_mapping, torch.ones(32, 64, device=cuda)
    calls = (lambda e: mlb.kv_append_fp4(*pools, slots, x, x, err=e), lambda e: mlb.kv_read_fp4(*pools, slots, err=e),
             lambda e: mlb.qk_norm_rope(x, x, m.positions, table, err=e),
             lambda e: mlb.qk_norm_rope_append_fp4(x, x, x, m.positions, table, *pools, slots, err=e),
             lambda e: st.run(mlb, cuda, err=e))
    before = [p.clone() for p in pools]
    for call in calls:
        for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=cuda),
                    torch.zeros(0, dtype=torch.int32, device=cuda)):
            with pytest.raises(ValueError, match="err must be"):
                call(bad)
    assert all(torch.equal(a, b) for a, b in zip(pools, before))
    for call in calls:
        err = torch.zeros(1, dtype=torch.int32, device=cuda)
        call(err)
        assert int(err.item()) == 0


def test_release_waits_for_streams_that_used_a_captured_buffer(mlb, cuda):
    """A large buffer that a capture was given is not followed from stream to stream: release waits for all of them,
    before the buffer in use can be outgrown and freed as any other."""
    backend, dev = mlb.get_backend("b200"), torch.zeros(1, device=cuda).device
    ws, rows = backend._workspace, 1 << 13
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ws.get(rows, 8, 128, dev)[0].fill_(0.0)
    del g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = ws.get(rows, 8, 128, dev)[0]
        torch.cuda._sleep(50_000_000)  # some tens of milliseconds
        o.fill_(1.0)
    backend.release_scratch()
    assert side.query()
