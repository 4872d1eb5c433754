"""The 4-bit cache's operators on the GPU against their definitions in 64 bits (oracle/fp4_ref.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import cases
from oracle import fp4_ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def pool(nb, hkv, dh, fill=0):
    return torch.full((nb, hkv, 17, dh // 2), fill, dtype=torch.uint8)


def special_rows(n, hkv, dh, dtype, seed=0):
    """Rows over the format's range: normal ones of many magnitudes, all-zero runs, exact borders between levels and
    between scales, infinities, NaN, values past the ends of the range, negative zero."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, hkv, dh, generator=g) * torch.exp2(torch.randint(-24, 18, (n, hkv, 1), generator=g).float())
    flat = x.view(-1, 32)
    flat[0] = 0.0
    flat[1] = -0.0
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for i, s in enumerate((1.0, 1.125, 2.0**-14, 2.0**-17, 10240.0, 1.875)):
        flat[2 + i] = (border * s).repeat(4) * torch.tensor([1.0, -1.0]).repeat(16)
    flat[8, 3], flat[8, 4], flat[9, 0] = math.inf, -math.inf, math.nan
    flat[10] = 1e30 if dtype != torch.float16 else 65504.0
    flat[11] = 6 * 1.0625  # a quotient half way between two scales
    if dtype == torch.float32:  # quotients that lie next to a border by less than fp32 resolves
        b = (border * 1.875).repeat(4)
        flat[12] = torch.nextafter(b, torch.full_like(b, math.inf))
        flat[13] = torch.nextafter(b, torch.zeros_like(b))
        flat[12, -1] = flat[13, -1] = 6 * 1.875
    return x.to(dtype)


def strided(x, how):
    """The same rows as a contiguous tensor, a view of a fused projection, or rows off 16-byte alignment."""
    n, h, d = x.shape
    if how == "plain":
        return x
    wide = torch.empty((n, h + 2, d) if how == "fused" else (n, h, d + 3), dtype=x.dtype, device=x.device)
    view = wide[:, 1:h + 1] if how == "fused" else wide[:, :, 1:d + 1]
    return view.copy_(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dh,hkv,how", [(64, 3, "plain"), (128, 8, "fused"), (128, 1, "odd"), (256, 2, "odd"), (64, 2, "fused")])
def test_append_and_read_equal_the_definition(mlb, cuda, dtype, dh, hkv, how):
    n, nb = 37, 9
    k, v = special_rows(n, hkv, dh, dtype, 1), special_rows(n, hkv, dh, dtype, 2)
    slots = torch.randperm(nb * 16, generator=torch.Generator().manual_seed(3))[:n]
    slots[5], slots[11] = -1, nb * 16  # out of range: skipped and flagged
    kp, vp = pool(nb, hkv, dh, 0xA5), pool(nb, hkv, dh, 0x5A)
    kd, vd = kp.to(cuda), vp.to(cuda)
    fp4_ref.append(kp, slots.tolist(), k)
    fp4_ref.append(vp, slots.tolist(), v)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    mlb.kv_append_fp4(kd, vd, slots.to(cuda), strided(k.to(cuda), how), strided(v.to(cuda), how), err)
    assert int(err.item()) == 1
    for got, want in ((kd.cpu(), kp), (vd.cpu(), vp)):  # bytes of other slots included
        assert (got != want).sum().item() == 0
    good = (slots >= 0) & (slots < nb * 16)
    ask = torch.cat([slots, slots[:3]])  # some rows twice
    for out_dtype in TYPES:
        err.zero_()
        rk, rv = mlb.kv_read_fp4(kd, vd, ask.to(cuda), out_dtype, err)
        assert int(err.item()) == 1
        for got, p in ((rk, kp), (rv, vp)):
            want = fp4_ref.values(p).view(-1, hkv, dh)[ask.clamp(0, nb * 16 - 1)]
            want[~torch.cat([good, good[:3]])] = 0
            assert torch.equal(got.cpu().double(), want)


def test_append_of_no_rows_and_of_one(mlb, cuda):
    kd, vd = pool(2, 2, 64).to(cuda), pool(2, 2, 64).to(cuda)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    slots = torch.empty(0, dtype=torch.long, device=cuda)
    mlb.kv_append_fp4(kd, vd, slots, none, none)
    assert mlb.kv_read_fp4(kd, vd, slots)[0].shape == (0, 2, 64)
    assert not kd.any() and not vd.any()
    x = torch.randn(1, 2, 64, device=cuda)
    mlb.kv_append_fp4(kd, vd, torch.tensor([31], device=cuda), x, x)
    want = pool(2, 2, 64)
    fp4_ref.append(want, [31], x.cpu())
    assert torch.equal(kd.cpu(), want) and torch.equal(vd.cpu(), want)


# ---------------------------------------------------------------- norm and rotation


def rope_inputs(n, h, hkv, dh, rot, dtype, norm, seed=0, far=100000):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(n, h, dh, generator=g).to(dtype), (3 * torch.randn(n, hkv, dh, generator=g)).to(dtype)
    pos = torch.randint(0, far, (n,), generator=g)
    w = [(1 + 0.3 * torch.randn(dh, generator=g)).to(dtype) if on else None for on in norm]
    return q, k, pos, w


def check_rope(got, x, w, pos, table, eps):
    """fp32 roundings: the sum of squares (16 terms a lane, then halvings: at most 21 additions, halved by the root), the
    reciprocal root (2 units) and three products are at most 19 * 2^-24; the rotation adds 3 * 2^-24 of |a| + |b|.
    Then half a step of the output type (and a subnormal's)."""
    want, mag = fp4_ref.norm_rope(x, w, pos, table.cpu(), eps)
    fine = 22 * 2.0**-24 * mag
    info = torch.finfo(got.dtype)
    tol = fine + info.eps / 2 * (want.abs() + fine) + info.tiny * info.eps
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,h,hkv,dh,rot,norm,how", [
    (1, 32, 8, 128, 128, (True, True), "plain"), (67, 28, 4, 128, 128, (True, True), "fused"),
    (5, 7, 1, 64, 64, (False, False), "odd"), (33, 6, 2, 256, 128, (True, False), "fused"),
    (9, 8, 8, 64, 16, (False, True), "odd"), (13, 3, 5, 256, 256, (True, True), "plain"),
    (4, 4, 2, 128, 0, (True, True), "plain"), (700, 16, 2, 128, 64, (True, True), "fused"),
    (3, 0, 2, 64, 64, (False, True), "plain"), (3, 2, 0, 64, 64, (True, False), "plain")])
def test_norm_rope(mlb, cuda, dtype, n, h, hkv, dh, rot, norm, how):
    q, k, pos, (wq, wk) = rope_inputs(n, h, hkv, dh, rot, dtype, norm)
    table = mlb.rotary_table(100000, rot, device=cuda) if rot else torch.empty(100000, 0, device=cuda)
    on = [None if w is None else w.to(cuda) for w in (wq, wk)]
    qd, kd = strided(q.to(cuda), how), strided(k.to(cuda), how)
    qo, ko = mlb.qk_norm_rope(qd, kd, pos.to(cuda), table, *on, eps=1e-5)
    assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        check_rope(got, x, w, pos, table, 1e-5)
    mlb.qk_norm_rope(qd, kd, pos.to(cuda), table, *on, eps=1e-5, out=(qd, kd))  # in place
    assert torch.equal(qd, qo) and torch.equal(kd, ko)


def test_norm_rope_leaves_rows_of_bad_positions(mlb, cuda):
    q, k, pos, w = rope_inputs(6, 4, 2, 64, 64, torch.bfloat16, (True, True), far=50)
    pos[1], pos[4] = 50, -1
    table = mlb.rotary_table(50, 64, device=cuda)
    out = (torch.full_like(q, 7.0).to(cuda), torch.full_like(k, 7.0).to(cuda))
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    args = (q.to(cuda), k.to(cuda), pos.to(cuda), table, w[0].to(cuda), w[1].to(cuda))
    qo, ko = mlb.qk_norm_rope(*args, out=out, err=err)
    assert int(err.item()) == 16
    ok = [0, 2, 3, 5]
    assert (qo[[1, 4]] == 7).all() and (ko[[1, 4]] == 7).all()
    check_rope(qo[ok], q[ok], w[0], pos[ok], table, 1e-6)
    check_rope(ko[ok], k[ok], w[1], pos[ok], table, 1e-6)


def test_rotary_table_at_far_positions(mlb, cuda):
    t = mlb.rotary_table(1 << 17, 128, device=cuda).cpu().double()
    inv = 500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    p = torch.tensor([0, 1, 777, (1 << 17) - 1])
    ang = p.double()[:, None] * inv
    want = torch.cat([ang.cos(), ang.sin()], dim=1)
    assert ((t[p] - want).abs() <= 2.0**-24).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,h,hkv,dh,norm,how", [
    (1, 32, 8, 128, (True, True), "fused"), (50, 28, 4, 128, (True, False), "fused"), (21, 7, 1, 64, (False, False), "odd"),
    (17, 6, 3, 256, (True, True), "plain"), (9, 5, 3, 64, (False, True), "plain"), (500, 8, 8, 128, (False, False), "odd")])
def test_norm_rope_append_equals_the_two_calls(mlb, cuda, dtype, n, h, hkv, dh, norm, how):
    q, k, pos, w = rope_inputs(n, h, hkv, dh, dh, dtype, norm, seed=4, far=3000)
    v = special_rows(max(n, 8), hkv, dh, dtype, 5)[:n]
    nb = n // 16 + 4
    slots = torch.randperm(nb * 16, generator=torch.Generator().manual_seed(6))[:n]
    if n > 8:
        slots[3], pos[7] = -5, 3000
    table = mlb.rotary_table(3000, dh, device=cuda)
    on = [None if x is None else x.to(cuda) for x in w]
    qd, kd, vd = (strided(x.to(cuda), how) for x in (q, k, v))
    pools = [pool(nb, hkv, dh, 0x33).to(cuda) for _ in range(4)]
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 7.0).to(cuda)
    mlb.qk_norm_rope_append_fp4(qd, kd, vd, pos.to(cuda), table, pools[0], pools[1], slots.to(cuda), *on, out=out, err=err)
    assert int(err.item()) == (17 if n > 8 else 0)
    qo, ko = mlb.qk_norm_rope(qd, kd, pos.to(cuda), table, *on,
                              out=(torch.full_like(q, 7.0).to(cuda), torch.full_like(k, 7.0).to(cuda)))
    two = slots.clone()
    if n > 8:
        two[7] = -1  # a row without a position is not stored
    mlb.kv_append_fp4(pools[2], pools[3], two.to(cuda), ko, vd)
    assert torch.equal(out, qo)
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


# ---------------------------------------------------------------- attention


class Step:
    """A seeded step on 4-bit pools: every slot that no row owns (and every slot past a row's end) holds bytes whose
    scale reads as NaN, so a value that should not be seen shows."""

    def __init__(self, mlb, cuda, h, hkv, dh, steps, dtype, seed=0, shared=0, nb=None, q_scale=1.0, first=0, how="plain"):
        g = torch.Generator().manual_seed(seed)
        r = np.random.default_rng(seed)
        need = [-(-(c + n) // 16) for c, n in steps]
        nb = nb or sum(need) + 5
        ids = (first + r.permutation(nb - first)).tolist()
        prefix = [ids.pop() for _ in range(shared)]
        self.seqs = [(c, n, prefix[:m] + [ids.pop() for _ in range(m - min(m, shared))]) for (c, n), m in zip(steps, need)]
        self.h, self.hkv, self.dh, self.dtype = h, hkv, dh, dtype
        n = sum(x for _, x in steps)
        self.q = (torch.randn(n, h, dh, generator=g) * q_scale).to(dtype)
        self.q_dev = strided(self.q.to(cuda), how)
        self.k_pool, self.v_pool = (torch.full((nb, hkv, 17, dh // 2), 0xFF, dtype=torch.uint8, device=cuda) for _ in range(2))
        owned = sorted({b * 16 + p % 16 for c, m, blk in self.seqs for p in range(c + m) for b in [blk[p // 16]]})
        slots = torch.tensor(owned, device=cuda)
        rows = [(torch.randn(len(owned), hkv, dh, generator=g) * s).to(dtype).to(cuda) for s in (1.0, 0.5)]
        mlb.kv_append_fp4(self.k_pool, self.v_pool, slots, *rows)
        self.meta = mlb.AttentionMetadata.build([mlb.SeqStep(*s) for s in self.seqs], 16, cuda)

    def plan(self, mlb, cuda, tables=True, pages=0):
        return mlb.plan_attention(self.meta.query_start_loc, self.meta.seq_lens, self.meta.block_tables_i32.shape[1], self.h,
                                  self.hkv, cuda, pages_per_unit=pages, pool_dtype=torch.uint8,
                                  block_tables_host=self.meta.block_tables_host if tables else None)

    def run(self, mlb, cuda, tables=True, pages=0, **kw):
        m = self.meta
        return mlb.paged_attention_fp4(self.q_dev, self.k_pool, self.v_pool, m.block_tables_i32, m.seq_lens_i32, m.qo_indptr,
                                       self.plan(mlb, cuda, tables, pages), **kw)

    def check(self, got, scale=None):
        want, bound = fp4_ref.attention(self.q, fp4_ref.values(self.k_pool), fp4_ref.values(self.v_pool), self.seqs, scale)
        info = torch.finfo(self.dtype)
        tol = bound + info.eps / 2 * (want.abs() + bound) + info.tiny * info.eps
        off = (got.cpu().double() - want).abs()
        assert (off <= tol).all(), f"worst |diff| / bound {(off / tol).max().item():.3g}, |diff| {off.max().item():.3g}"


HEADS = [(8, 2, 64), (32, 8, 128), (28, 4, 128), (4, 4, 64), (8, 1, 128), (6, 2, 256), (5, 1, 64)]
ROWS = {"decode": [(c - 1, 1) for c in (1, 2, 15, 16, 17, 31, 33, 255, 256, 257, 700)],
        "mixed": cases.MIXED_STEPS,
        "prefill": [(0, 130), (37, 16), (0, 1), (250, 70), (5, 15), (16, 0), (3, 2)]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
def test_attention(mlb, cuda, heads, rows, dtype):
    st = Step(mlb, cuda, *heads, ROWS[rows], dtype, how="plain" if heads[0] % 2 else "fused")
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = mlb.Workspace()
    for tables, pages in ((True, 0), (False, 0), (False, 3)):  # query tiles, whole rows, rows cut into pieces
        st.check(st.run(mlb, cuda, tables, pages, workspace=ws, err=err))
    assert int(err.item()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(32, 8, 128), (8, 2, 64), (8, 1, 128), (4, 4, 64)], ids=lambda h: "x".join(map(str, h)))
def test_attention_of_long_chunks(mlb, cuda, heads, dtype):
    """Query tiles over many key tiles (the rings of the tensor-core kernel turn over), whole and cut into pieces, odd
    numbers of tiles, beside decode rows."""
    st = Step(mlb, cuda, *heads, [(1500, 300), (0, 513), (2100, 17), (900, 1), (3000, 40)], dtype)
    st.check(st.run(mlb, cuda))
    st.check(st.run(mlb, cuda, pages=7))


@pytest.mark.parametrize("heads", [(32, 8, 128), (8, 2, 64), (8, 8, 128), (6, 2, 256)], ids=lambda h: "x".join(map(str, h)))
def test_attention_behind_a_shared_prefix(mlb, cuda, heads):
    steps = [(30 * 16 + 3 * i, 1) for i in range(40)] + [(30 * 16, 20)]
    for how in ("plain", "odd"):  # odd: query rows off 16-byte alignment
        st = Step(mlb, cuda, *heads, steps, torch.bfloat16, shared=30, how=how)
        assert st.plan(mlb, cuda).num_shared_units > 0
        st.check(st.run(mlb, cuda))


def test_attention_with_sharp_scores_and_scale(mlb, cuda):
    """Scores of several hundred: the maximum moves late, early keys weigh nothing; and a scale of the caller's."""
    st = Step(mlb, cuda, 32, 8, 128, [(900, 1), (40, 33), (2000, 1)], torch.float16, q_scale=30.0)
    st.check(st.run(mlb, cuda))
    st.check(st.run(mlb, cuda, scale=0.5), scale=0.5)


@pytest.mark.parametrize("size", [2.0**-130, 1e-30, 1e20])
def test_attention_of_queries_far_from_one(mlb, cuda, size):
    st = Step(mlb, cuda, 8, 2, 128, [(100, 1), (64, 20)], torch.bfloat16, q_scale=size)
    scale = min(1.0 / size, 3e37) / 4
    st.check(st.run(mlb, cuda, scale=scale), scale=np.float32(scale).item())


def test_attention_zero_and_nan_queries_stay_in_their_rows(mlb, cuda):
    st = Step(mlb, cuda, 8, 2, 64, [(70, 1), (200, 1), (9, 20)], torch.bfloat16)
    st.q[0] = 0.0
    st.q_dev.copy_(st.q)
    st.check(st.run(mlb, cuda))  # a zero query weighs every key alike
    ref = st.run(mlb, cuda)
    st.q_dev[1, 3, 5] = float("nan")
    for pages in (0, 2):
        got = st.run(mlb, cuda, pages=pages, tables=pages == 0)
        assert got[1, 3].isnan().all()
        st.q_dev[1, 3] = 0
        want = st.run(mlb, cuda, pages=pages, tables=pages == 0)
        st.q_dev[1, 3, 5] = float("nan")
        got[1, 3] = want[1, 3]
        assert torch.equal(got, want)
    assert torch.equal(ref[2:], st.run(mlb, cuda)[2:])
    st.q_dev[7, 0, 9] = float("nan")  # a row of a query tile
    got = st.run(mlb, cuda)
    assert got[7, 0].isnan().all() and got[7, 1:].isfinite().all() and torch.equal(got[8:], ref[8:])


def test_refusals(mlb, cuda):
    """What the GPU calls refuse: types, shapes, devices and strides they are not built for."""
    st = Step(mlb, cuda, 8, 2, 64, [(20, 1), (3, 18)], torch.bfloat16)
    m, plan, kp, vp, q = st.meta, st.plan(mlb, cuda), st.k_pool, st.v_pool, st.q_dev
    good = dict(q=q, k_cache=kp, v_cache=vp, block_tables=m.block_tables_i32, seq_lens=m.seq_lens_i32,
                qo_indptr=m.qo_indptr, plan=plan)
    other = mlb.plan_attention([0, 19], [40], 3, 8, 2, cuda, pool_dtype=torch.uint8)  # as many tokens, another batch
    for bad in (dict(q=q.float()), dict(q=q[:, :, :32]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(q=q[:18]),
                dict(q=q.cpu()), dict(k_cache=kp.to(torch.int16)), dict(k_cache=kp[:, :, :16]), dict(v_cache=vp[:5]),
                dict(v_cache=vp.cpu()), dict(block_tables=m.block_tables), dict(block_tables=m.block_tables_i32[:, :1]),
                dict(seq_lens=m.seq_lens_i32.cpu()), dict(plan=other), dict(out=torch.empty_like(q)[:18]),
                dict(out=torch.empty_like(q, dtype=torch.float16)), dict(scale=0.0), dict(scale=-1.0)):
        with pytest.raises(ValueError):
            mlb.paged_attention_fp4(**{**good, **bad})
    k, slots = torch.zeros(3, 2, 64, device=cuda), torch.arange(3, device=cuda)
    for bad in (dict(k=k.to(torch.int32)), dict(k=k[:, :1]), dict(v=k[:2]), dict(v=k.half()), dict(slot_mapping=slots.int()),
                dict(slot_mapping=slots[:2]), dict(slot_mapping=slots.cpu()), dict(k=k.cpu()), dict(k_cache=kp[::2]),
                dict(k=k.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            mlb.kv_append_fp4(**{**dict(k_cache=kp, v_cache=vp, slot_mapping=slots, k=k, v=k), **bad})
    for bad in (dict(slot_mapping=slots[None]), dict(dtype=torch.int8), dict(slot_mapping=slots.float())):
        with pytest.raises(ValueError):
            mlb.kv_read_fp4(**{**dict(k_cache=kp, v_cache=vp, slot_mapping=slots), **bad})
    table, w = torch.zeros(9, 64, device=cuda), torch.ones(64, device=cuda)
    for bad in (dict(q=k.half()), dict(q=k[:2]), dict(q=k[:, :, :32]), dict(positions=slots.int()), dict(positions=slots[:2]),
                dict(cos_sin=table.half()), dict(cos_sin=table[:, :40]), dict(cos_sin=table[:, ::2]), dict(q_weight=w[:32]),
                dict(k_weight=w.half()), dict(k_weight=w.cpu()), dict(eps=-1.0), dict(out=(k[:2], k)),
                dict(out=(k.half(), k)), dict(out=(k[:1].expand(3, 2, 64), k)), dict(cos_sin=torch.zeros(9, 24, device=cuda))):
        with pytest.raises(ValueError):
            mlb.qk_norm_rope(**{**dict(q=k, k=k, positions=slots, cos_sin=table), **bad})
    ok = dict(q=k, k=k, v=k, positions=slots, cos_sin=table, k_cache=kp, v_cache=vp, slot_mapping=slots)
    for bad in (dict(v=k[:2]), dict(v=k.half()), dict(slot_mapping=slots[:2]), dict(cos_sin=table[:, :32].contiguous()),
                dict(k=k[:, :1], v=k[:, :1]), dict(out=k[:2])):
        with pytest.raises(ValueError):
            mlb.qk_norm_rope_append_fp4(**{**ok, **bad})
    with pytest.raises(ValueError, match="block size"):
        mlb.get_backend("b200").forward(q, k, k, kp, vp, mlb.AttentionMetadata.build([mlb.SeqStep(0, 19, [0])], 32, cuda))


@pytest.mark.parametrize("tables", [True, False])
def test_attention_skips_pages_of_bad_block_ids(mlb, cuda, tables):
    st = Step(mlb, cuda, 32, 8, 128, [(100, 1), (150, 40)], torch.bfloat16)
    bad = st.meta.block_tables_i32.clone()
    bad[0, 2], bad[1, 4], bad[1, 0] = st.k_pool.shape[0], -7, 1 << 30
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    m = st.meta
    got = mlb.paged_attention_fp4(st.q_dev, st.k_pool, st.v_pool, bad, m.seq_lens_i32, m.qo_indptr,
                                  st.plan(mlb, cuda, tables), err=err)
    assert int(err.item()) == 2
    # the pages count as empty: the same rows in 64 bits without their keys
    kv, vv = fp4_ref.values(st.k_pool), fp4_ref.values(st.v_pool)
    at = 0
    for (c, n, ids), holes in zip(st.seqs, ((2,), (0, 4))):
        for i in range(n):
            seen = torch.tensor([p for p in range(c + i + 1) if p // 16 not in holes])
            blk = torch.tensor(ids)[seen // 16]
            k, v = (x[blk, seen % 16].repeat_interleave(4, dim=1) for x in (kv, vv))
            p = torch.softmax(torch.einsum("hd,lhd->hl", st.q[at].double(), k) / math.sqrt(128), dim=-1)
            want = torch.einsum("hl,lhd->hd", p, v)
            # bf16 output (2^-8 relative, of |o| <= max|v| < 2) beside 2^-11 of P
            assert ((got[at].cpu().double() - want).abs() <= 2.0**-9 * 2 + 2.0**-9 * want.abs()).all()
            at += 1


def test_attention_in_a_pool_past_32_bit_offsets(mlb, cuda):
    """Blocks whose records lie more than 2^32 bytes into the pool."""
    nb = (1 << 32) // (8 * 17 * 64) + 4000
    st = Step(mlb, cuda, 32, 8, 128, [(600, 1), (1000, 30)], torch.bfloat16, nb=nb, first=nb - 300)
    st.k_pool_small = st.k_pool[nb - 300:].clone()
    seqs = [(c, n, [b - (nb - 300) for b in ids]) for c, n, ids in st.seqs]
    got = st.run(mlb, cuda)
    want, bound = fp4_ref.attention(st.q, fp4_ref.values(st.k_pool[nb - 300:]), fp4_ref.values(st.v_pool[nb - 300:]), seqs)
    tol = bound + 2.0**-8 * (want.abs() + bound)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_attention_leaves_rows_behind_the_last_sequence_and_other_columns(mlb, cuda):
    st = Step(mlb, cuda, 8, 2, 64, [(20, 1), (3, 18)], torch.bfloat16)
    wide = torch.full((19, 10, 64), 5.0, dtype=torch.bfloat16, device=cuda)
    out = wide[:, 1:9]
    st.run(mlb, cuda, out=out)
    st.check(out)
    assert (wide[:, 0] == 5).all() and (wide[:, 9] == 5).all()


def test_attention_is_deterministic_and_captures(mlb, cuda):
    st = Step(mlb, cuda, 32, 8, 128, [(3000, 1), (500, 1), (0, 40)] + [(600 + i, 1) for i in range(6)], torch.float16)
    ws, m = mlb.Workspace(), st.meta
    plan = st.plan(mlb, cuda)
    run = lambda: mlb.paged_attention_fp4(st.q_dev, st.k_pool, st.v_pool, m.block_tables_i32, m.seq_lens_i32,  # noqa: E731
                                          m.qo_indptr, plan, ws)
    ref = run()
    assert torch.equal(ref, run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ref, other)
    graphs, outs = [], []
    for _ in range(2):  # two graphs over one workspace, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for g in (*graphs, *graphs):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], ref) and torch.equal(outs[1], ref)
    st.q_dev.copy_(torch.flip(st.q_dev, [0]))
    want = run()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)


def test_a_grown_workspace_leaves_a_captured_graph_its_buffer(mlb, cuda):
    st = Step(mlb, cuda, 8, 2, 128, [(3000, 1), (500, 1)], torch.float16)
    ws, m = mlb.Workspace(), st.meta
    plan = st.plan(mlb, cuda)
    assert plan.num_partial_rows
    run = lambda: mlb.paged_attention_fp4(st.q_dev, st.k_pool, st.v_pool, m.block_tables_i32, m.seq_lens_i32,  # noqa: E731
                                          m.qo_indptr, plan, ws)
    ref = run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    rows = plan.num_partial_rows
    ws.get(100 * rows, 8, 128, ref.device)
    others = [torch.full((rows * 8 * 128,), float("nan"), device=cuda) for _ in range(8)]  # would take a freed buffer
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref) and all(x.isnan().all() for x in others)


@pytest.mark.parametrize("steps,shared", [([(3000, 1), (500, 1), (0, 40), (37, 16), (9, 3)], 0), ([(300 + i, 1) for i in range(9)], 16)])
def test_attention_into_targets(mlb, cuda, steps, shared):
    """Rows for several destinations, among other heads' rows, as KV-head sharding stores them."""
    st = Step(mlb, cuda, 32, 8, 128, steps, torch.bfloat16, shared=shared)
    ref, n = st.run(mlb, cuda), len(st.q)
    bufs = [torch.full((n, 40, 128), float("nan"), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    to = mlb.ops.out_targets([b.data_ptr() for b in bufs], 5, 40 * 128, 128)
    assert st.run(mlb, cuda, targets=to) is None
    for b in bufs:
        assert torch.equal(b[:, 5:37], ref) and b[:, :5].isnan().all() and b[:, 37:].isnan().all()


@pytest.mark.parametrize("exchange", ["packets", "barrier"])
def test_backend_gathers_rows_of_a_4bit_cache(mlb, cuda, exchange):
    """One rank of KV-head sharding's own transport (no peer to wait for): the rows of a plain forward."""
    import torch.distributed as dist

    sharding = __import__(mlb.__name__ + ".sharding", fromlist=["PeerOutputs"])
    own_group = not dist.is_initialized()
    if own_group:
        dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        st = Step(mlb, cuda, 32, 8, 128, [(700, 1), (300, 1), (10, 40), (37, 5)], torch.bfloat16)
        n, g = len(st.q), torch.Generator().manual_seed(4)
        k, v = (torch.randn(n, 8, 128, generator=g).to(torch.bfloat16).to(cuda) for _ in range(2))
        backend = mlb.get_backend("b200", check_errors=True, pages_per_unit=16)
        pools = [(st.k_pool.clone(), st.v_pool.clone()) for _ in range(2)]
        ref = backend.forward(st.q_dev, k, v, *pools[0], st.meta)
        plan = backend.plan(st.meta, 32, 8, st.q_dev.device, torch.uint8)
        assert 1 < plan.max_pieces <= mlb.ops.WIDE_REDUCE_PIECES  # one reduction's order of sums on both sides
        peers = sharding.PeerOutputs(n + 3, 32, 128, torch.bfloat16, cuda, slots=2, exchange=exchange)
        for slot in (0, 1):
            peers.output(slot, n).fill_(float("nan"))
            assert backend.forward(st.q_dev, k, v, *pools[1], st.meta, peer_gather=(peers, slot, 0)) is None
            assert torch.equal(peers.output(slot, n), ref)
        assert torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
        peers.raise_errors()
        peers.close()
    finally:
        if own_group:
            dist.destroy_process_group()


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rot", [128, 64])
def test_backend_step_on_a_4bit_cache(mlb, cuda, dtype, rot):
    """Two steps of one layer through the backend: norm and rotation, append, attention; a block copied before the
    second step writes it."""
    shape = mlb.KVShape(2, 2, 128)
    cache = mlb.PagedKVCacheFP4(shape, 40, cuda)
    bm = mlb.BlockManager(40, 16)
    backend = mlb.get_backend("b200", check_errors=True)
    table = mlb.rotary_table(512, rot, device=cuda)
    g = torch.Generator().manual_seed(9)
    w = [(1 + 0.2 * torch.randn(128, generator=g)).to(dtype) for _ in range(2)]
    rotary = mlb.Rotary(table, w[0].to(cuda), w[1].to(cuda), eps=1e-5)
    kv = [torch.zeros(40, 2, 17, 64, dtype=torch.uint8) for _ in range(2)]
    blocks = [bm.allocate(5), bm.allocate(2)]
    for cached, new in (([0, 0], [70, 20]), ([70, 20], [1, 3])):
        if cached[0]:  # row 0's last block is shared with another table: the step's write goes to a copy
            bm.acquire([blocks[0][4]])
            pairs = bm.cow_for_append(blocks[0], 70, 1)
            cache.copy_blocks([a for a, _ in pairs], [b for _, b in pairs])
            for p in kv:
                for a, b in pairs:
                    p[b] = p[a]
        meta = mlb.AttentionMetadata.build([mlb.SeqStep(c, n, list(b)) for c, n, b in zip(cached, new, blocks)], 16, cuda)
        n = sum(new)
        qkv = torch.randn(n, 12, 128, generator=g).to(dtype)
        dev = qkv.to(cuda)
        out = backend.forward(dev[:, :8], dev[:, 8:10], dev[:, 10:], cache.k[1], cache.v[1], meta, rotary=rotary)
        pos, slots = meta.positions.cpu(), meta.slot_mapping.cpu().tolist()
        qo, ko = mlb.qk_norm_rope(dev[:, :8], dev[:, 8:10], meta.positions, table, rotary.q_weight, rotary.k_weight, 1e-5)
        check_rope(qo, qkv[:, :8], w[0], pos, table, 1e-5)
        check_rope(ko, qkv[:, 8:10], w[1], pos, table, 1e-5)
        for p, x in ((kv[0], ko.cpu()), (kv[1], qkv[:, 10:])):
            fp4_ref.append(p, slots, x)
        assert torch.equal(cache.k[1].cpu(), kv[0]) and torch.equal(cache.v[1].cpu(), kv[1])
        want, bound = fp4_ref.attention(qo.cpu(), fp4_ref.values(kv[0]), fp4_ref.values(kv[1]),
                                        [(c, m, list(b)) for c, m, b in zip(cached, new, blocks)])
        tol = bound + torch.finfo(dtype).eps / 2 * (want.abs() + bound)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        rk, rv = cache.read(1, meta.slot_mapping, dtype)
        assert torch.equal(rk.cpu().double(), fp4_ref.values(kv[0]).view(-1, 2, 128)[meta.slot_mapping.cpu()])
        assert torch.equal(rv.cpu().double(), fp4_ref.values(kv[1]).view(-1, 2, 128)[meta.slot_mapping.cpu()])
    assert not cache.k[0].any()  # the other layer's pool is untouched


def test_backend_rotary_on_16bit_pools(mlb, cuda):
    """`rotary` in front of the 16-bit path: the same as rotating first."""
    case = cases.mixed_step(4, 32, 8, 128)
    backend = mlb.get_backend("b200")
    meta = mlb.AttentionMetadata.build([mlb.SeqStep(c, n, list(b)) for c, n, b in case.seqs], 16, cuda)
    q, k, v, kp, vp = (getattr(case, x).to(torch.bfloat16).to(cuda) for x in ("q", "k", "v", "k_pool", "v_pool"))
    table = mlb.rotary_table(512, 128, device=cuda)
    pools = [(kp.clone(), vp.clone()) for _ in range(2)]
    got = backend.forward(q, k, v, *pools[0], meta, rotary=mlb.Rotary(table))
    qo, ko = mlb.qk_norm_rope(q, k, meta.positions, table)
    want = backend.forward(qo, ko, v, *pools[1], meta)
    assert torch.equal(got, want) and torch.equal(pools[0][0], pools[1][0]) and torch.equal(pools[0][1], pools[1][1])
