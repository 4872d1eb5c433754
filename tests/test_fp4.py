"""The 4-bit cache without a GPU: the definition the GPU tests compare with, the pool's sizes, and the refusals of the
entry points (every call here is refused, or has nothing to do, before a launch)."""

from __future__ import annotations

import re
import weakref
from importlib import import_module
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import fp4_ref


@pytest.fixture(scope="module")
def L(mlb):
    return import_module(mlb.__name__ + "._lib")


def test_definition_against_a_search_of_every_value():
    """Every (scale, code) pair spelled out: the scale is the nearest to max / 6, the code the nearest level."""
    g = np.random.default_rng(3)
    for size in (1e-7, 1e-4, 0.02, 1.0, 300.0, 2e4, 1e6):
        x = (g.standard_normal((5, 64)) * size).astype(np.float32)
        code, byte = fp4_ref.quantise(torch.from_numpy(x))
        for row in range(5):
            for run in range(2):
                v = np.clip(x[row, 32 * run:32 * run + 32].astype(np.float64), -61440, 61440)
                s = fp4_ref.SCALES[byte[row, run]]
                assert abs(np.abs(v).max() / 6 - s) == np.abs(np.abs(v).max() / 6 - fp4_ref.SCALES).min()
                c = code[row, 32 * run:32 * run + 32]
                stored = np.where(c >= 8, -1, 1) * fp4_ref.LEVELS[c % 8] * s
                every = np.concatenate([fp4_ref.LEVELS, -fp4_ref.LEVELS]) * s
                # distances to levels s apart by products, the codes chosen by quotients: equal to a rounding
                assert (np.abs(stored - v) <= np.abs(v[:, None] - every).min(1) * (1 + 1e-12)).all()


def test_definition_scale_bytes_are_float16_shifted():
    half = (np.arange(227, dtype=np.uint16) << 7).view(np.float16).astype(np.float64)
    assert np.array_equal(half, fp4_ref.SCALES)
    assert 6 * fp4_ref.SCALES[226] == 61440.0


def test_definition_append_then_values_touch_only_their_slots():
    p = torch.full((3, 2, 17, 32), 0x77, dtype=torch.uint8)
    before = fp4_ref.values(p)
    x = torch.randn(2, 2, 64)
    fp4_ref.append(p, [5, 47], x)
    after = fp4_ref.values(p).view(48, 2, 64)
    rest = [i for i in range(48) if i not in (5, 47)]
    assert torch.equal(after[rest], before.view(48, 2, 64)[rest])
    assert (after[[5, 47]] - x.double()).abs().max() <= x.abs().max() / 6  # half the widest gap between levels


def test_definition_attention_is_plain_softmax():
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(4, 16, 2, 64, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(3, 4, 64, generator=g)
    out, bound = fp4_ref.attention(q, k, v, [(20, 1, [2, 0]), (0, 2, [3])])
    kk, vv = k[[2, 0]].view(32, 2, 64)[:21, 1], v[[2, 0]].view(32, 2, 64)[:21, 1]
    p = torch.softmax(kk @ q[0, 3].double() / 8, dim=0)
    assert torch.allclose(out[0, 3], p @ vv)
    assert torch.allclose(out[1, 0], v[3, 0, 0])  # the first token of a fresh row sees itself alone
    assert (bound > 0).all() and (bound < 2.0**-9).all()


def test_pool_sizes(mlb):
    shape = mlb.KVShape(3, 8, 128)
    c = mlb.PagedKVCacheFP4(shape, 5, "cpu")
    assert c.k[2].shape == c.v[0].shape == (5, 8, 17, 64) and c.k[1].dtype == torch.uint8 and c.k[1].is_contiguous()
    per = mlb.PagedKVCacheFP4.bytes_per_block(shape)
    assert per * 5 == c.storage.numel()
    assert per / mlb.PagedKVCache.bytes_per_block(shape, torch.bfloat16) == 17 / 64
    assert mlb.PagedKVCacheFP4.blocks_for_bytes(shape, torch.uint8, 10 * per + 1) == 10
    with pytest.raises(ValueError, match="uint8"):
        mlb.PagedKVCacheFP4.bytes_per_block(shape, torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim"):
        mlb.PagedKVCacheFP4(mlb.KVShape(1, 1, 96), 5, "cpu")


def test_entry_points_refuse_tensors_of_the_cpu(mlb):
    p = torch.zeros(2, 2, 17, 32, dtype=torch.uint8)
    x, slots = torch.zeros(3, 2, 64), torch.arange(3)
    with pytest.raises(ValueError, match="CUDA"):
        mlb.kv_append_fp4(p, p, slots, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        mlb.kv_read_fp4(p, p, slots)
    with pytest.raises(ValueError, match="CUDA"):
        mlb.qk_norm_rope(x, x, slots, torch.zeros(4, 64))
    with pytest.raises(ValueError, match="CUDA"):
        mlb.qk_norm_rope_append_fp4(x, x, x, slots, torch.zeros(4, 64), p, p, slots)
    plan = mlb.plan_attention([0, 3], [3], 1, 2, 2, "cpu", pool_dtype=torch.uint8)
    i32 = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mlb.paged_attention_fp4(x.bfloat16(), p, p, i32, i32[0], i32[0], plan)


def test_backend_refuses_queries_before_it_writes(mlb):
    backend = mlb.get_backend("b200")
    meta = mlb.AttentionMetadata.build([mlb.SeqStep(0, 2, [1])], 16, "cpu")
    pools = [torch.full((3, 2, 17, 64), 7, dtype=torch.uint8) for _ in range(2)]
    k = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    for q in (torch.zeros(2, 8, 128), torch.zeros(2, 18, 128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="at most 8 heads per KV head"):
            backend.forward(q, k.to(q.dtype), k.to(q.dtype), *pools, meta)
    with pytest.raises(ValueError, match="block size"):
        backend.forward(k, k, k, *pools, mlb.AttentionMetadata.build([mlb.SeqStep(0, 2, [1])], 32, "cpu"))
    assert all((p == 7).all() for p in pools)


def test_rotary_table_refusals_and_values(mlb):
    for rows, rot in ((0, 64), (8, 0), (8, 24), (-1, 16)):
        with pytest.raises(ValueError, match="rotary_table"):
            mlb.rotary_table(rows, rot, device="cpu")
    with pytest.raises(ValueError, match="inv_freq"):
        mlb.rotary_table(4, 32, device="cpu", inv_freq=torch.ones(15))
    t = mlb.rotary_table(4, 16, device="cpu", inv_freq=torch.full((8,), 0.5))
    assert t.shape == (4, 16) and torch.allclose(t[3, :8], torch.full((8,), 1.5).cos())
    assert torch.allclose(t[3, 8:], torch.full((8,), 1.5).sin())


F = 1 << 20  # a pointer that is never followed


def test_append_and_read_refusals(L):
    lib = L.lib()
    ok = dict(kc=F, vc=F, nb=4, slots=F, k=F, v=F, dt=2, n=3, hkv=2, dh=64)

    def append(**kw):
        a = {**ok, **kw}
        return lib.mlb_kv_append_fp4(a["kc"], a["vc"], a["nb"], a["slots"], a["k"], 128, 64, a["v"], 128, 64, a["dt"], a["n"],
                                     a["hkv"], a["dh"], None, None)

    def read(**kw):
        a = {**ok, **kw}
        return lib.mlb_kv_read_fp4(a["kc"], a["vc"], a["nb"], a["slots"], a["k"], a["v"], a["dt"], a["n"], a["hkv"], a["dh"],
                                   None, None)

    for call in (append, read):
        for bad, code, word in ((dict(dt=3), L.MLB_EINVAL, "dtype"), (dict(dh=96), L.MLB_EUNSUPPORTED, "head_dim"),
                                (dict(n=-1), L.MLB_EINVAL, "sizes"), (dict(hkv=0), L.MLB_EINVAL, "sizes"),
                                (dict(nb=0), L.MLB_EINVAL, "sizes"), (dict(kc=None), L.MLB_EINVAL, "null"),
                                (dict(slots=None), L.MLB_EINVAL, "null"), (dict(v=None), L.MLB_EINVAL, "null"),
                                (dict(vc=F + 8), L.MLB_EINVAL, "aligned"), (dict(n=1 << 40), L.MLB_EINVAL, "too many rows")):
            assert call(**bad) == code and word in L.last_error(), bad
        assert call(n=0, kc=None, k=None) == L.MLB_OK
    assert read(k=F + 4) == L.MLB_EINVAL and "aligned" in L.last_error()


def test_norm_rope_refusals(L):
    lib = L.lib()
    ok = dict(q=F, k=F, dt=2, n=3, h=4, hkv=2, dh=64, pos=F, cs=F, np=10, rot=64, qw=None, kw=None, eps=1e-6, qo=F, ko=F)

    def rope(**kw):
        a = {**ok, **kw}
        return lib.mlb_qk_norm_rope(a["q"], 256, 64, a["k"], 128, 64, a["dt"], a["n"], a["h"], a["hkv"], a["dh"], a["pos"],
                                    a["cs"], a["np"], a["rot"], a["qw"], a["kw"], a["eps"], a["qo"], 256, 64, a["ko"], 128,
                                    64, None, None)

    for bad, code, word in ((dict(dt=9), L.MLB_EINVAL, "dtype"), (dict(dh=32), L.MLB_EUNSUPPORTED, "head_dim"),
                            (dict(rot=24), L.MLB_EUNSUPPORTED, "rot_dim"), (dict(rot=80), L.MLB_EUNSUPPORTED, "rot_dim"),
                            (dict(rot=-16), L.MLB_EUNSUPPORTED, "rot_dim"), (dict(eps=-1.0), L.MLB_EINVAL, "eps"),
                            (dict(eps=float("nan")), L.MLB_EINVAL, "eps"), (dict(h=0, hkv=0), L.MLB_EINVAL, "sizes"),
                            (dict(q=None), L.MLB_EINVAL, "null"), (dict(ko=None), L.MLB_EINVAL, "null"),
                            (dict(pos=None), L.MLB_EINVAL, "null"), (dict(cs=None), L.MLB_EINVAL, "null"),
                            (dict(cs=F + 4), L.MLB_EINVAL, "aligned"), (dict(kw=F + 2), L.MLB_EINVAL, "aligned"),
                            (dict(np=-1), L.MLB_EINVAL, "sizes")):
        assert rope(**bad) == code and word in L.last_error(), bad
    assert rope(n=0, q=None, pos=None) == L.MLB_OK

    def both(rot=64, nb=4, slots=F, v=F, n=3):
        return lib.mlb_qk_norm_rope_append_fp4(F, 256, 64, F, 128, 64, v, 128, 64, 2, n, 4, 2, 64, F, F, 10, rot, None, None,
                                               1e-6, F, 256, 64, F, F, nb, slots, None, None)

    for bad, code, word in ((dict(rot=32), L.MLB_EUNSUPPORTED, "whole head"), (dict(nb=0), L.MLB_EINVAL, "pool sizes"),
                            (dict(slots=None), L.MLB_EINVAL, "null"), (dict(v=None), L.MLB_EINVAL, "null")):
        assert both(**bad) == code and word in L.last_error(), bad
    assert both(n=0, slots=None) == L.MLB_OK


def test_attention_refusals(L):
    lib = L.lib()
    ok = dict(q=F, kc=F, vc=F, dt=2, nb=4, h=8, hkv=2, dh=64, scale=0.1, nu=1, units=F, ns=0, shared=None, po=None, rows=0,
              out=F)

    def attend(**kw):
        a = {**ok, **kw}
        return lib.mlb_paged_attention_fp4(a["q"], 512, 64, a["kc"], a["vc"], a["dt"], a["nb"], a["h"], a["hkv"], a["dh"],
                                           a["scale"], F, 1, F, F, 1, a["units"], a["nu"], a["shared"], a["ns"], None,
                                           a["po"], a["po"], a["rows"], a["out"], 512, 64, None, None, None)

    for bad, code, word in ((dict(dt=0), L.MLB_EUNSUPPORTED, "16-bit"), (dict(dh=192), L.MLB_EUNSUPPORTED, "head_dim"),
                            (dict(h=9), L.MLB_EINVAL, "multiple"), (dict(h=18), L.MLB_EUNSUPPORTED, "query heads"),
                            (dict(scale=0.0), L.MLB_EINVAL, "scale"), (dict(scale=-1.0), L.MLB_EINVAL, "scale"),
                            (dict(scale=float("nan")), L.MLB_EINVAL, "scale"), (dict(scale=float("inf")), L.MLB_EINVAL, "scale"),
                            (dict(nu=-1), L.MLB_EINVAL, "sizes"), (dict(nb=0), L.MLB_EINVAL, "sizes"),
                            (dict(q=None), L.MLB_EINVAL, "null"), (dict(units=None), L.MLB_EINVAL, "null"),
                            (dict(ns=2), L.MLB_EINVAL, "null"), (dict(ns=3, shared=F), L.MLB_EINVAL, "pairs"),
                            (dict(out=None), L.MLB_EINVAL, "null out"), (dict(rows=4), L.MLB_EINVAL, "workspace"),
                            (dict(kc=F + 1), L.MLB_EINVAL, "aligned"), (dict(nu=1 << 40), L.MLB_EINVAL, "grid")):
        assert attend(**bad) == code and word in L.last_error(), bad
    assert attend(nu=0, q=None) == L.MLB_OK


def test_wide_reduction_refusals(L):
    lib = L.lib()

    def reduce(po=F, n=4, h=8, dh=64, dt=2, tpt=2, out=F, rows=4):
        return lib.mlb_splitk_reduce_wide(po, F, rows, F, F, tpt, n, h, dh, out, 512, 64, dt, None, None)

    for bad, code, word in ((dict(po=None), L.MLB_EINVAL, "null"), (dict(dt=9), L.MLB_EINVAL, "dtype"),
                            (dict(dh=96), L.MLB_EUNSUPPORTED, "head_dim"), (dict(tpt=0), L.MLB_EINVAL, "sizes"),
                            (dict(n=-1), L.MLB_EINVAL, "sizes"), (dict(out=None), L.MLB_EINVAL, "null out"),
                            (dict(n=1 << 40), L.MLB_EINVAL, "grid")):
        assert reduce(**bad) == code and word in L.last_error(), bad
    assert reduce(n=0) == L.MLB_OK and reduce(rows=0) == L.MLB_OK


def test_calls_by_words(L):
    """The numbers are the header's; counts and ints are checked; the entry point behind refuses as it does directly."""
    header = (Path(__file__).parents[1] / "include" / "mlb_paged_kv.h").read_text()
    numbers = {n: int(v) for n, v in re.findall(r"MLB_CALL_(\w+) = (\d+)", header)}
    assert len(numbers) == 7 and all(getattr(L, n).number == v for n, v in numbers.items())
    call, e = L.lib().mlb_call_words, L.KV_APPEND_FP4
    args = [1 << 20, 1 << 20, 10, 64, 64, 1024, 128, 64, 1024, 128, 2, 0, 8, 128, 0, 0]
    assert call(e.number, e.pack(*args), e.num_words) == L.MLB_OK  # no tokens: nothing to do
    assert call(e.number, e.pack(*args), e.num_words - 1) == L.MLB_EINVAL and "15 words for 16" in L.last_error()
    assert call(e.number, None, e.num_words) == L.MLB_EINVAL
    assert call(99, e.pack(*args), e.num_words) == L.MLB_EINVAL and "99" in L.last_error()
    wide = args[:12] + [8 + (1 << 32)] + args[13:]  # a head count that an int would cut to 8
    assert call(e.number, e.pack(*wide), e.num_words) == L.MLB_EINVAL and "does not fit" in L.last_error()
    bad = args[:13] + [96] + args[14:]
    assert call(e.number, e.pack(*bad), e.num_words) == L.MLB_EUNSUPPORTED
    words = L.last_error()
    assert L.lib().mlb_kv_append_fp4(*bad) == L.MLB_EUNSUPPORTED and L.last_error() == words
    r = L.QK_NORM_ROPE  # a float among the words
    rope = [64, 0, 0, 64, 0, 0, 2, 1, 1, 1, 128, 64, 64, 8, 128, 0, 0, -1.0, 64, 0, 0, 64, 0, 0, 0, 0]
    assert call(r.number, r.pack(*rope), r.num_words) == L.MLB_EINVAL and "eps" in L.last_error()


def test_plan_for_4bit_pools(mlb):
    """The split rule of 4-bit pools covers every page once, whatever it picks, and leaves other pools' plans alone."""
    for lens, heads in (([1], (8, 2)), ([32001], (32, 8)), ([131072] * 16, (32, 8)), ([700, 5, 4096, 17] * 30, (28, 4)),
                        ([1000000, 3], (8, 1))):
        qo, width = list(range(len(lens) + 1)), -(-max(lens) // 16)
        plan = mlb.plan_attention(qo, lens, width, *heads, "cpu", pool_dtype=torch.uint8)
        seen = {}
        for seq, _, begin, end, *_ in plan.units_host.tolist():
            assert 0 <= begin < end <= -(-lens[seq] // 16)
            seen.setdefault(seq, []).append((begin, end))
        for s, n in enumerate(lens):
            runs = sorted(seen[s])
            assert runs[0][0] == 0 and runs[-1][1] == -(-n // 16)
            assert all(a[1] == b[0] for a, b in zip(runs, runs[1:]))
            assert plan.reduce_chunks_host[s] == len(runs)
        assert plan.max_pieces == plan.reduce_chunks_host.max()
        plain, half = (mlb.plan_attention(qo, lens, width, *heads, "cpu", pool_dtype=d) for d in (None, torch.bfloat16))
        assert np.array_equal(plain.units_host, half.units_host)


def test_workspace_keeps_what_it_has_outgrown(mlb):
    """A captured graph may hold the address of a buffer that a later call found too small."""
    ws, dev = mlb.Workspace(), torch.device("cpu")
    first = ws.get(4, 2, 64, dev)
    assert [t.numel() for t in first] == [512, 8] and ws.get(3, 2, 64, dev)[0] is first[0]
    refs = [weakref.ref(t) for t in first]
    del first
    grown = ws.get(5, 2, 64, dev)
    assert [t.numel() for t in grown] == [768, 12] and all(r() is not None for r in refs)
    other = ws.get(9, 2, 64, torch.device("meta"))
    assert other[0].device.type == "meta" and other[0].numel() == 9 * 2 * 64
    assert ws.get(6, 2, 64, dev)[0] is grown[0]  # back on the first device: no new buffer
