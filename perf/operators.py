"""Measured cases of the operators around the 4-bit paged KV cache: per-head norm and rotation of queries and
keys, the quantising append, the two of them in one pass, and paged attention over the 4-bit pages.

A 4-bit pool is uint8 [num_blocks, Hkv, 17, Dh / 2].  Rows 0..15 of a (block, head) are its 16 tokens' codes, two
e2m1 values a byte (the even dimension in the low nibble).  Row 16 holds the scales, one byte for each run of 32
dimensions of a token, at [run][2 * (token % 8) + token // 8]: a byte b stands for the float16 whose bits are
b << 7 (5 exponent bits and 3 mantissa bits, no sign).  A stored value is code * scale.
"""

from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

PACKAGE = "mini-llm-inference-server_b200"
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16
RUN = 32  # dimensions that share a scale
TOP_SCALE = 10240.0  # the largest scale: 6 times it is still a finite float16
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
THETA = 500000.0


# ---------------------------------------------------------------- cases


def _attend(name, rows, ctx, new, heads, dtype, shared=0, mixed=False, lens=1):
    return {"name": name, "op": "attend", "rows": rows, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0],
            "new_hi": new[1], "shared": shared, "mixed": mixed, "heads": heads[0], "kv_heads": heads[1],
            "head_dim": heads[2], "dtype": dtype, "lens": lens}


def _rows(name, op, tokens, heads, dtype, norm=True, far=131072, rot=None):
    return {"name": name, "op": op, "tokens": tokens, "heads": heads[0], "kv_heads": heads[1],
            "head_dim": heads[2], "rot": heads[2] if rot is None else rot, "dtype": dtype, "norm": norm, "far": far}


def listed():
    return [
        # the smallest decode step (batch 4, short contexts): its time is launch and round-trip latency
        _attend("attend_tiny", 4, (1, 256), (1, 1), (8, 2, 64), "bf16"),
        # one user with a long context: the whole GPU works on one row
        _attend("attend_row_32k", 1, (32001, 32001), (1, 1), (32, 8, 128), "f16"),
        # the ordinary decode step of an 8B model: 64 rows, contexts 512 to 4096
        _attend("attend_decode64", 64, (512, 4096), (1, 1), (32, 8, 128), "bf16"),
        # the largest: 16 rows of 128 Ki tokens, what a 4-bit cache is kept for
        _attend("attend_long16", 16, (131072, 131072), (1, 1), (32, 8, 128), "bf16"),
        # a prefix-cache hit: 128 decode rows behind the same 512 blocks
        _attend("attend_shared128", 128, (8208, 8704), (1, 1), (32, 8, 128), "bf16", shared=512),
        # chunked prefill on top of cached tokens
        _attend("attend_chunks", 4, (2100, 8192), (1024, 2048), (32, 8, 128), "f16"),
        # a decode step's queries and keys, views of one fused projection
        _rows("rope_decode64", "rope", 64, (32, 8, 128), "bf16"),
        # a long prefill's queries and keys, model without norms of queries and keys
        _rows("rope_prefill8k", "rope", 8192, (32, 8, 128), "bf16", norm=False),
        # the append of a decode step
        _rows("append_decode64", "append", 64, (32, 8, 128), "bf16"),
        # the append of a large prefill
        _rows("append_prefill16k", "append", 16384, (32, 8, 128), "f16"),
        # everything before the attention of a decode step in one call
        _rows("rope_append_decode64", "rope_append", 64, (32, 8, 128), "bf16", norm=False),
        # the same for a prefill of odd length
        _rows("rope_append_prefill", "rope_append", 4001, (28, 4, 128), "bf16", norm=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 2), (32, 8), (28, 4), (16, 16), (8, 1), (40, 8), (12, 2), (6, 2)]


def draw(rng):
    heads = (*rng.choice(HEADS), rng.choice([64, 128, 128, 256]))
    op = rng.choice(["attend", "attend", "attend", "rope", "append", "rope_append"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "attend":
        kind = rng.choice(["decode", "decode", "chunks", "mixed", "shared"])
        lens = rng.randrange(1 << 30)
        width = heads[1] * heads[2]
        if kind == "decode":
            rows = _log(rng, 1, 160)
            hi = _log(rng, 1, min(131072, max(16, (1 << 29) // (rows * width))))
            c = _attend("", rows, (max(1, hi // rng.choice([1, 2, 8])), hi), (1, 1), heads, dtype, lens=lens)
        elif kind == "shared":
            rows, pages = _log(rng, 4, 96), _log(rng, 8, 300)
            tail = _log(rng, 2, 400)
            c = _attend("", rows, (16 * pages + 1, 16 * pages + tail), (1, 1), heads, dtype, shared=pages, lens=lens)
        else:
            rows = _log(rng, 1, 4 if kind == "chunks" else 12)
            new = _log(rng, 2, 1500 if kind == "chunks" else 200)
            c = _attend("", rows, (new, new + _log(rng, 1, 4096)), (max(1, new // 3), new), heads, dtype,
                        mixed=kind == "mixed", lens=lens)
    else:
        norm = op != "rope_append" and rng.random() < 0.5
        dtype = rng.choice(["bf16", "f16", "f32"])
        rot = heads[2] if op == "rope_append" or rng.random() < 0.6 else heads[2] // 2
        c = _rows("", op, _log(rng, 1, 9000), heads, dtype, norm=norm, far=_log(rng, 64, 131072), rot=rot)
    del c["name"]
    return c


def _lengths(case):
    """(tokens in the cache before the step, new tokens) of each row; they go by the case alone."""
    r = np.random.default_rng(case["lens"])
    new = r.integers(case["new_lo"], case["new_hi"] + 1, size=case["rows"])
    if case["mixed"]:
        new[::2] = 1
    ctx = np.maximum(r.integers(case["ctx_lo"], case["ctx_hi"] + 1, size=case["rows"]), new)
    return ctx - new, new


def work(case):
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    e = DTYPE[case["dtype"]].itemsize
    row = 17 * d // 32  # bytes of one token of one head: d / 2 of codes and d / 32 of scales
    if case["op"] == "attend":
        cached, new = _lengths(case)
        ctx = cached + new
        unique = int(ctx.sum()) - case["shared"] * BLOCK * (case["rows"] - 1) * (case["shared"] > 0)
        keys = sum(int(n) * int(c) + int(n) * (int(n) + 1) // 2 for c, n in zip(cached, new))
        return {"bytes": 2 * unique * hkv * row + 2 * int(new.sum()) * h * d * e, "flops": 4 * keys * h * d}
    n = case["tokens"]
    q, kv = n * h * d * e, n * hkv * d * e
    table = n * case["rot"] * 4 + 8 * n
    if case["op"] == "rope":  # q and k in and out, one row of the table and one position a token
        return {"bytes": 2 * (q + kv) + table, "flops": 8 * n * (h + hkv) * d}
    if case["op"] == "append":  # k and v in, codes written; then codes read and the values they stand for written
        return {"bytes": 4 * kv + 4 * n * hkv * row + 16 * n, "flops": 12 * n * hkv * d}
    return {"bytes": 2 * q + 4 * kv + 4 * n * hkv * row + table + 16 * n, "flops": 12 * n * (h + 2 * hkv) * d}


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, scale, dtype):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _random_pool(g, blocks, hkv, d):
    """A pool of the values that an append of 0.5 N(0, 1) leaves, written block by block to bound the memory."""
    pool = torch.empty((blocks, hkv, 17, d // 2), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (hkv * BLOCK * d))
    for b in range(0, blocks, step):
        n = min(step, blocks - b)
        x = torch.randn((n, hkv, BLOCK, d), generator=g, device="cuda") * 0.5
        code, byte = _quantise(x, torch.float32)
        pool[b:b + n, :, :BLOCK] = code[..., 0::2] | (code[..., 1::2] << 4)
        pool[b:b + n, :, BLOCK] = byte.view(n, hkv, 2, 8, d // RUN).permute(0, 1, 4, 3, 2).reshape(n, hkv, d // 2)
    return pool


def prepare(case, seed):
    g = _gen(seed)
    h, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    dtype = DTYPE[case["dtype"]]
    if case["op"] == "attend":
        cached, new = _lengths(case)
        pages = -(-(cached + new) // BLOCK)
        total = int(pages.sum())
        blocks = total + total // 4 + 1
        ids = np.random.default_rng(seed).permutation(blocks)
        cut = np.concatenate([[0], np.cumsum(pages)])
        tables = [ids[cut[i]:cut[i + 1]].copy() for i in range(len(pages))]
        for t in tables[1:] if case["shared"] else []:
            t[:case["shared"]] = tables[0][:case["shared"]]
        padded = np.zeros((len(tables), int(pages.max())), dtype=np.int64)
        for i, t in enumerate(tables):
            padded[i, :len(t)] = t
        state = {"op": "attend", "q": _normal(g, (int(new.sum()), h, d), 1.0, dtype),
                 "k_cache": _random_pool(g, blocks, hkv, d), "v_cache": _random_pool(g, blocks, hkv, d),
                 "tables": torch.from_numpy(padded).cuda(), "cached": torch.from_numpy(cached).cuda(),
                 "new": torch.from_numpy(new).cuda(), "max_new": int(new.max())}
        if own:  # the step's metadata and plan: made once a step, used by every layer of it
            mlb = importlib.import_module(PACKAGE)
            meta = mlb.AttentionMetadata.build_arrays(cached, new, np.concatenate(tables), pages, BLOCK, "cuda")
            # rows of head_dim 256 are planned without the block tables: query tiles are built up to 128
            plan = mlb.plan_attention(meta.query_start_loc, meta.seq_lens, padded.shape[1], h, hkv, "cuda",
                                      block_tables_host=meta.block_tables_host if d <= 128 else None,
                                      pool_dtype=torch.uint8)
            state.update(meta=meta, plan=plan, workspace=mlb.Workspace())
        return state
    n = case["tokens"]
    # queries, keys and values as a fused projection leaves them: views of one tensor
    qkv = _normal(g, (n, h + 2 * hkv, d), 1.0, dtype)
    state = {"op": case["op"], "q": qkv[:, :h], "k": qkv[:, h:h + hkv], "v": qkv[:, h + hkv:]}
    if case["op"] != "append":
        rot, far = case["rot"], case["far"]
        inv = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        angle = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * inv
        state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], dim=1).float()
        state["positions"] = torch.randint(0, far, (n,), generator=g, device="cuda")
        state["q_weight"] = _normal(g, (d,), 0.2, dtype) + 1 if case["norm"] else None
        state["k_weight"] = _normal(g, (d,), 0.2, dtype) + 1 if case["norm"] else None
    if case["op"] != "rope":
        blocks = -(-n // BLOCK) + 3
        state["slots"] = torch.randperm(blocks * BLOCK, generator=g, device="cuda")[:n]
        state["k_cache"], state["v_cache"] = (
            torch.zeros((blocks, hkv, 17, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    return state


# ---------------------------------------------------------------- plain forms


def _quantise(x, wide=torch.float64):
    """e2m1 codes [..., d] and scale bytes [..., d / 32] of x: scale = max |x| of the run / 6 rounded to the byte
    format, code = x / scale rounded to the nearest level, ties to even codes; quotients in 64 bits, where the
    nearest level of a value next to a border is still the right one."""
    x = x.to(wide).nan_to_num(nan=0.0).clamp(-6 * TOP_SCALE, 6 * TOP_SCALE)
    runs = x.view(*x.shape[:-1], x.shape[-1] // RUN, RUN)
    want = (runs.abs().amax(-1) / 6).clamp(max=TOP_SCALE)
    step = torch.ldexp(torch.ones_like(want), (torch.frexp(want).exponent - 1).clamp(min=-14) - 3)
    scale = torch.round(want / step) * step
    byte = (scale.to(torch.float16).view(torch.int16) >> 7).to(torch.uint8)
    r = (runs / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]).abs()
    r = torch.where(scale[..., None] > 0, r, torch.zeros_like(r))
    code = ((r > 0.25).to(torch.uint8) + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5.0))
    return (code | (torch.signbit(runs).to(torch.uint8) << 3)).view(x.shape), byte


def _levels(dtype):
    return torch.tensor([*LEVELS, *(-v for v in LEVELS)], dtype=dtype, device="cuda")


def _scale(byte):
    return (byte.to(torch.int16) << 7).view(torch.float16)


def _write(pool, slots, x):
    hkv, d = x.shape[1:]
    code, byte = _quantise(x)
    block, t = slots // BLOCK, slots % BLOCK
    pool[block, :, t] = code[..., 0::2] | (code[..., 1::2] << 4)
    heads, runs = torch.arange(hkv, device="cuda"), torch.arange(d // RUN, device="cuda")
    at = runs * BLOCK + (2 * (t % 8) + t // 8)[:, None]
    pool[block[:, None, None], heads[None, :, None], BLOCK, at[:, None, :]] = byte


def _read(pool, slots, dtype):
    hkv, d = pool.shape[1], 2 * pool.shape[3]
    block, t = slots // BLOCK, slots % BLOCK
    packed = pool[block, :, t]
    code = torch.stack([packed & 15, packed >> 4], dim=-1).view(len(slots), hkv, d)
    heads, runs = torch.arange(hkv, device="cuda"), torch.arange(d // RUN, device="cuda")
    at = runs * BLOCK + (2 * (t % 8) + t // 8)[:, None]
    scale = _scale(pool[block[:, None, None], heads[None, :, None], BLOCK, at[:, None, :]])
    value = _levels(torch.float32)[code.int()].view(len(slots), hkv, d // RUN, RUN) * scale.float()[..., None]
    return value.view(len(slots), hkv, d).to(dtype)


def _pages(pool, tables):
    """The rows' keys or values in 32 bits: [S, Hkv, pages * 16, d]."""
    hkv, half = pool.shape[1], pool.shape[3]
    s, w = tables.shape
    page = pool[tables]  # [S, W, Hkv, 17, d / 2]
    packed = page[:, :, :, :BLOCK]
    code = torch.stack([packed & 15, packed >> 4], dim=-1).view(s, w, hkv, BLOCK, 2 * half)
    scale = _scale(page[:, :, :, BLOCK].reshape(s, w, hkv, half // 16, 8, 2)).permute(0, 1, 2, 5, 4, 3)
    scale = scale.reshape(s, w, hkv, BLOCK, half // 16, 1).float()
    value = _levels(torch.float32)[code.int()].view(s, w, hkv, BLOCK, half // 16, RUN) * scale
    return value.view(s, w, hkv, BLOCK, 2 * half).transpose(1, 2).reshape(s, hkv, w * BLOCK, 2 * half)


def _plain_attend(st):
    q, cached, new = st["q"], st["cached"], st["new"]
    s, m, (n, h, d) = len(new), st["max_new"], q.shape
    hkv = st["k_cache"].shape[1]
    k, v = _pages(st["k_cache"], st["tables"]), _pages(st["v_cache"], st["tables"])
    owner = torch.repeat_interleave(torch.arange(s, device="cuda"), new, output_size=n)
    nth = torch.arange(n, device="cuda") - (new.cumsum(0) - new)[owner]
    padded = torch.zeros((s, m, h, d), device="cuda")
    padded[owner, nth] = q.float()
    rows = padded.view(s, m, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(s, hkv, m * (h // hkv), d)
    score = torch.matmul(rows, k.transpose(2, 3)) / math.sqrt(d)
    last = cached[:, None] + torch.arange(m, device="cuda")  # position of each new token: it sees keys up to its own
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, :, None]
    seen = seen.repeat_interleave(h // hkv, dim=1)[:, None]
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    out = out.view(s, hkv, m, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(s, m, h, d)
    return out[owner, nth].to(q.dtype)


def _plain_rope(x, weight, positions, cos_sin):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[positions][:, None].split(half, dim=-1)
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], dim=-1).to(x.dtype)


def run(st):
    if own:
        ops = importlib.import_module(PACKAGE).ops
        if st["op"] == "attend":
            meta = st["meta"]
            return ops.paged_attention_fp4(st["q"], st["k_cache"], st["v_cache"], meta.block_tables_i32,
                                           meta.seq_lens_i32, meta.qo_indptr, st["plan"], st["workspace"])
        if st["op"] == "rope":
            return ops.qk_norm_rope(st["q"], st["k"], st["positions"], st["cos_sin"], st["q_weight"], st["k_weight"],
                                    eps=EPS)
        if st["op"] == "append":
            ops.kv_append_fp4(st["k_cache"], st["v_cache"], st["slots"], st["k"], st["v"])
            return ops.kv_read_fp4(st["k_cache"], st["v_cache"], st["slots"], st["k"].dtype)
        q = ops.qk_norm_rope_append_fp4(st["q"], st["k"], st["v"], st["positions"], st["cos_sin"], st["k_cache"],
                                        st["v_cache"], st["slots"], st["q_weight"], st["k_weight"], eps=EPS)
        return (q, *ops.kv_read_fp4(st["k_cache"], st["v_cache"], st["slots"], st["k"].dtype))
    if st["op"] == "attend":
        return _plain_attend(st)
    q, k = st["q"], st["k"]
    if st["op"] != "append":
        q = _plain_rope(q, st["q_weight"], st["positions"], st["cos_sin"])
        k = _plain_rope(k, st["k_weight"], st["positions"], st["cos_sin"])
        if st["op"] == "rope":
            return q, k
    _write(st["k_cache"], st["slots"], k)
    _write(st["v_cache"], st["slots"], st["v"])
    stored = (_read(st["k_cache"], st["slots"], k.dtype), _read(st["v_cache"], st["slots"], k.dtype))
    return stored if st["op"] == "append" else (q, *stored)


# ---------------------------------------------------------------- from the definition, in 64 bits


def _exact_stored(x):
    """What a 4-bit pool holds of x: the distance to every level is compared, the nearer one wins."""
    d = x.shape[-1]
    runs = x.double().nan_to_num(nan=0.0).clamp(-6 * TOP_SCALE, 6 * TOP_SCALE).reshape(-1, RUN)
    grid = (torch.arange(227, dtype=torch.int16, device="cuda") << 7).view(torch.float16).double()  # every scale
    want = runs.abs().amax(-1) / 6

    def nearest(value, table):  # index of the nearest entry, the even one of two equally near
        hi = torch.searchsorted(table, value).clamp(1, len(table) - 1)
        lo = hi - 1
        up, down = table[hi] - value, value - table[lo]
        return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)

    scale = grid[nearest(want, grid)][:, None]
    level = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    ratio = torch.where(scale > 0, runs.abs() / torch.where(scale > 0, scale, 1.0), 0.0)
    return (level[nearest(ratio.clamp(max=6.0), level)] * scale * torch.sign(runs)).view(*x.shape[:-1], d)


def _exact_rope(x, weight, positions, cos_sin):
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * weight.double()
    r = cos_sin.shape[1] // 2
    t = cos_sin.double().index_select(0, positions).unsqueeze(1)
    out = y.clone()
    out[..., :r] = y[..., :r] * t[..., :r] - y[..., r:2 * r] * t[..., r:]
    out[..., r:2 * r] = y[..., r:2 * r] * t[..., :r] + y[..., :r] * t[..., r:]
    return out


def _exact_rows(pool, ids, length):
    """Keys or values of one row in 64 bits: [Hkv, length, d], token by token of its pages."""
    page = pool.index_select(0, ids).permute(1, 0, 2, 3)  # [Hkv, pages, 17, d / 2]
    hkv, pages, _, half = page.shape
    nibble = torch.empty((hkv, pages, BLOCK, 2 * half), dtype=torch.long, device="cuda")
    nibble[..., 0::2] = (page[:, :, :BLOCK] % 16).long()
    nibble[..., 1::2] = torch.div(page[:, :, :BLOCK], 16, rounding_mode="floor").long()
    sign = 1.0 - 2.0 * (nibble >= 8).double()
    value = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")[nibble % 8] * sign
    b = page[:, :, BLOCK].reshape(hkv, pages, half // 16, BLOCK).long()
    order = torch.tensor([2 * (t % 8) + t // 8 for t in range(BLOCK)], device="cuda")
    b = b[..., order].transpose(2, 3)  # [Hkv, pages, token, run]
    e, m = (b // 8).double(), (b % 8).double()
    scale = torch.where(e > 0, (1 + m / 8) * torch.exp2(e - 15), m / 8 * 2.0**-14)
    return (value * scale.repeat_interleave(RUN, dim=-1)).reshape(hkv, pages * BLOCK, 2 * half)[:, :length]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] != "attend":
        q, k = st["q"], st["k"]
        if case["op"] != "append":
            q = _exact_rope(q, st["q_weight"], st["positions"], st["cos_sin"])
            k = _exact_rope(k, st["k_weight"], st["positions"], st["cos_sin"])
            if case["op"] == "rope":
                return q, k
            k = k.to(st["k"].dtype)  # the keys are rounded to their own type before they are stored
        stored = (_exact_stored(k), _exact_stored(st["v"]))
        return stored if case["op"] == "append" else (q, *stored)
    q, group = st["q"].double(), case["heads"] // case["kv_heads"]
    out, at = torch.empty_like(q), 0
    for i, (c, n) in enumerate(zip(*_lengths(case))):
        c, n = int(c), int(n)
        ids = st["tables"][i, :-(-(c + n) // BLOCK)]
        k, v = _exact_rows(st["k_cache"], ids, c + n), _exact_rows(st["v_cache"], ids, c + n)
        for j in range(0, n, 256):  # new tokens of the row, some at a time
            m = min(256, n - j)
            x = q[at + j:at + j + m].reshape(m, -1, group, case["head_dim"]).permute(1, 0, 2, 3).flatten(1, 2)
            s = x @ k.mT / math.sqrt(case["head_dim"])
            hidden = torch.arange(c + n, device="cuda") > (c + j + torch.arange(m, device="cuda"))[:, None]
            s = s.masked_fill(hidden.repeat_interleave(group, dim=0), -math.inf)
            o = torch.softmax(s, dim=-1) @ v
            out[at + j:at + j + m] = o.unflatten(1, (m, group)).transpose(0, 1).flatten(1, 2)
        at += n
    return out
