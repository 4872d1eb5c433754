"""Torch-facing wrappers of the C ABI: tensors in, raw pointers + strides + the current CUDA stream out.

Every function validates what the kernels rely on (shapes, dtypes, devices, contiguity of the pools)
and raises `ValueError` like the reference does for malformed input (metadata.py:75-76); device-side
range faults (a bad slot or block id) are skipped by the kernels and recorded in an optional int32
error word instead of faulting the GPU.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from ._lib import (MAX_OUT_DESTS, MEMBER_INT32S, SHARED_UNIT_INT32S, WORK_UNIT_INT32S, AppendRows, OutTargets, check,
                   lib)

DTYPE_CODE = {torch.float32: _lib.MLB_F32, torch.float16: _lib.MLB_F16, torch.bfloat16: _lib.MLB_BF16}
BLOCK_SIZE = 16


def _code(t: torch.Tensor, what: str) -> int:
    try:
        return DTYPE_CODE[t.dtype]
    except KeyError:
        raise ValueError(f"{what}: dtype {t.dtype} not supported (float32, float16, bfloat16)") from None


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device: torch.device) -> int:
    """Handle of torch's current stream on `device` (the raw query: a decode step makes ~100 of these)."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check_pool(pool: torch.Tensor, what: str) -> None:
    if pool.dim() != 4 or not pool.is_contiguous():
        raise ValueError(f"{what}: pools are contiguous [num_blocks, block_size, Hkv, Dh], got {tuple(pool.shape)}")
    if not pool.is_cuda:
        raise ValueError(f"{what}: pools must be CUDA tensors")


def _check_rows(x: torch.Tensor, hkv: int, dh: int, what: str) -> None:
    if x.dim() != 3 or x.shape[1:] != (hkv, dh) or (x.shape[0] and x.stride(2) != 1):
        raise ValueError(f"{what}: rows must be [N, {hkv}, {dh}] with unit stride on the last dim, "
                         f"got {tuple(x.shape)} strides {x.stride()}")


# ---------------------------------------------------------------- K1: append


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, k: torch.Tensor,
              v: torch.Tensor, err: torch.Tensor | None = None) -> None:
    """write_kv (paged_torch_ref.py:23-28) on the GPU: pools[slot_mapping[i]] = k[i] / v[i], cast to the
    pool dtype (round to nearest even).  k, v may be strided views [N, Hkv, Dh]."""
    _check_pool(k_cache, "kv_append")
    _check_pool(v_cache, "kv_append")
    nb, bs, hkv, dh = k_cache.shape
    if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise ValueError("kv_append: k_cache and v_cache differ")
    _check_rows(k, hkv, dh, "kv_append k")
    _check_rows(v, hkv, dh, "kv_append v")
    n = k.shape[0]
    if v.shape[0] != n or slot_mapping.shape != (n,):
        raise ValueError(f"kv_append: {n} k rows, {v.shape[0]} v rows, slot_mapping {tuple(slot_mapping.shape)}")
    if slot_mapping.dtype != torch.long or not slot_mapping.is_contiguous():
        raise ValueError("kv_append: slot_mapping must be a contiguous int64 tensor")
    if k.dtype != v.dtype:
        raise ValueError("kv_append: k and v dtypes differ")
    for t in (v_cache, slot_mapping, k, v):
        if t.device != k_cache.device:
            raise ValueError("kv_append: all tensors must be on the pools' device")
    if n == 0:
        return
    rc = lib().mlb_kv_append(k_cache.data_ptr(), v_cache.data_ptr(), _code(k_cache, "kv_append"), nb, bs,
                             slot_mapping.data_ptr(), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
                             v.stride(0), v.stride(1), _code(k, "kv_append"), n, hkv, dh, _ptr(err),
                             _stream(k_cache.device))
    check(rc, "kv_append")


# ---------------------------------------------------------------- K2: plan, attention, reduction


@dataclass
class AttentionPlan:
    """A step's split of paged-attention work (built once per AttentionMetadata, reused by every layer)."""

    units: torch.Tensor  # device int32 [num_units, 8]: mlb_work_unit records
    num_units: int
    shared_units: torch.Tensor  # device int32 [num_shared_units, 8]: mlb_shared_unit records (may be empty)
    num_shared_units: int
    members: torch.Tensor  # device int32 [num_members, 4]: mlb_share_member records
    reduce_rows: torch.Tensor  # device int32 [N]
    reduce_chunks: torch.Tensor  # device int32 [N]
    num_partial_rows: int
    tokens_per_tile: int
    num_heads: int
    num_kv_heads: int
    num_tokens: int
    units_host: np.ndarray  # the same records on the host (inspection and tests)
    shared_host: np.ndarray
    members_host: np.ndarray
    reduce_rows_host: np.ndarray
    reduce_chunks_host: np.ndarray  # [N] pieces per token on the host
    has_query_tiles: bool = False  # kind-1 shared units (rows of >= 16 new tokens) in the plan
    max_pieces: int = 0  # the most pieces of one token
    num_seqs: int = 0
    max_blocks: int = 0  # width of the block tables it was planned for
    last_position: int = -1  # the largest position of a new token


def _i32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.int32))


def plan_attention(qo_indptr: list[int], seq_lens: list[int], max_blocks: int, num_heads: int, num_kv_heads: int,
                   device: torch.device | str, block_size: int = BLOCK_SIZE, num_sms: int | None = None,
                   pages_per_unit: int = 0, block_tables_host: np.ndarray | None = None,
                   pool_dtype: torch.dtype | None = None) -> AttentionPlan:
    """Split the step into units (host work, like FlashInfer's plan(); flashinfer_backend.py:48-64).

    qo_indptr / seq_lens are the host lists AttentionMetadata keeps (metadata.py:39-40), so planning
    needs no device round trip.  With `block_tables_host` (int32 [S, W]) decode rows that share leading
    blocks (prefix-cache hits) are planned as shared-prefix units (16-bit and 4-bit pools only).  The plan is
    copied to the device in one transfer.  `pool_dtype` torch.uint8: the plan is for 4-bit pools
    (`paged_attention_fp4`); any plan is right for any pool, the split size is what differs.
    """
    device = torch.device(device)
    qo, lens = _i32(qo_indptr), _i32(seq_lens)
    s = len(lens)
    if qo.shape != (s + 1,):
        raise ValueError(f"plan: qo_indptr has {qo.shape[0]} entries for {s} sequences")
    n_tok = int(qo[-1]) if s else 0
    if num_sms is None:
        num_sms = torch.cuda.get_device_properties(device).multi_processor_count if device.type == "cuda" else 148
    tables = None if block_tables_host is None else _i32(block_tables_host)
    if tables is not None and (tables.ndim != 2 or tables.shape[0] != s):
        raise ValueError(f"plan: block_tables_host must be [{s}, W], got {tables.shape}")
    if pool_dtype is torch.uint8 and pages_per_unit <= 0:
        pages_per_unit = _lib.PAGES_PER_UNIT_FP4
    L = lib()
    nu, ns, nm, npart = (ctypes.c_int64(0) for _ in range(4))
    head = (qo.ctypes.data, lens.ctypes.data, s, max_blocks, None if tables is None else tables.ctypes.data,
            0 if tables is None else tables.shape[1], num_heads, num_kv_heads, block_size, num_sms, pages_per_unit)
    check(L.mlb_plan_attention(*head, None, 0, ctypes.byref(nu), None, 0, ctypes.byref(ns), None, 0,
                               ctypes.byref(nm), None, None, n_tok, ctypes.byref(npart)), "plan_attention")
    units = np.zeros((max(nu.value, 1), WORK_UNIT_INT32S), dtype=np.int32)
    shared = np.zeros((max(ns.value, 1), SHARED_UNIT_INT32S), dtype=np.int32)
    members = np.zeros((max(nm.value, 1), MEMBER_INT32S), dtype=np.int32)
    rows = np.empty(max(n_tok, 1), dtype=np.int32)
    chunks = np.empty(max(n_tok, 1), dtype=np.int32)
    check(L.mlb_plan_attention(*head, units.ctypes.data, units.shape[0], ctypes.byref(nu), shared.ctypes.data,
                               shared.shape[0], ctypes.byref(ns), members.ctypes.data, members.shape[0],
                               ctypes.byref(nm), rows.ctypes.data, chunks.ctypes.data, n_tok, ctypes.byref(npart)),
          "plan_attention")
    u, sh, m = nu.value, ns.value, nm.value
    # one host -> device copy for the whole plan
    parts = [units[:u].reshape(-1), shared[:sh].reshape(-1), members[:m].reshape(-1), rows[:n_tok], chunks[:n_tok]]
    offs = np.cumsum([0] + [p.size for p in parts])
    host = torch.from_numpy(np.concatenate(parts))
    dev = host.pin_memory().to(device, non_blocking=True) if device.type == "cuda" else host.clone()
    seg = [dev[offs[i]:offs[i + 1]] for i in range(len(parts))]
    return AttentionPlan(seg[0].view(u, WORK_UNIT_INT32S), u, seg[1].view(sh, SHARED_UNIT_INT32S), sh,
                         seg[2].view(m, MEMBER_INT32S), seg[3], seg[4], npart.value,
                         max(1, 8 // (num_heads // num_kv_heads)), num_heads, num_kv_heads, n_tok,
                         units[:u].copy(), shared[:sh].copy(), members[:m].copy(), rows[:n_tok].copy(),
                         chunks[:n_tok].copy(), bool(sh and ((shared[:sh, 6] & 0xFF) == 1).any()),
                         int(chunks[:n_tok].max()) if n_tok else 0, s, max_blocks,
                         int(lens[qo[1:] > qo[:-1]].max()) - 1 if n_tok else -1)


class _Scratch:
    """One pair of a workspace's buffers, and what has been done with it."""

    __slots__ = ("o", "lse", "small", "captured", "streams")

    def __init__(self, size_o: int, size_l: int, device: torch.device) -> None:
        self.o, self.lse = (torch.empty(max(n, 1), dtype=torch.float32, device=device) for n in (size_o, size_l))
        self.small = 4 * (self.o.numel() + self.lse.numel()) <= Workspace.SMALL_BYTES
        self.captured = False  # handed out during a stream capture: a graph holds its address
        self.streams: set[int] = set()  # streams that the allocator knows it is used on


class Workspace:
    """Split-K scratch (fp32 partial rows + their log-sum-exp), grown on demand and reused across calls; one buffer of
    each kind per device.  An outgrown one that was handed out during a stream capture stays allocated, since the graph
    holds its address, until `release`; so does a small one.  What replaces those is larger by half at least, so that
    all of them together stay below three times the largest.  Every other outgrown buffer goes back to the allocator
    before its successor is made, which is no larger than asked for."""

    SMALL_BYTES = 1 << 24  # a decode step's scratch: kept whatever held it, so that its calls need not look

    def __init__(self) -> None:
        self._pairs: dict[torch.device, list[_Scratch]] = {}  # outgrown ones that stay, then the one in use

    def get(self, rows: int, heads: int, dh: int, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
        need_o, need_l = rows * heads * dh, rows * heads
        pairs = self._pairs.get(device)
        if not pairs or pairs[-1].o.numel() < need_o or pairs[-1].lse.numel() < need_l:
            pairs = self._grow(need_o, need_l, device)
        p = pairs[-1]
        if not p.small and not p.captured and device.type == "cuda":
            if _capturing(device):
                p.captured = True
            elif _stream(device) not in p.streams:  # it is freed only when every stream is done with it
                p.streams.add(_stream(device))
                for t in (p.o, p.lse):
                    t.record_stream(torch.cuda.current_stream(device))
        return p.o, p.lse

    def _grow(self, need_o: int, need_l: int, device: torch.device) -> list[_Scratch]:
        pairs = self._pairs.setdefault(device, [])
        if pairs:
            last = pairs[-1]
            size_o, size_l = last.o.numel(), last.lse.numel()
            if last.small or last.captured:
                size_o, size_l = 3 * size_o // 2, 3 * size_l // 2
            else:
                del pairs[-1]
            del last
            need_o, need_l = max(need_o, size_o), max(need_l, size_l)
        pairs.append(_Scratch(need_o, need_l, device))
        return pairs

    def release(self) -> None:
        """Free every outgrown buffer, once the GPU is done with them.  No graph that was captured with this workspace
        before may be replayed after."""
        for device, pairs in self._pairs.items():
            if device.type == "cuda":
                torch.cuda.synchronize(device)
            del pairs[:-1]
            for p in pairs:
                p.captured = False


def _capturing(device: torch.device) -> bool:
    """Whether torch's current stream on `device` is being captured into a graph."""
    if torch.cuda.current_device() == device.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, qo_indptr: torch.Tensor, plan: AttentionPlan,
                    workspace: Workspace | None = None, out: torch.Tensor | None = None, scale: float | None = None,
                    err: torch.Tensor | None = None, targets: OutTargets | None = None,
                    append: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor | None:
    """paged_attention (paged_torch_ref.py:40-74) on the GPU: q [N, H, Dh] -> [N, H, Dh] in q's dtype.

    block_tables int32 [S, W], seq_lens int32 [S], qo_indptr int32 [S + 1] are AttentionMetadata's
    device tensors (block_tables_i32, seq_lens_i32, qo_indptr).  The pools must already hold this
    step's k/v (kv_append first), unless `append` = (k, v, slot_mapping) asks the attention launch to do
    the append itself (see `attention_partials`).  Launches the shared-prefix and per-sequence attention
    kernels, then the split-K reduction when the plan split any sequence.  With `targets` (see
    `out_targets`) the rows go to those destinations instead and nothing is returned.
    """
    workspace = workspace or Workspace()
    out = attention_partials(q, k_cache, v_cache, block_tables, seq_lens, qo_indptr, plan, workspace, out, scale,
                             err, targets, append)
    splitk_reduce(plan, workspace, out, targets, q.dtype, q.shape[2], q.device)
    return out


def out_targets(dests: list[int], head_offset: int, stride_tok: int, stride_head: int) -> OutTargets:
    """mlb_out_targets: store every final row (token t, local head h) at element offset
    t * stride_tok + (head_offset + h) * stride_head of each destination address in `dests`."""
    if not 1 <= len(dests) <= MAX_OUT_DESTS:
        raise ValueError(f"out_targets: 1..{MAX_OUT_DESTS} destinations, got {len(dests)}")
    t = OutTargets()
    t.num_dests, t.head_offset, t.stride_tok, t.stride_head = len(dests), head_offset, stride_tok, stride_head
    for i, d in enumerate(dests):
        t.dests[i] = d
    return t


def attention_partials(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, qo_indptr: torch.Tensor, plan: AttentionPlan, workspace: Workspace,
                       out: torch.Tensor | None = None, scale: float | None = None,
                       err: torch.Tensor | None = None, targets: OutTargets | None = None,
                       append: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor | None:
    """The attention kernels (K2s, K2a): unsplit sequences are final in `out` (or `targets`); split ones
    leave fp32 partial rows in `workspace` for `splitk_reduce`.

    append = (k, v, slot_mapping): kv_append fused into the attention launch (mlb_paged_attention_append;
    torch_ref.py:46-48 writes, then attends).  The caller guarantees what that entry point needs:
    slot_mapping is the one the block tables give, and every written block is in one sequence's context
    pages only (AttentionMetadata.append_private); `can_fuse_append` checks the rest."""
    _check_pool(k_cache, "paged_attention")
    _check_pool(v_cache, "paged_attention")
    nb, bs, hkv, dh = k_cache.shape
    if q.dim() != 3 or q.shape[2] != dh or (q.shape[0] and q.stride(2) != 1):
        raise ValueError(f"paged_attention: q must be [N, H, {dh}] with unit last stride, got {tuple(q.shape)}")
    n, h = q.shape[0], q.shape[1]
    if q.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype or v_cache.shape != k_cache.shape:
        raise ValueError(f"paged_attention: q {q.dtype} and pools {k_cache.dtype}/{v_cache.dtype} must agree")
    if (plan.num_heads, plan.num_kv_heads, plan.num_tokens) != (h, hkv, n):
        raise ValueError("paged_attention: the plan was built for another shape")
    for t, name in ((block_tables, "block_tables"), (seq_lens, "seq_lens"), (qo_indptr, "qo_indptr")):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != q.device:
            raise ValueError(f"paged_attention: {name} must be a contiguous int32 tensor on {q.device}")
    if targets is not None:
        out = None
    elif out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("paged_attention: out must match q")
    if n == 0 or plan.num_units + plan.num_shared_units == 0:
        return out
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    po = plse = None
    if plan.num_partial_rows:
        po, plse = workspace.get(plan.num_partial_rows, h, dh, q.device)
    args = (q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
            _code(q, "paged_attention"), nb, bs, h, hkv, dh, scale, block_tables.data_ptr(), block_tables.stride(0),
            seq_lens.data_ptr(), qo_indptr.data_ptr(), seq_lens.shape[0], plan.units.data_ptr(), plan.num_units,
            plan.shared_units.data_ptr(), plan.num_shared_units, plan.members.data_ptr(), _ptr(po), _ptr(plse),
            plan.num_partial_rows, _ptr(out), *_strides(out), _targets(targets))
    if append is None:
        rc = lib().mlb_paged_attention(*args, _ptr(err), _stream(q.device))
        check(rc, "paged_attention")
        return out
    k, v, slots = append
    if not can_fuse_append(plan, k_cache, k, v):
        raise ValueError("paged_attention: this append cannot ride in the attention launch (see can_fuse_append)")
    if slots.dtype != torch.long or not slots.is_contiguous() or slots.shape != (n,) or slots.device != q.device:
        raise ValueError(f"paged_attention: slot_mapping must be a contiguous int64 [{n}] tensor on {q.device}")
    rows = AppendRows()
    rows.k, rows.v, rows.slot_mapping, rows.num_tokens = k.data_ptr(), v.data_ptr(), slots.data_ptr(), n
    rows.k_stride_tok, rows.k_stride_head, rows.v_stride_tok, rows.v_stride_head = (k.stride(0), k.stride(1),
                                                                                    v.stride(0), v.stride(1))
    rc = lib().mlb_paged_attention_append(*args, ctypes.byref(rows), _ptr(err), _stream(q.device))
    check(rc, "paged_attention_append")
    return out


def can_fuse_append(plan: AttentionPlan, k_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> bool:
    """Whether kv_append can ride in the attention launch, as far as the plan and tensors go: 16-bit pools
    with head_dim 64 / 128, k / v [N, Hkv, Dh] in the pools' dtype on their device with 16-byte aligned
    rows, N the plan's token count, and no query-tile units (rows of >= 16 new tokens).  The metadata's
    half of the condition is AttentionMetadata.append_private."""
    dt = k_cache.dtype
    if plan.has_query_tiles or (dt is not torch.bfloat16 and dt is not torch.float16) or k_cache.shape[3] not in (64, 128):
        return False
    shape = (plan.num_tokens, k_cache.shape[2], k_cache.shape[3])
    for t in (k, v):
        if t.dtype is not dt or t.shape != shape or t.device != k_cache.device:
            return False
        if shape[0]:
            s0, s1, s2 = t.stride()
            if s2 != 1 or (s0 | s1) & 7 or t.data_ptr() & 15:  # 16-byte rows: strides x 2 B multiples of 16
                return False
    return True


def splitk_reduce(plan: AttentionPlan, workspace: Workspace, out: torch.Tensor | None,
                  targets: OutTargets | None = None, dtype: torch.dtype | None = None, head_dim: int | None = None,
                  device: torch.device | None = None) -> None:
    """K2b: combine the split sequences' partial rows into `out` (no-op when the plan split nothing).
    With `targets`, the rows go there instead; dtype / head_dim / device then describe them."""
    if not plan.num_partial_rows or plan.num_tokens == 0:
        return
    if targets is None:
        if out is None:
            raise ValueError("splitk_reduce: no out and no targets")
        dtype, head_dim, device = out.dtype, out.shape[2], out.device
    n, h = plan.num_tokens, plan.num_heads
    po, plse = workspace.get(plan.num_partial_rows, h, head_dim, device)
    rc = lib().mlb_splitk_reduce(po.data_ptr(), plse.data_ptr(), plan.num_partial_rows, plan.reduce_rows.data_ptr(),
                                 plan.reduce_chunks.data_ptr(), plan.tokens_per_tile, n, h, head_dim, _ptr(out),
                                 *_strides(out), DTYPE_CODE[dtype], _targets(targets), _stream(device))
    check(rc, "splitk_reduce")


def splitk_reduce_gather(plan: AttentionPlan, workspace: Workspace, targets: OutTargets, self_dest: int,
                         dtype: torch.dtype, head_dim: int, device: torch.device) -> None:
    """The split-K reduction carrying the output all-gather (mlb_splitk_reduce_gather): after
    `attention_partials` wrote the unsplit rows into destination `self_dest` only, every row of the step
    is stored into every destination.  Follow it with the peers' barrier (`PeerOutputs.barrier`)."""
    po = plse = None
    if plan.num_partial_rows:
        po, plse = workspace.get(plan.num_partial_rows, plan.num_heads, head_dim, device)
    rc = lib().mlb_splitk_reduce_gather(_ptr(po), _ptr(plse), plan.num_partial_rows, plan.reduce_rows.data_ptr(),
                                        plan.reduce_chunks.data_ptr(), plan.tokens_per_tile, plan.num_tokens,
                                        plan.num_heads, head_dim, DTYPE_CODE[dtype], ctypes.byref(targets), self_dest,
                                        _stream(device))
    check(rc, "splitk_reduce_gather")


def splitk_reduce_exchange(plan: AttentionPlan, workspace: Workspace, peers, slot: int, dtype: torch.dtype,
                           head_dim: int, device: torch.device, err: torch.Tensor | None = None) -> None:
    """The output all-gather as flagged packets (mlb_splitk_reduce_exchange): after `attention_partials` left
    this rank's unsplit rows in its own buffer of `slot` (`peers.local_targets`), one launch finishes this
    rank's rows, sends them to every peer and waits for theirs; no barrier follows.  `peers` is the
    `sharding.PeerOutputs` of the step (its packet areas and state words)."""
    po = plse = None
    if plan.num_partial_rows:
        po, plse = workspace.get(plan.num_partial_rows, plan.num_heads, head_dim, device)
    rc = lib().mlb_splitk_reduce_exchange(_ptr(po), _ptr(plse), plan.num_partial_rows, plan.reduce_rows.data_ptr(),
                                          plan.reduce_chunks.data_ptr(), plan.tokens_per_tile, plan.num_tokens,
                                          plan.num_heads, head_dim, DTYPE_CODE[dtype], peers.slot_address(slot),
                                          peers.num_heads * head_dim, head_dim, peers.packet_areas(),
                                          peers.capacity, peers.rank, peers.world, peers.state_address,
                                          peers.timeout_ns, peers.err.data_ptr() if err is None else err.data_ptr(),
                                          _stream(device))
    check(rc, "splitk_reduce_exchange")


def _strides(out: torch.Tensor | None) -> tuple[int, int]:
    return (out.stride(0), out.stride(1)) if out is not None else (0, 0)


def _targets(t: OutTargets | None):
    return ctypes.byref(t) if t is not None else None


# ---------------------------------------------------------------- 4-bit pools

FP4_ROWS = BLOCK_SIZE + 1  # rows of a (block, head): 16 tokens' codes, then their scales
FP4_RUN = 32  # dims that share a scale
WIDE_REDUCE_PIECES = 8  # few rows of more pieces than this are reduced by a CTA per head instead of a warp


def is_fp4(pool: torch.Tensor) -> bool:
    """Whether `pool` is a 4-bit pool (uint8 [num_blocks, Hkv, 17, Dh / 2], see include/mlb_paged_kv.h)."""
    return pool.dtype is torch.uint8


def pool_kv_heads(pool: torch.Tensor) -> int:
    return pool.shape[1] if is_fp4(pool) else pool.shape[2]


def fp4_pool_shape(num_blocks: int, num_kv_heads: int, head_dim: int) -> tuple[int, int, int, int]:
    """Shape of a 4-bit pool: 8.5 x head_dim bytes per (block, head) instead of 32 x head_dim in 16 bits."""
    if head_dim not in (64, 128, 256):
        raise ValueError(f"4-bit pools: head_dim {head_dim} (supported: 64, 128, 256)")
    return num_blocks, num_kv_heads, FP4_ROWS, head_dim // 2


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _launch(entry: _lib.Entry, what: str, device: int, *args) -> None:
    """Call an entry point with the current stream of `device` (an ordinal), made current if it is not already."""
    if _current_device() == device:
        stream = _raw_stream(device) if _raw_stream else torch.cuda.current_stream(device).cuda_stream
        rc = lib().mlb_call_words(entry.number, entry.pack(*args, stream), entry.num_words)
    else:
        with torch.cuda.device(device):
            stream = torch.cuda.current_stream(device).cuda_stream
            rc = lib().mlb_call_words(entry.number, entry.pack(*args, stream), entry.num_words)
    if rc:
        check(rc, what)


def _adr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _err_adr(err: torch.Tensor | None, device: int, what: str) -> int:
    """Address of a device error word (int32, on the device of the launch), 0 for none."""
    if err is None:
        return 0
    if err.dtype is not torch.int32 or err.get_device() != device or not err.numel():
        raise ValueError(f"{what}: err must be an int32 tensor on the pools' device, got {err.dtype} "
                         f"{tuple(err.shape)} on {err.device}")
    return err.data_ptr()


# A decode step makes several of these calls per layer, each a few microseconds on the GPU: every entry point below
# tests its arguments with one expression of cheap attributes, and only where that fails with the checks that say what
# is wrong (or that the case is an uncommon one that is fine: an empty tensor's strides).


def _check_fp4_pools(k_cache: torch.Tensor, v_cache: torch.Tensor, what: str) -> tuple[int, int, int]:
    """(num_blocks, Hkv, Dh) of a pair of 4-bit pools."""
    shape = k_cache.shape
    dev = k_cache.get_device()
    if (len(shape) == 4 and shape[2] == FP4_ROWS and dev >= 0 and k_cache.dtype is torch.uint8
            and k_cache.is_contiguous() and v_cache.shape == shape and v_cache.dtype is torch.uint8
            and v_cache.is_contiguous() and v_cache.get_device() == dev):
        return shape[0], shape[1], 2 * shape[3]
    _check_pool(k_cache, what)
    _check_pool(v_cache, what)
    if k_cache.dtype is not torch.uint8 or k_cache.shape[2] != FP4_ROWS:
        raise ValueError(f"{what}: 4-bit pools are uint8 [num_blocks, Hkv, {FP4_ROWS}, Dh / 2], got {k_cache.dtype} "
                         f"{tuple(k_cache.shape)}")
    if v_cache.shape != k_cache.shape or v_cache.dtype is not torch.uint8 or v_cache.device != k_cache.device:
        raise ValueError(f"{what}: k_cache and v_cache differ")
    return k_cache.shape[0], k_cache.shape[1], 2 * k_cache.shape[3]


def _check_index(t: torch.Tensor, n: int, device: torch.device, what: str, name: str) -> None:
    if t.dtype is not torch.long or t.shape != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: {name} must be a contiguous int64 [{n}] tensor on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def kv_append_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, k: torch.Tensor,
                  v: torch.Tensor, err: torch.Tensor | None = None) -> None:
    """`kv_append` into 4-bit pools: rows k[i] / v[i] (float32, float16 or bfloat16, strided views allowed) are
    rounded to e2m1 codes with a scale for each 32 dims (mlb_kv_append_fp4) and stored at slot_mapping[i].  Slots
    must be distinct."""
    what = "kv_append_fp4"
    nb, hkv, dh = _check_fp4_pools(k_cache, v_cache, what)
    dev, shape, ks, vs, code = k_cache.get_device(), k.shape, k.stride(), v.stride(), DTYPE_CODE.get(k.dtype)
    if not (len(shape) == 3 and shape[1] == hkv and shape[2] == dh and v.shape == shape and ks[2] == 1 and vs[2] == 1
            and code is not None and v.dtype is k.dtype and k.get_device() == dev and v.get_device() == dev
            and slot_mapping.dtype is torch.long and slot_mapping.shape == shape[:1] and slot_mapping.is_contiguous()
            and slot_mapping.get_device() == dev):
        _check_rows(k, hkv, dh, f"{what} k")
        _check_rows(v, hkv, dh, f"{what} v")
        if v.shape[0] != shape[0] or k.dtype != v.dtype:
            raise ValueError(f"{what}: k and v differ ({tuple(k.shape)} {k.dtype}, {tuple(v.shape)} {v.dtype})")
        if k.device != k_cache.device or v.device != k_cache.device:
            raise ValueError(f"{what}: all tensors must be on the pools' device")
        _check_index(slot_mapping, shape[0], k_cache.device, what, "slot_mapping")
        _code(k, what)
    if shape[0]:
        _launch(_lib.KV_APPEND_FP4, what, dev, k_cache.data_ptr(), v_cache.data_ptr(), nb, slot_mapping.data_ptr(),
                k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], code, shape[0], hkv, dh, _err_adr(err, dev, what))


def kv_read_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                dtype: torch.dtype = torch.bfloat16, err: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values that 4-bit pools hold at slot_mapping: (k, v) rows [N, Hkv, Dh] of `dtype` (exact in all three).
    The same slot may be asked for more than once; a slot out of range reads as zeros."""
    what = "kv_read_fp4"
    nb, hkv, dh = _check_fp4_pools(k_cache, v_cache, what)
    if dtype not in DTYPE_CODE:
        raise ValueError(f"{what}: dtype {dtype} not supported (float32, float16, bfloat16)")
    if slot_mapping.dim() != 1:
        raise ValueError(f"{what}: slot_mapping must be 1-D")
    n = slot_mapping.shape[0]
    dev = k_cache.get_device()
    if not (slot_mapping.dtype is torch.long and slot_mapping.is_contiguous() and slot_mapping.get_device() == dev):
        _check_index(slot_mapping, n, k_cache.device, what, "slot_mapping")
    k = k_cache.new_empty((n, hkv, dh), dtype=dtype)
    v = torch.empty_like(k)
    if n:
        _launch(_lib.KV_READ_FP4, what, dev, k_cache.data_ptr(), v_cache.data_ptr(), nb, slot_mapping.data_ptr(),
                k.data_ptr(), v.data_ptr(), DTYPE_CODE[dtype], n, hkv, dh, _err_adr(err, dev, what))
    return k, v


def wide_reduction(plan: AttentionPlan) -> bool:
    """Whether a step's split rows are reduced by a CTA per (token, head) (mlb_splitk_reduce_wide) or by a warp.  Both
    launch over every token.  1000 CTAs cost 1.04 us, split or not; the warp's rows cost it 0.07 us a piece up to 32
    pieces and 0.2 us a piece above, whatever their number (us, warp / CTA, 32 heads: one row of 63 pieces 13.2 / 3.6,
    beside 255 others 13.2 / 9.3, 511 13.3 / 17.7, 8191 35 / 272; 16 rows of 30 4.2 / 3.6; 64 rows of 16 3.5 / 7.4;
    4 of 9 2.25 / 2.19; 16 rows of 131072 tokens in 16, attention and all, 387 / 385)."""
    pieces = plan.max_pieces
    return pieces > WIDE_REDUCE_PIECES and plan.num_tokens * plan.num_heads <= pieces * (128 if pieces > 32 else 32)


def attention_partials_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                           seq_lens: torch.Tensor, qo_indptr: torch.Tensor, plan: AttentionPlan,
                           workspace: Workspace, out: torch.Tensor | None = None, scale: float | None = None,
                           err: torch.Tensor | None = None, targets: OutTargets | None = None) -> torch.Tensor | None:
    """`attention_partials` over 4-bit pools: unsplit rows are final in `out` (or `targets`), split ones leave
    partial rows in `workspace` for `splitk_reduce`."""
    what = "paged_attention_fp4"
    nb, hkv, dh = _check_fp4_pools(k_cache, v_cache, what)
    dev, shape, qs, code = q.get_device(), q.shape, q.stride(), DTYPE_CODE.get(q.dtype)
    if not (len(shape) == 3 and shape[2] == dh and qs[2] == 1 and (code == _lib.MLB_F16 or code == _lib.MLB_BF16)
            and dev == k_cache.get_device() and plan.num_tokens == shape[0] and plan.num_heads == shape[1]
            and plan.num_kv_heads == hkv and block_tables.dim() == 2 and block_tables.shape[0] == plan.num_seqs
            and block_tables.shape[1] >= plan.max_blocks
            and seq_lens.shape == (plan.num_seqs,) and qo_indptr.shape == (plan.num_seqs + 1,)):
        if len(shape) != 3 or shape[2] != dh or (shape[0] and qs[2] != 1):
            raise ValueError(f"{what}: q must be [N, H, {dh}] with unit last stride, got {tuple(q.shape)}")
        if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
            raise ValueError(f"{what}: q must be float16 or bfloat16, got {q.dtype}")
        if ((plan.num_heads, plan.num_kv_heads, plan.num_tokens) != (shape[1], hkv, shape[0])
                or block_tables.dim() != 2 or block_tables.shape[0] != plan.num_seqs
                or block_tables.shape[1] < plan.max_blocks
                or tuple(seq_lens.shape) != (plan.num_seqs,) or tuple(qo_indptr.shape) != (plan.num_seqs + 1,)):
            raise ValueError(f"{what}: the plan was built for another shape")
        if q.device != k_cache.device:
            raise ValueError(f"{what}: q must be on the pools' device")
    for t, name in ((block_tables, "block_tables"), (seq_lens, "seq_lens"), (qo_indptr, "qo_indptr"),
                    (plan.units, "the plan")):
        if t.dtype is not torch.int32 or not t.is_contiguous() or t.get_device() != dev:
            raise ValueError(f"{what}: {name} must be a contiguous int32 tensor on {q.device}")
    n, h, _ = shape
    if targets is not None:
        out, o0, o1 = None, 0, 0
    else:
        if out is None:
            out, o0, o1 = torch.empty_like(q, memory_format=torch.contiguous_format), h * dh, dh
        elif out.shape != shape or out.dtype != q.dtype or out.get_device() != dev or (n and out.stride(2) != 1):
            raise ValueError(f"{what}: out must match q")
        else:
            o0, o1, _ = out.stride()
    if n == 0 or plan.num_units + plan.num_shared_units == 0:
        return out
    po = plse = None
    if plan.num_partial_rows:
        po, plse = workspace.get(plan.num_partial_rows, h, dh, q.device)
    _launch(_lib.PAGED_ATTENTION_FP4, what, dev, q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(),
            code, nb, h, hkv, dh, 1.0 / math.sqrt(dh) if scale is None else float(scale), block_tables.data_ptr(),
            block_tables.stride(0), seq_lens.data_ptr(), qo_indptr.data_ptr(), seq_lens.shape[0], plan.units.data_ptr(),
            plan.num_units, plan.shared_units.data_ptr(), plan.num_shared_units, plan.members.data_ptr(), _adr(po),
            _adr(plse), plan.num_partial_rows, _adr(out), o0, o1, 0 if targets is None else ctypes.addressof(targets),
            _err_adr(err, dev, what))
    return out


def paged_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        seq_lens: torch.Tensor, qo_indptr: torch.Tensor, plan: AttentionPlan,
                        workspace: Workspace | None = None, out: torch.Tensor | None = None,
                        scale: float | None = None, err: torch.Tensor | None = None,
                        targets: OutTargets | None = None) -> torch.Tensor | None:
    """`paged_attention` over 4-bit pools: q [N, H, Dh] float16 or bfloat16 -> [N, H, Dh] in q's dtype, the pools
    holding this step's rows already (`kv_append_fp4`).  Same metadata tensors, plan and workspace (calls that may
    overlap on the GPU need a workspace each)."""
    workspace = workspace or Workspace()
    out = attention_partials_fp4(q, k_cache, v_cache, block_tables, seq_lens, qo_indptr, plan, workspace, out, scale,
                                 err, targets)
    if plan.num_partial_rows and plan.num_tokens:
        dev = q.get_device()
        po, plse = workspace.get(plan.num_partial_rows, plan.num_heads, q.shape[2], q.device)
        _launch(_lib.SPLITK_REDUCE_WIDE if wide_reduction(plan) else _lib.SPLITK_REDUCE, "splitk_reduce", dev, po.data_ptr(),
                plse.data_ptr(), plan.num_partial_rows, plan.reduce_rows.data_ptr(), plan.reduce_chunks.data_ptr(),
                plan.tokens_per_tile, plan.num_tokens, plan.num_heads, q.shape[2], _adr(out), *_strides(out),
                DTYPE_CODE[q.dtype], 0 if targets is None else ctypes.addressof(targets))
    return out


# ---------------------------------------------------------------- norm and rotation of queries and keys


def rotary_table(num_positions: int, rot_dim: int, theta: float = 500000.0, device: torch.device | str = "cuda",
                 inv_freq: torch.Tensor | None = None) -> torch.Tensor:
    """The rotation table of `qk_norm_rope`: float32 [num_positions, rot_dim], cos of each position's rot_dim / 2
    angles, then their sin.  Angles are formed in 64 bits (position x frequency needs more than 32 at far
    positions).  `inv_freq` [rot_dim / 2] replaces theta^(-2i / rot_dim) (a model's scaled frequencies)."""
    if rot_dim <= 0 or rot_dim % 16 or num_positions <= 0:
        raise ValueError(f"rotary_table: rot_dim {rot_dim} must be a positive multiple of 16, num_positions "
                         f"{num_positions} positive")
    if inv_freq is None:
        inv_freq = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    elif inv_freq.shape != (rot_dim // 2,):
        raise ValueError(f"rotary_table: inv_freq must be [{rot_dim // 2}], got {tuple(inv_freq.shape)}")
    inv = inv_freq.to(device=device, dtype=torch.float64)
    angle = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


@dataclass
class Rotary:
    """What a layer does to its queries and keys before attention: the table, and the weights of the norms of the
    query and key heads (None: no norm)."""

    cos_sin: torch.Tensor
    q_weight: torch.Tensor | None = None
    k_weight: torch.Tensor | None = None
    eps: float = 1e-6


def _check_rope(what: str, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                q_weight: torch.Tensor | None, k_weight: torch.Tensor | None) -> tuple:
    """(dtype code, q's shape, KV heads, device ordinal, q's strides, k's strides)"""
    qs, dt, dev, code = q.shape, q.dtype, q.get_device(), DTYPE_CODE.get(q.dtype)
    ks, q_st, k_st = k.shape, q.stride(), k.stride()
    if (len(qs) == 3 and len(ks) == 3 and qs[0] == ks[0] and qs[2] == ks[2] and qs[2] in (64, 128, 256)
            and q_st[2] == 1 and k_st[2] == 1 and code is not None and k.dtype is dt and dev >= 0
            and k.get_device() == dev and positions.dtype is torch.long and positions.shape == qs[:1]
            and positions.is_contiguous() and positions.get_device() == dev and cos_sin.dtype is torch.float32
            and cos_sin.dim() == 2 and cos_sin.is_contiguous() and cos_sin.get_device() == dev
            and (q_weight is None or (q_weight.shape == qs[2:] and q_weight.dtype is dt and q_weight.is_contiguous()
                                      and q_weight.get_device() == dev))
            and (k_weight is None or (k_weight.shape == qs[2:] and k_weight.dtype is dt and k_weight.is_contiguous()
                                      and k_weight.get_device() == dev))):
        return code, qs, ks[1], dev, q_st, k_st
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{what}: q must be [N, H, Dh] and k [N, Hkv, Dh], got {tuple(q.shape)}, {tuple(k.shape)}")
    dh = q.shape[2]
    _check_rows(q, q.shape[1], dh, what)
    _check_rows(k, k.shape[1], dh, what)
    if q.dtype != k.dtype or q.device != k.device or not q.is_cuda:
        raise ValueError(f"{what}: q and k must be CUDA tensors of one dtype on one device")
    if dh not in (64, 128, 256):
        raise ValueError(f"{what}: head_dim {dh} (supported: 64, 128, 256)")
    _check_index(positions, q.shape[0], q.device, what, "positions")
    if (cos_sin.dtype is not torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous()
            or cos_sin.device != q.device):
        raise ValueError(f"{what}: cos_sin must be a contiguous float32 [num_positions, rot_dim] tensor on {q.device}")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.shape != (dh,) or w.dtype != q.dtype or w.device != q.device or not w.is_contiguous()):
            raise ValueError(f"{what}: {name} must be a contiguous [{dh}] tensor of q's dtype on {q.device}")
    return _code(q, what), qs, ks[1], dev, q_st, k_st


def _check_row_out(what: str, out: torch.Tensor, x: torch.Tensor) -> None:
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{what}: out must match its input, got {tuple(out.shape)} {out.dtype} on {out.device}")
    if out.numel() == 0:
        return
    n, h, dh = out.shape
    a, b = sorted([(out.stride(0), n), (out.stride(1), h)])
    if out.stride(2) != 1 or (a[1] > 1 and a[0] < dh) or (b[1] > 1 and b[0] < max(a[0] * (a[1] - 1), 0) + dh):
        raise ValueError(f"{what}: out rows must not overlap, got strides {out.stride()}")
    if out.data_ptr() == x.data_ptr() and out.stride() != x.stride():
        raise ValueError(f"{what}: out on the memory of its input must have its strides")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 out: tuple[torch.Tensor, torch.Tensor] | None = None,
                 err: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm of each query and key head (weights [Dh] of q's dtype; None: no norm) and their rotation by position,
    one launch (mlb_qk_norm_rope): q [N, H, Dh], k [N, Hkv, Dh] -> the same shapes and dtype, computed in fp32.
    q and k may be views of a fused projection.  positions int64 [N] (AttentionMetadata.positions); cos_sin from
    `rotary_table`, its rot_dim at most Dh (the dims behind it are not rotated).  out = (q_out, k_out) may be
    (q, k), else memory that overlaps neither.  Rows whose position is outside the table are left unwritten (and
    flagged in err): without `out` they hold no values, and must not be appended or attended."""
    what = "qk_norm_rope"
    code, (n, h, dh), hkv, dev, qs, ks = _check_rope(what, q, k, positions, cos_sin, q_weight, k_weight)
    if out is None:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        qos, kos = (h * dh, dh), (hkv * dh, dh)
    else:
        qo, ko = out
        _check_row_out(what, qo, q)
        _check_row_out(what, ko, k)
        qos, kos = qo.stride(), ko.stride()
    rows, rot = cos_sin.shape
    _launch(_lib.QK_NORM_ROPE, what, dev, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], code,
            n, h, hkv, dh, positions.data_ptr(), cos_sin.data_ptr(), rows, rot, _adr(q_weight), _adr(k_weight),
            eps, qo.data_ptr(), qos[0], qos[1], ko.data_ptr(), kos[0], kos[1], _err_adr(err, dev, what))
    return qo, ko


def qk_norm_rope_append_fp4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                            cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                            slot_mapping: torch.Tensor, q_weight: torch.Tensor | None = None,
                            k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                            out: torch.Tensor | None = None, err: torch.Tensor | None = None) -> torch.Tensor:
    """`qk_norm_rope` and `kv_append_fp4` of its keys and of v in one launch: the cache and the returned queries are
    bit-identical to the two calls'.  cos_sin must rotate the whole head (rot_dim == Dh).  out may be q, else memory
    that overlaps none of the inputs.  A token whose position is outside the table is neither stored nor returned."""
    what = "qk_norm_rope_append_fp4"
    nb, hkv, dh = _check_fp4_pools(k_cache, v_cache, what)
    code, (n, h, q_dh), k_heads, dev, qs, ks = _check_rope(what, q, k, positions, cos_sin, q_weight, k_weight)
    vs = v.stride()
    if not (k_heads == hkv and q_dh == dh and v.shape == (n, hkv, dh) and vs[2] == 1 and v.dtype is k.dtype
            and v.get_device() == dev and k_cache.get_device() == dev and slot_mapping.dtype is torch.long
            and slot_mapping.shape == (n,) and slot_mapping.is_contiguous() and slot_mapping.get_device() == dev):
        _check_rows(k, hkv, dh, f"{what} k")
        _check_rows(v, hkv, dh, f"{what} v")
        if v.shape[0] != n or v.dtype != k.dtype or v.device != k.device or k_cache.device != k.device:
            raise ValueError(f"{what}: q, k, v and the pools must agree in rows, dtype and device")
        _check_index(slot_mapping, n, q.device, what, "slot_mapping")
    if out is None:
        out, os = torch.empty_like(q, memory_format=torch.contiguous_format), (h * dh, dh)
    else:
        _check_row_out(what, out, q)
        os = out.stride()
    rows, rot = cos_sin.shape
    _launch(_lib.QK_NORM_ROPE_APPEND_FP4, what, dev, q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1],
            v.data_ptr(), vs[0], vs[1], code, n, h, hkv, dh, positions.data_ptr(), cos_sin.data_ptr(), rows, rot,
            _adr(q_weight), _adr(k_weight), eps, out.data_ptr(), os[0], os[1], k_cache.data_ptr(), v_cache.data_ptr(), nb,
            slot_mapping.data_ptr(), _err_adr(err, dev, what))
    return out


# ---------------------------------------------------------------- metadata expansion on the device


def build_metadata(upload: torch.Tensor, num_ids: int, num_seqs: int, num_tokens: int, num_pages: int, width: int,
                   block_size: int, out64: torch.Tensor, out32: torch.Tensor) -> None:
    """mlb_build_metadata: expand a step's compact int64 upload (block ids, ids_indptr, qo_indptr, seq_lens,
    kv_indptr, kv_last_page_len) into the two buffers AttentionMetadata's device tensors view
    (metadata.py:71-103's arrays, computed on the GPU)."""
    s = num_seqs
    need = {"upload": (upload, torch.long, num_ids + 5 * s + 3),
            "out64": (out64, torch.long, 2 * num_tokens + s * width + s),
            "out32": (out32, torch.int32, s * width + 4 * s + 2 + num_pages)}
    for name, (t, dt, n) in need.items():
        if t.dtype != dt or not t.is_contiguous() or not t.is_cuda or t.device != upload.device or t.numel() < n:
            raise ValueError(f"build_metadata: {name} must be a contiguous {dt} CUDA tensor of >= {n} elements")
    rc = lib().mlb_build_metadata(upload.data_ptr(), num_ids, s, num_tokens, num_pages, width, block_size,
                                  out64.data_ptr(), out32.data_ptr(), _stream(upload.device))
    check(rc, "build_metadata")


# ---------------------------------------------------------------- K3: block copy


def pool_pointer_table(pools: list[torch.Tensor]) -> torch.Tensor:
    """Device int64 array of pool base addresses (every layer's K and V), the block copy's `pools`."""
    if not pools:
        raise ValueError("block_copy: no pools")
    first = pools[0]
    for p in pools:
        _check_pool(p, "block_copy")
        if p.shape != first.shape or p.dtype != first.dtype or p.device != first.device:
            raise ValueError("block_copy: every pool must have the same shape, dtype and device")
    ptrs = torch.tensor([p.data_ptr() for p in pools], dtype=torch.int64)
    return ptrs.to(first.device)


def block_copy(pool_ptrs: torch.Tensor, template: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               err: torch.Tensor | None = None) -> None:
    """pool[dst[i]] = pool[src[i]] for every pool in `pool_ptrs` (see `pool_pointer_table`); `template` is
    any one of the pools (it fixes num_blocks and the block size in bytes).  src / dst: device int32."""
    if src.shape != dst.shape or src.dim() != 1:
        raise ValueError("block_copy: src and dst must be 1-D and of equal length")
    for t, name in ((src, "src"), (dst, "dst")):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != template.device:
            raise ValueError(f"block_copy: {name} must be a contiguous int32 tensor on {template.device}")
    if src.numel() == 0:
        return
    nb = template.shape[0]
    block_bytes = template[0].numel() * template.element_size()
    rc = lib().mlb_block_copy(pool_ptrs.data_ptr(), pool_ptrs.numel(), nb, block_bytes, src.data_ptr(),
                              dst.data_ptr(), src.numel(), _ptr(err), _stream(template.device))
    check(rc, "block_copy")
