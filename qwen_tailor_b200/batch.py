"""Batched decode building blocks on CUDA: drop-in for the operators and pools of the reference's ``qwen35/batch.py``.

State lives in slot pools that the kernels update in place (reference layout, batch.py:1-17):
  ssm  : n_linear x [S+1, 16, 128, 128] fp32      slot s = one sequence
  conv : n_linear x [(S+1)*2, 3, 6144]  bf16      double buffered: a step reads buffer pos&1 and writes the other one
  K, V : n_full   x [S+1, 2, Lmax, 256] bf16      the attention kernel appends each sequence's new row at its position
  slot S is a trash slot that the padding rows of a bucketed batch point at.
In-place writes are ordered against later readers by CUDA stream order.
"""
from __future__ import annotations

from array import array
from math import prod
from numbers import Integral
from typing import Sequence

import torch

from . import _lib
from ._lib import check, on_device, ptr, raw_stream, require_same_device, stream_ptr
from .config import Cfg
from .gated_delta import _f32
from .kernels import _rows

HV, DK, DV, CD, PW = 16, 128, 128, 6144, 8224


def deltanet_b(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, slots, pos, out=None):
    """proj [B, 8224] bf16; slots / pos int32 [B] (pos = tokens already in the slot's state).  Returns y [B, 2048] bf16 and updates
    ssm_pool[slot] and the conv buffer (pos&1)^1 of the slot IN PLACE (batch.py:128-135).  ``out`` (optional, additive): a
    contiguous bf16 [B, 2048] tensor that receives y instead of a fresh one."""
    _lib.require_cuda(proj, conv_pool, conv_w, ssm_pool, slots, pos)
    proj, stride = _rows(proj)
    B = proj.shape[0]
    assert ssm_pool.dtype == torch.float32 and ssm_pool.is_contiguous() and conv_pool.dtype == torch.bfloat16 and conv_pool.is_contiguous()
    assert slots.dtype == torch.int32 and pos.dtype == torch.int32 and slots.numel() == B and pos.numel() == B
    if out is None:
        y = torch.empty((B, HV * DV), dtype=torch.bfloat16, device=proj.device)
    else:
        assert out.dtype == torch.bfloat16 and out.is_contiguous() and tuple(out.shape) == (B, HV * DV) and out.device == proj.device
        y = out
    cw = conv_w.to(torch.bfloat16).reshape(-1).contiguous()
    check(_lib.load().gdn_deltanet_b(ptr(proj), stride, ptr(conv_pool), ptr(cw), ptr(_f32(A_log)), ptr(_f32(dt_bias)), ptr(ssm_pool),
                                     ptr(slots), ptr(pos), ssm_pool.shape[0], ptr(y), B, stream_ptr(proj.device)), "deltanet_b")
    return y


def attn_paged(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len, M=1, max_ctx=None):
    """GQA decode attention over a paged KV cache (no counterpart in the reference, whose K/V pools are contiguous per slot).

    q [R,8,256], k_new / v_new [R,2,256] bf16 (normed + roped), R = B*M; pages [n_pages, 2, page_size, 256] bf16;
    block_table int32 [B, max_pages]; ctx_len int32 [B] = tokens already cached.  Row b*M+j attends the cached keys of sequence b
    and the new rows 0..j; the new rows are appended at ctx_len[b]+j (in place).  Returns o [R,8,256] bf16."""
    _lib.require_cuda(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len)
    R, H, D = q.shape
    n_pages, KV, page_size, _ = k_pages.shape
    if (H, KV, D) != (8, 2, 256) or not 1 <= M <= 4 or R % M:
        raise ValueError(f"attn: only 8 query heads, 2 KV heads, head_dim 256 and 1 <= M <= 4 are supported (H={H}, KV={KV}, D={D}, M={M})")
    B = R // M
    for t in (q, k_new, v_new, k_pages, v_pages):
        assert t.dtype == torch.bfloat16 and t.is_contiguous()
    assert block_table.dtype == torch.int32 and ctx_len.dtype == torch.int32 and block_table.is_contiguous()
    max_pages = block_table.shape[1]
    if max_ctx is None:
        max_ctx = max_pages * page_size
    lib = _lib.load()
    ws = torch.empty((max(lib.gqa_decode_workspace_bytes(B, max_ctx), 16) + 3) // 4, dtype=torch.float32, device=q.device)
    o = torch.empty((R, H, D), dtype=torch.bfloat16, device=q.device)
    check(lib.gqa_decode_paged(ptr(q), ptr(k_new), ptr(v_new), ptr(k_pages), ptr(v_pages), ptr(block_table), ptr(ctx_len), ptr(o), ptr(ws),
                               ws.numel() * 4, B, M, page_size, max_pages, n_pages, max_ctx, stream_ptr(q.device)), "attn")
    return o


def attn_paged_static(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len, M=1, max_ctx=None):
    """``attn_paged`` without any allocation on the way to the kernel except the output tensor: the split-KV partials go to a
    12 MiB scratch array built into the library instead of a torch workspace.  Meant for hosts that may not allocate device
    memory while serving (their C callers pass a preallocated output and use the C entry point ``gqa_decode_paged_static``
    directly).  Raises ValueError for more than 256 sequences per call (what the array is sized for).  Calls that overlap on one
    GPU share the array and must not run concurrently; the first call on a device should happen outside stream capture."""
    _lib.require_cuda(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len)
    R, H, D = q.shape
    n_pages, KV, page_size, _ = k_pages.shape
    if (H, KV, D) != (8, 2, 256) or not 1 <= M <= 4 or R % M:
        raise ValueError(f"attn: only 8 query heads, 2 KV heads, head_dim 256 and 1 <= M <= 4 are supported (H={H}, KV={KV}, D={D}, M={M})")
    B = R // M
    for t in (q, k_new, v_new, k_pages, v_pages):
        assert t.dtype == torch.bfloat16 and t.is_contiguous()
    assert block_table.dtype == torch.int32 and ctx_len.dtype == torch.int32 and block_table.is_contiguous()
    max_pages = block_table.shape[1]
    if max_ctx is None:
        max_ctx = max_pages * page_size
    o = torch.empty((R, H, D), dtype=torch.bfloat16, device=q.device)
    check(_lib.load().gqa_decode_paged_static(ptr(q), ptr(k_new), ptr(v_new), ptr(k_pages), ptr(v_pages), ptr(block_table), ptr(ctx_len), ptr(o),
                                              B, M, page_size, max_pages, n_pages, max_ctx, stream_ptr(q.device)), "attn (static scratch)")
    return o


def attn_tree(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len, parents, out=None):
    """GQA attention of a TREE of drafted tokens over a paged KV cache: the verify step of tree speculation, as ``attn_paged`` with M > 1
    is that of a chain (no counterpart in the reference).

    parents int32 [B, N], N <= 64: node i of sequence b hangs below node parents[b, i] < i; -1 = below the last cached token (a root;
    there may be several, but ``accept_tree`` only follows the first); a smaller value = an unused node.  q [B*N, H, 256], k_new / v_new [B*N, KV, 256] bf16 (normed and roped at
    position ctx_len[b] + depth of the node), pages [n_pages, KV, page_size, 256] (any page size), block_table int32 [B, max_pages],
    ctx_len int32 [B].  H is a multiple of KV, at most 16 query heads share one.
    Node i attends the cached keys of its sequence, its ancestors and itself; its k / v rows are appended at ctx_len[b] + i (in place;
    ``compact_rows`` moves the accepted ones together afterwards).  Rows of unused nodes are not appended and their output is zero.
    One node per sequence (N = 1, parents = -1) is plain decode.  Returns o [B*N, H, 256] bf16 (``out``, if given).
    A malformed tree, context or page number is reported by ``_lib.device_status()``."""
    dev = require_same_device(q, k_new, v_new, k_pages, v_pages, block_table, ctx_len, parents, out)
    for name, t in (("block_table", block_table), ("ctx_len", ctx_len), ("parents", parents)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"attn_tree: {name} must be contiguous int32")
    for t in (q, k_new, v_new, k_pages, v_pages):
        if t.dtype != torch.bfloat16 or not t.is_contiguous():
            raise ValueError("attn_tree: q, k_new, v_new and the pages must be contiguous bf16")
    if parents.dim() != 2 or q.dim() != 3 or k_pages.dim() != 4 or block_table.dim() != 2:
        raise ValueError("attn_tree: parents [B, N], q [B*N, H, 256], pages [n_pages, KV, page_size, 256] and block_table [B, max_pages] expected")
    (B, N), (R, H, D), (n_pages, KV, page_size, _) = parents.shape, q.shape, k_pages.shape
    if not 1 <= N <= 64 or D != 256 or KV < 1 or H % KV or not 1 <= H // KV <= 16:
        raise ValueError(f"attn_tree: 1 <= N <= 64 nodes, head_dim 256 and H a multiple of KV, at most 16 * KV, are supported (N={N}, H={H}, KV={KV}, D={D})")
    if R != B * N or k_new.shape != (R, KV, D) or v_new.shape != k_new.shape or v_pages.shape != k_pages.shape or k_pages.shape[3] != D \
            or block_table.shape[0] != B or ctx_len.shape != (B,):
        raise ValueError(f"attn_tree: shapes do not agree: q {tuple(q.shape)}, k_new {tuple(k_new.shape)}, v_new {tuple(v_new.shape)}, pages {tuple(k_pages.shape)} / "
                         f"{tuple(v_pages.shape)}, block_table {tuple(block_table.shape)}, ctx_len {tuple(ctx_len.shape)}, parents {tuple(parents.shape)}")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
        raise ValueError("attn_tree: out must be a contiguous bf16 tensor of q's shape")
    if B == 0:
        return out
    lib = _lib.load()
    with on_device(dev):
        size = lib.gqa_tree_attn_workspace_bytes(B, N, H, KV)
        ws = q.new_empty((size,), dtype=torch.uint8)
        check(lib.gqa_tree_attn(q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), ctx_len.data_ptr(),
                                parents.data_ptr(), out.data_ptr(), ws.data_ptr(), size, B, N, H, KV, page_size, block_table.shape[1], n_pages, raw_stream(dev)), "attn_tree")
    return out


def attn_b(q, k, v, Kp, Vp, slots, pos, M=1):
    """q [R,H,D], k / v [R,KV,D] (normed + roped), pools [S+1,KV,Lmax,D]; R = B*M rows (row b*M+j = position pos[b]+j of slot
    slots[b]; slots / pos int32 [B]).  Returns o [R,H,D] bf16 and appends k / v at pos[b]+j (in place)  (batch.py:230-237).
    The slot pool is a paged cache with one page of Lmax rows per sequence."""
    return attn_paged(q, k, v, Kp, Vp, slots.reshape(-1, 1), pos, M=M, max_ctx=Kp.shape[2])


def blit(dst, src, n, d0, s0, ny=1, dstride=0, sstride=0):
    """dst.flat[d0 + y*dstride + i] = src.flat[s0 + y*sstride + i]  for i < n, y < ny   (in place; batch.py:367-372).
    Returns dst (the reference returns a token to evaluate; stream order plays that role here)."""
    _lib.require_cuda(dst, src)
    assert dst.dtype == src.dtype and dst.dtype in (torch.bfloat16, torch.float32), (dst.dtype, src.dtype)
    assert dst.is_contiguous() and src.is_contiguous()
    assert d0 + (ny - 1) * dstride + n <= dst.numel() and s0 + (ny - 1) * sstride + n <= src.numel(), "blit out of range"
    check(_lib.load().gdn_state_copy(ptr(dst), ptr(src), dst.element_size(), n, d0, s0, ny, dstride, sstride, stream_ptr(dst.device)), "blit")
    return dst


def hrec(hist, Hn, slots, pos):
    """hist[slots[b], pos[b], :] = Hn[b]  (in place; hist [S+1, Lh, H] bf16): the hidden-state history of speculative mode
    (batch.py:375-399).  slots, pos: int32 [B] on the device; an out-of-range entry skips its row and sets the device status.
    Returns hist (the reference returns a token to evaluate; here stream order does that job)."""
    _lib.require_cuda(hist, Hn, slots, pos)
    assert hist.dtype == torch.bfloat16 and Hn.dtype == torch.bfloat16 and hist.is_contiguous() and hist.dim() == 3
    assert slots.dtype == torch.int32 and pos.dtype == torch.int32
    Hn = Hn.contiguous()
    B, H = Hn.shape
    assert hist.shape[2] == H and slots.numel() == B and pos.numel() == B
    check(_lib.load().gdn_hrec(ptr(hist), ptr(Hn), ptr(slots), ptr(pos), B, hist.shape[0], hist.shape[1], H, stream_ptr(hist.device)), "hrec")
    return hist


def _pool_ptrs(who, pools, stacked):
    """The pools of ``pools`` (each a contiguous bf16 or fp32 tensor, all of one shape; stacked: each holds several along a leading
    layer dimension) as (first tensor, shape of one pool, device pointers)."""
    if not pools:
        raise ValueError(f"{who}: no pools")
    first = pools[0]
    require_same_device(*pools)
    shape, dtype, ptrs = first.shape, first.dtype, array("Q")
    if dtype not in (torch.bfloat16, torch.float32) or len(shape) < (3 if stacked else 2) or 0 in shape[1:]:
        raise ValueError(f"{who}: pools must be non-empty bf16 or fp32 tensors, got {dtype} {tuple(shape)}")
    step = prod(shape[1:]) * first.element_size()
    for t in pools:
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{who}: pools must be contiguous tensors of one shape and type")
        p = t.data_ptr()
        if stacked:
            ptrs.extend(range(p, p + step * shape[0], step))
        else:
            ptrs.append(p)
    return first, shape[1:] if stacked else shape, ptrs


def _address(a):
    return a.buffer_info()[0]


def copy_entries(pools: Sequence[torch.Tensor], dst: Sequence[int], src: Sequence[int], rows=None, stacked=False):
    """pool[dst[i]] = pool[src[i]] for every pool and i, in place, in one launch (no counterpart in the reference, which copies layer by
    layer with ``blit``): K/V pages, recurrent states or conv windows of all layers when a sequence is forked, checkpointed or moved.

    pools: contiguous tensors [n_entries, ...] of one shape and type (bf16 or fp32); stacked=True: each has a leading layer dimension.
    dst, src: host integers.  One source may be copied to many entries; no dst may repeat or be a src (ValueError).
    rows (an int, or one per pair): only the first rows of every head of pages [n_entries, heads, page_size, dim] are copied.
    Every 512 pairs take one launch."""
    first, shape, ptrs = _pool_ptrs("copy_entries", pools, stacked)
    try:
        d, s = array("i", dst), array("i", src)
        each = None if rows is None or isinstance(rows, Integral) else array("q", rows)
    except OverflowError as e:
        raise ValueError(f"copy_entries: entries and rows are 32-bit numbers ({e})") from None
    n = len(d)
    if n != len(s):
        raise ValueError(f"copy_entries: {n} destinations for {len(s)} sources")
    if n == 0:
        return
    item, lens = first.element_size(), None
    n_sub, sub_bytes = 1, prod(shape[1:]) * item
    if rows is not None:
        if len(shape) != 4:
            raise ValueError(f"copy_entries: rows needs pools [n_entries, heads, page_size, dim], got entries of {tuple(shape[1:])}")
        row, one = shape[3] * item, each is None
        r = (int(rows),) if one else each
        if (not one and len(r) != n) or min(r) < 0 or max(r) > shape[2]:
            raise ValueError(f"copy_entries: rows must be one number or {n}, from 0 to {shape[2]}")
        n_sub, sub_bytes = shape[1], shape[2] * row
        lens = array("q", [x * row for x in r])
        if one:
            lens *= n
    dev = first.device
    with on_device(dev):
        rc = _lib.load().gdn_entries_copy(_address(ptrs), len(ptrs), shape[0], n_sub, sub_bytes, _address(d), _address(s), _address(lens) if lens is not None else None, n,
                                          raw_stream(dev))
    if rc == -4:                                                     # an entry out of range, named twice as a destination, or both source and destination
        raise ValueError(_lib.load().gdn_last_error_string().decode())
    check(rc, "copy_entries")


def compact_rows(pools: Sequence[torch.Tensor], block_table, base, keep, n_keep, dst_table=None, stacked=False):
    """Row base[b] + keep[b, j] of sequence b moves to row base[b] + j for j < n_keep[b], in every pool and head, in one launch: the K/V
    rows of an accepted path move together behind the context (base = ctx_len, keep / n_keep from ``accept_tree``), or any subset of a
    sequence's rows to its front (base = 0).  No counterpart in the reference.

    pools: page pools [n_pages, heads, page_size, dim] (bf16 or fp32; K and V of all layers), stacked=True: with a leading layer
    dimension.  block_table int32 [B, max_pages]; base, n_keep int32 [B]; keep int32 [B, L], strictly ascending.  All on the device.
    dst_table: the rows are written through this table instead (pages that the call does not read, or the same table): the
    source keeps its rows.
    The pages that rows are written to belong to one sequence: a page that another one shares (``PagePool.fork``, a checkpoint) changes
    for both, so with base = 0 only sequences of their own pages move in place, and no two sequences of a call write the same page.  One warp
    walks the rows of a sequence in a pool and head: made for the handful that a round keeps.  From the first keep entry that is out of order or range the rest of a sequence is left alone and
    ``_lib.device_status()`` reports it."""
    first, shape, ptrs = _pool_ptrs("compact_rows", pools, stacked)
    dst_table = block_table if dst_table is None else dst_table
    dev = require_same_device(first, block_table, base, keep, n_keep, dst_table)
    for name, t in (("block_table", block_table), ("dst_table", dst_table), ("base", base), ("keep", keep), ("n_keep", n_keep)):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"compact_rows: {name} must be contiguous int32")
    if len(shape) != 4 or keep.dim() != 2 or block_table.dim() != 2:
        raise ValueError("compact_rows: pools [n_pages, heads, page_size, dim], block_table [B, max_pages] and keep [B, L] expected")
    B, L = keep.shape
    if block_table.shape[0] != B or dst_table.shape != block_table.shape or base.shape != (B,) or n_keep.shape != (B,):
        raise ValueError(f"compact_rows: shapes do not agree: block_table {tuple(block_table.shape)}, dst_table {tuple(dst_table.shape)}, base {tuple(base.shape)}, "
                         f"keep {tuple(keep.shape)}, n_keep {tuple(n_keep.shape)}")
    if block_table.shape[1] == 0:
        raise ValueError("compact_rows: an empty block table")
    if len(set(ptrs)) < len(ptrs):
        raise ValueError("compact_rows: a pool is named twice (its rows would move twice)")
    n_pages, heads, page_size, dim = shape
    with on_device(dev):
        check(_lib.load().gdn_rows_compact(_address(ptrs), len(ptrs), n_pages, heads, page_size, dim * first.element_size(), block_table.data_ptr(), dst_table.data_ptr(),
                                           block_table.shape[1], base.data_ptr(), keep.data_ptr(), n_keep.data_ptr(), B, L, raw_stream(dev)), "compact_rows")


class Pools:
    """Slot pools of the batched decode step (batch.py:405-462)."""

    def __init__(self, cfg: Cfg, slots: int, max_len: int, device="cuda"):
        self.cfg, self.S, self.Lmax = cfg, slots, max_len
        nl, na = cfg.n_linear, cfg.n_full
        self.conv = [torch.zeros(((slots + 1) * 2, 3, CD), dtype=torch.bfloat16, device=device) for _ in range(nl)]
        self.ssm = [torch.zeros((slots + 1, HV, DV, DK), dtype=torch.float32, device=device) for _ in range(nl)]
        self.K = [torch.zeros((slots + 1, cfg.n_kv, max_len, cfg.head_dim), dtype=torch.bfloat16, device=device) for _ in range(na)]
        self.V = [torch.zeros((slots + 1, cfg.n_kv, max_len, cfg.head_dim), dtype=torch.bfloat16, device=device) for _ in range(na)]

    def nbytes(self):
        return sum(a.numel() * a.element_size() for g in (self.conv, self.ssm, self.K, self.V) for a in g)

    @staticmethod
    def slot_bytes(cfg: Cfg, max_len: int, double_conv=True):
        """Bytes one sequence occupies in the pools (the pools hold slots + 1 of these).  double_conv=False: a stand-alone state."""
        nl, na = cfg.n_linear, cfg.n_full
        return (nl * (HV * DV * DK * 4 + (2 if double_conv else 1) * 3 * CD * 2) + na * 2 * cfg.n_kv * max_len * cfg.head_dim * 2)

    def as_tree(self):
        return {"conv": self.conv, "ssm": self.ssm, "K": self.K, "V": self.V}

    def load(self, slot: int, state: dict, pos: int):
        """Copy a prefilled single-sequence state (kv [1,2,max_len,256] pairs, conv [1,3,6144], ssm [1,16,128,128], valid after
        ``pos`` tokens) into ``slot``, in place."""
        assert 0 <= slot < self.S and 0 < pos <= self.Lmax, (slot, pos)
        par = pos & 1
        for i, (c, s) in enumerate(zip(state["conv"], state["ssm"])):
            blit(self.conv[i], c.contiguous(), CD * 3, (slot * 2 + par) * 3 * CD, 0)
            blit(self.ssm[i], s.contiguous(), HV * DV * DK, slot * HV * DV * DK, 0)
        nkv, D = self.cfg.n_kv, self.cfg.head_dim
        for i, (K, V) in enumerate(state["kv"]):
            smax = K.shape[2]
            for pool, src in ((self.K[i], K), (self.V[i], V)):
                blit(pool, src.contiguous(), pos * D, slot * nkv * self.Lmax * D, 0, ny=nkv, dstride=self.Lmax * D, sstride=smax * D)

    def read(self, slot: int, pos: int, max_len: int | None = None):
        """The slot's state as a single-sequence state dict (fresh tensors)."""
        ml = max_len or self.Lmax
        par = pos & 1
        st = {"kv": [], "conv": [self.conv[i][slot * 2 + par][None].clone() for i in range(len(self.conv))],
              "ssm": [self.ssm[i][slot][None].clone() for i in range(len(self.ssm))]}
        for K, V in zip(self.K, self.V):
            def one(Pl):
                out = torch.zeros((1, Pl.shape[1], ml, Pl.shape[3]), dtype=Pl.dtype, device=Pl.device)
                n = min(pos, ml)
                out[0, :, :n] = Pl[slot, :, :n]
                return out
            st["kv"].append((one(K), one(V)))
        return st
