"""Batched speculative verify on CUDA: drop-in for ``deltanet_bm`` / ``SpecPools`` of the reference's ``qwen35/batch_spec.py``
and for the snapshot / rollback protocol around them (qwen35/spec.py:37-65).

Snapshot pools (batch_spec.py:16-22):
  ssm  : n_linear x [NS+1, M, 16,128,128] fp32   snapshot j = state after the j-th token of the sequence's last verify; a round
                                                 starts from snapshot ``sel`` and overwrites all M snapshots in place
  conv : n_linear x [(NS+1)*2, M, 3, 6144] bf16  double buffered: a round reads buffer ``par`` and writes the other one
  entry NS is the trash entry of padded rows.
Rollback after a verify is an index choice: the next round passes ``sel = n_new``, nothing is copied.
"""
from __future__ import annotations

from array import array

import torch

from . import _lib
from ._lib import check, on_device, ptr, raw_stream, require_same_device, stream_ptr
from .batch import CD, DK, DV, HV, PW, blit
from .config import Cfg
from .gated_delta import _f32
from .kernels import _rows


def deltanet_bm(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, sslots, sels, pars, M):
    """proj [B*M, 8224] bf16 (row b*M+j = token j of sequence b); sslots / sels / pars int32 [B]: the sequence's entry in the snapshot
    pools, the snapshot it starts from, and the conv buffer it reads.  Returns y [B*M, 2048] bf16; writes snapshots 0..M-1 of
    ssm_pool[sslot] and conv buffer par^1 IN PLACE (batch_spec.py:142-150)."""
    _lib.require_cuda(proj, conv_pool, conv_w, ssm_pool, sslots, sels, pars)
    proj, stride = _rows(proj)
    B = sslots.shape[0]
    assert proj.shape[0] == B * M, (proj.shape, B, M)
    assert ssm_pool.dtype == torch.float32 and ssm_pool.is_contiguous() and ssm_pool.shape[1] == M
    assert conv_pool.dtype == torch.bfloat16 and conv_pool.is_contiguous() and conv_pool.shape[1] == M
    assert sslots.dtype == torch.int32 and sels.dtype == torch.int32 and pars.dtype == torch.int32
    y = torch.empty((B * M, HV * DV), dtype=torch.bfloat16, device=proj.device)
    cw = conv_w.to(torch.bfloat16).reshape(-1).contiguous()
    check(_lib.load().gdn_deltanet_bm(ptr(proj), stride, ptr(conv_pool), ptr(cw), ptr(_f32(A_log)), ptr(_f32(dt_bias)), ptr(ssm_pool),
                                      ptr(sslots), ptr(sels), ptr(pars), ssm_pool.shape[0], ptr(y), B, M, stream_ptr(proj.device)), "deltanet_bm")
    return y


def accept_length(toks, ids):
    """n_new [B] int32 = number of leading drafts that the verify confirmed: sum(cumprod(toks[:, 1:] == ids[:, :k]))
    (spec.py:60-61, batch_spec.py:380-381).  The result is the next round's ``sel``."""
    k = toks.shape[1] - 1
    eq = (toks[:, 1:] == ids[:, :k]).to(torch.int32)
    return torch.cumprod(eq, dim=1).sum(dim=1).to(torch.int32)


def accept_tree(parents, toks, ids):
    """The path of a tree that the target confirms, found on the device (``accept_length`` for trees): from the first root, as long as
    there is one, to the lowest-numbered child whose token the target chose after its parent.  The root is the token that the last round
    confirmed; other roots and what hangs below them are never on the path (nothing here says what the target chose before them).

    parents int32 [B, N] as for ``attn_tree``, N <= 64; toks int32 [B, N] the nodes' tokens (those of roots are taken as confirmed); ids
    int32 [B, N] the target's token after every node.  Returns n_path int32 [B] and path int32 [B, N] (the path's nodes in order, then
    -1): what ``deltanet_commit`` and ``compact_rows`` take.  The round's next token is ids[b, path[b, n_path[b] - 1]]."""
    dev = require_same_device(parents, toks, ids)
    shape = parents.shape
    for t in (parents, toks, ids):
        if t.dtype != torch.int32 or not t.is_contiguous() or len(shape) != 2 or t.shape != shape:
            raise ValueError("accept_tree: parents, toks and ids must be contiguous int32 [B, N]")
    B, N = shape
    if not 1 <= N <= 64:
        raise ValueError(f"accept_tree: 1 <= N <= 64 nodes, got {N}")
    path = torch.empty_like(parents)
    n_path = parents.new_empty((B,))
    with on_device(dev):
        check(_lib.load().gdn_tree_accept(parents.data_ptr(), toks.data_ptr(), ids.data_ptr(), path.data_ptr(), n_path.data_ptr(), B, N, raw_stream(dev)), "accept_tree")
    return n_path, path


def deltanet_tree(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents, out=None):
    """Speculative verify of a TREE of drafted tokens on slot pools (no counterpart in the reference, whose ``deltanet_bm`` verifies a
    chain and writes a state snapshot after every token).  Nothing in the pools changes: ``deltanet_commit`` advances them along the
    path that was accepted.

    proj [B*N, 8224] bf16 (row b*N+i = node i of sequence b, row stride a multiple of 4 elements); parents int32 [B, N] as for
    ``attn_tree``, N <= 64; conv_pool, ssm_pool, slots, pos as for ``deltanet_b``.  Node i continues the conv window and the state that
    its parent leaves.  Returns y [B*N, 2048] bf16; rows of unused nodes are zero.  Conv, silu, norms, gates and the solve are
    computed in fp32; the operands of tensor-core products are sums of two bf16 numbers (what is left out is 2^-16 of the factors); y is rounded once.
    The chained kernels round to bf16 after each step, so the two agree to bf16 rounding."""
    dev = require_same_device(proj, conv_pool, conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents, out)
    if proj.dtype != torch.bfloat16 or proj.dim() != 2 or proj.shape[1] < PW or proj.stride(1) != 1:
        raise ValueError(f"deltanet_tree: proj must be bf16 [rows, >= 8224] with unit inner stride, got {tuple(proj.shape)} {proj.dtype}")
    stride = proj.stride(0)
    if parents.dtype != torch.int32 or parents.dim() != 2 or not parents.is_contiguous():
        raise ValueError("deltanet_tree: parents must be contiguous int32 [B, N]")
    B, N = parents.shape
    _check_pools("deltanet_tree", conv_pool, ssm_pool)
    _check_index("deltanet_tree", B, slots=slots, pos=pos)
    if not 1 <= N <= 64 or proj.shape[0] != B * N or stride % 4:
        raise ValueError(f"deltanet_tree: 1 <= N <= 64 nodes and proj [B*N, 8224] with a row stride that is a multiple of 4 expected (B={B}, N={N}, proj {tuple(proj.shape)}, stride {stride})")
    if out is None:
        out = ssm_pool.new_empty((B * N, HV * DV), dtype=torch.bfloat16)
    elif out.dtype != torch.bfloat16 or not out.is_contiguous() or tuple(out.shape) != (B * N, HV * DV):
        raise ValueError("deltanet_tree: out must be contiguous bf16 [B*N, 2048]")
    cw = conv_w if conv_w.dtype == torch.bfloat16 and conv_w.is_contiguous() else conv_w.to(torch.bfloat16).contiguous()
    if cw.numel() != CD * 4 or A_log.numel() != HV or dt_bias.numel() != HV:
        raise ValueError(f"deltanet_tree: conv_w [6144*4], A_log [16] and dt_bias [16] expected, got {tuple(conv_w.shape)}, {tuple(A_log.shape)}, {tuple(dt_bias.shape)}")
    A_log, dt_bias = _f32(A_log), _f32(dt_bias)
    with on_device(dev):
        check(_lib.load().gdn_tree_verify(proj.data_ptr(), stride, conv_pool.data_ptr(), cw.data_ptr(), A_log.data_ptr(), dt_bias.data_ptr(), ssm_pool.data_ptr(),
                                          slots.data_ptr(), pos.data_ptr(), parents.data_ptr(), ssm_pool.shape[0], out.data_ptr(), B, N, raw_stream(dev)), "deltanet_tree")
    return out


def _check_pools(who, conv_pool, ssm_pool):
    if ssm_pool.dtype != torch.float32 or not ssm_pool.is_contiguous() or ssm_pool.shape[1:] != (HV, DV, DK) or conv_pool.dtype != torch.bfloat16 \
            or not conv_pool.is_contiguous() or conv_pool.shape != (2 * ssm_pool.shape[0], 3, CD):
        raise ValueError(f"{who}: contiguous slot pools ssm fp32 [S, 16, 128, 128] and conv bf16 [2 S, 3, 6144] expected, got {tuple(ssm_pool.shape)} and {tuple(conv_pool.shape)}")


def _check_index(who, B, **arrays):
    for name, t in arrays.items():
        if t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be contiguous int32 [{B}]")


def _layers(who, name, x, L, ptrs, contiguous=True):
    """Appends the device pointers of the layers of ``x`` -- a sequence of L tensors of one layout, or one tensor with a leading layer
    dimension -- to ``ptrs``; returns a layer's (shape, strides, dtype, device)."""
    if isinstance(x, torch.Tensor):
        if x.dim() < 2 or x.shape[0] != L:
            raise ValueError(f"{who}: {name} {tuple(x.shape)} for {L} layers")
        shape, strides = x.shape[1:], x.stride()
        step, p = strides[0] * x.element_size(), x.data_ptr()
        if step:
            ptrs.extend(range(p, p + step * L, step))
        else:
            ptrs.extend([p] * L)
        strides, dtype, device = strides[1:], x.dtype, x.device
        flat = x.is_contiguous() if contiguous else True
    else:
        if len(x) != L:
            raise ValueError(f"{who}: {len(x)} {name} for {L} layers")
        first = x[0]
        shape, strides, dtype, device = first.shape, first.stride(), first.dtype, first.device
        for t in x:
            if t.shape != shape or t.stride() != strides or t.dtype != dtype or t.device != device:
                raise ValueError(f"{who}: the layers of {name} must have one shape, type, layout and device")
            ptrs.append(t.data_ptr())
        flat = first.is_contiguous() if contiguous else True
    if not flat:
        raise ValueError(f"{who}: {name} must be contiguous")
    return shape, strides, dtype, device


def deltanet_commit(projs, conv_pools, conv_ws, A_logs, dt_biases, ssm_pools, slots, pos, path, n_path, dst_slots=None):
    """Advances the recurrent state and the conv window of every GatedDeltaNet layer along an accepted path, in one launch (no
    counterpart in the reference).  Per layer, as a sequence of tensors or as one tensor with a leading layer dimension:
    projs [B*N, 8224] bf16 (what ``deltanet_tree`` was called with), conv_pools / ssm_pools (slot pools), conv_ws bf16, A_logs and
    dt_biases fp32.  slots, pos int32 [B]; path int32 [B, E], n_path int32 [B] from ``accept_tree`` (E may be smaller than N if no path is
    longer).  The state after the path goes to slot dst_slots[b] (default: in place), the window to its buffer (pos + n_path) & 1.
    n_path = 0 leaves a slot as it is (or copies it to its destination).  A sequence with a bad index is skipped, and so are sequences of
    which one writes a slot that another reads or writes; ``_lib.device_status()`` reports it.  The pools' last slot is exempt: it takes the
    padding of a batch, and what it holds afterwards is unspecified."""
    who, L = "deltanet_commit", len(ssm_pools)
    if L == 0:
        raise ValueError(f"{who}: no layers")
    ptrs = array("Q")
    row, strides, dtype, _ = proj = _layers(who, "projs", projs, L, ptrs, contiguous=False)
    conv, weights, a_log, dt_bias, ssm = (_layers(who, name, x, L, ptrs) for name, x in (("conv_pools", conv_pools), ("conv_ws", conv_ws), ("A_logs", A_logs),
                                                                                           ("dt_biases", dt_biases), ("ssm_pools", ssm_pools)))
    if dtype != torch.bfloat16 or len(row) != 2 or row[1] < PW or strides[1] != 1:
        raise ValueError(f"{who}: proj must be bf16 [rows, >= 8224] with unit inner stride, got {tuple(row)} {dtype}")
    n_slots = ssm[0][0]
    if ssm[2] != torch.float32 or ssm[0][1:] != (HV, DV, DK) or conv[2] != torch.bfloat16 or conv[0] != (2 * n_slots, 3, CD):
        raise ValueError(f"{who}: slot pools ssm fp32 [S, 16, 128, 128] and conv bf16 [2 S, 3, 6144] expected, got {tuple(ssm[0])} and {tuple(conv[0])}")
    if weights[2] != torch.bfloat16 or weights[0].numel() != CD * 4 or any(x[2] != torch.float32 or x[0].numel() != HV for x in (a_log, dt_bias)):
        raise ValueError(f"{who}: conv_ws bf16 [6144*4], A_logs and dt_biases fp32 [16] per layer expected")
    dst_slots = slots if dst_slots is None else dst_slots
    dev = require_same_device(slots, pos, path, n_path, dst_slots)
    if any(x[3] != dev for x in (proj, conv, weights, a_log, dt_bias, ssm)):
        raise ValueError(f"{who}: tensors on different devices in one call")
    if path.dtype != torch.int32 or path.dim() != 2 or not path.is_contiguous():
        raise ValueError(f"{who}: path must be contiguous int32 [B, E]")
    B, E = path.shape
    _check_index(who, B, slots=slots, pos=pos, n_path=n_path, dst_slots=dst_slots)
    N = row[0] // B if B else 1
    if B and (N < 1 or row[0] != B * N):
        raise ValueError(f"{who}: proj has {row[0]} rows for {B} sequences")
    for name, at in (("conv", L), ("ssm", 5 * L)):                   # (written: the layers run side by side)
        if L > 1 and len(set(ptrs[at:at + L])) < L:
            raise ValueError(f"{who}: one {name} pool for two layers")
    base = ptrs.buffer_info()[0]
    at = [base + 8 * L * i for i in range(6)]
    with on_device(dev):
        check(_lib.load().gdn_tree_commit(at[0], strides[0], *at[1:], L, slots.data_ptr(), dst_slots.data_ptr(), pos.data_ptr(), path.data_ptr(), n_path.data_ptr(),
                                          n_slots, B, N, E, raw_stream(dev)), who)


class SpecPools:
    """Recurrent snapshot pools of the sequences in speculative mode, the MTP layer's K/V pool and the round carry
    (batch_spec.py:242-270)."""

    def __init__(self, cfg: Cfg, nspec: int, nslots: int, M: int, max_len: int, device="cuda"):
        self.cfg, self.NS, self.M, self.Lmax = cfg, nspec, M, max_len
        nl = cfg.n_linear
        z = lambda shape, dt: torch.zeros(shape, dtype=dt, device=device)
        self.conv = [z(((nspec + 1) * 2, M, 3, CD), torch.bfloat16) for _ in range(nl)]
        self.ssm = [z((nspec + 1, M, HV, DV, DK), torch.float32) for _ in range(nl)]
        self.mK = z((nslots + 1, cfg.n_kv, max_len, cfg.head_dim), torch.bfloat16)
        self.mV = z((nslots + 1, cfg.n_kv, max_len, cfg.head_dim), torch.bfloat16)
        self.hist = z((nslots + 1, max_len, cfg.hidden), torch.bfloat16)
        self.carry = dict(H=z((nspec + 1, M, cfg.hidden), torch.bfloat16), toks=z((nspec + 1, M), torch.int32),
                          ids=z((nspec + 1, M), torch.int32), pos=z((nspec + 1,), torch.int32), sel=z((nspec + 1,), torch.int32))

    def as_tree(self):
        return {"conv": self.conv, "ssm": self.ssm, "mK": self.mK, "mV": self.mV}

    @staticmethod
    def entry_bytes(cfg: Cfg, M: int):
        return cfg.n_linear * M * (HV * DV * DK * 4 + 2 * 3 * CD * 2)

    @staticmethod
    def mtp_bytes(cfg: Cfg, max_len: int):
        """Per main slot: the MTP layer's K / V rows + the hidden-state history."""
        return 2 * cfg.n_kv * max_len * cfg.head_dim * 2 + max_len * cfg.hidden * 2

    # ---- moves between the plain pools and the snapshot pools (qwen35/serve.py:310-348) ----
    def enter(self, pools, slot: int, entry: int, pos: int):
        """plain -> spec: the slot's state becomes snapshot 0 / conv buffer 0 of ``entry``; the caller sets sel = 0, par = 0."""
        M = self.M
        par = pos & 1
        for i in range(len(self.ssm)):
            blit(self.ssm[i], pools.ssm[i], HV * DV * DK, entry * M * HV * DV * DK, slot * HV * DV * DK)
            blit(self.conv[i], pools.conv[i], 3 * CD, (entry * 2 + 0) * M * 3 * CD, (slot * 2 + par) * 3 * CD)

    def leave(self, pools, slot: int, entry: int, sel: int, par: int, pos: int):
        """spec -> plain: snapshot ``sel`` of ``entry`` (conv buffer ``par``) goes back into the slot, valid after ``pos`` tokens."""
        M = self.M
        for i in range(len(self.ssm)):
            blit(pools.ssm[i], self.ssm[i], HV * DV * DK, slot * HV * DV * DK, (entry * M + sel) * HV * DV * DK)
            blit(pools.conv[i], self.conv[i], 3 * CD, (slot * 2 + (pos & 1)) * 3 * CD, ((entry * 2 + par) * M + sel) * 3 * CD)
