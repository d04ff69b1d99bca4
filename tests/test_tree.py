"""CPU: the tree oracle against the chained oracle's rule and plain softmax, refusals of the C entry points before any launch, and the host
logic of page forks."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import gdn_oracle as orc, tree_oracle as tree
from qwen_tailor_b200 import Cfg, _lib
from qwen_tailor_b200.paged_pools import PagedPools
from qwen_tailor_b200.prefix_cache import PagePool

ONE = ctypes.c_void_p(16)


def test_lines_of_a_tree():
    assert tree.lines([-1, 0, 0, 2, -1, 4]) == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5]]
    assert tree.lines([-1, -2, 1, 0, 3, 9, -7]) == [[0], [], [], [0, 3], [0, 3, 4], [], []], "below an unused node, or not after its parent: unused"


def test_tree_rule_is_the_sequential_rule_on_a_chain():
    """Along a chain the tree oracle is gated_delta_rule on the same unrounded q, k, v, g, beta."""
    rng = np.random.default_rng(0)
    N = 5
    proj, window = rng.standard_normal((N, 8224)), rng.standard_normal((3, 6144))
    conv_w, A_log, dtb = rng.standard_normal(6144 * 4) * 0.5, rng.uniform(0, 2, 16), rng.standard_normal(16) * 0.1
    S0 = rng.standard_normal((16, 128, 128)) * 0.1
    rows = np.concatenate([window, proj[:, :6144]])
    tok = [tree.token(rows[j:j + 4], conv_w, proj[j, 8208:8224], proj[j, 8192:8208], A_log, dtb) for j in range(N)]
    y, S = orc.gated_delta_rule(*(np.stack([t[i] for t in tok]) for i in range(5)), S0)
    got = tree.deltanet_tree(proj, window, conv_w, A_log, dtb, S0, np.arange(N) - 1)
    assert np.allclose(got, y.reshape(N, -1), atol=1e-12)
    S1, w1 = tree.commit(proj, window, conv_w, A_log, dtb, S0, range(N))
    assert np.allclose(S1, S, atol=1e-12) and np.array_equal(w1, rows[-3:])


def test_accept_walks_the_lowest_matching_child():
    parents = np.array([-1, 0, 0, 2, 2, 3, -1, 6])
    ids = np.array([7, 0, 8, 5, 0, 1, 7, 7])
    assert tree.accept(parents, np.array([1, 9, 7, 8, 8, 5, 1, 7]), ids) == [0, 2, 3, 5]
    assert tree.accept(parents, np.array([1, 9, 9, 8, 8, 5, 1, 7]), ids) == [0]
    assert tree.accept([-2, -2], [0, 0], [0, 0]) == []


def test_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    p2 = (ctypes.c_void_p * 2)(16, 16)
    i2 = (ctypes.c_int * 2)(0, 1)
    attn = lambda B=1, N=4, H=8, KV=2, ws=1 << 40, q=ONE: lib.gqa_tree_attn(q, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ws, B, N, H, KV, 16, 1, 1, None)  # noqa: E731
    assert attn(N=65) == -1 and attn(N=0) == -1 and attn(H=9) == -1 and attn(H=34) == -1 and attn(KV=0) == -1
    assert attn(ws=0) == -1 and b"workspace" in lib.gdn_last_error_string()
    assert attn(q=None) == -8 and attn(q=ctypes.c_void_p(8)) == -3
    assert attn(B=0) == 0
    assert lib.gqa_tree_attn_workspace_bytes(4, 16, 8, 2) > 0 and lib.gqa_tree_attn_workspace_bytes(4, 16, 9, 2) == 0
    verify = lambda N=4, stride=8224, p=ONE, s=ONE: lib.gdn_tree_verify(ONE, stride, ONE, ONE, ONE, ONE, s, ONE, ONE, p, 4, ONE, 1, N, None)  # noqa: E731
    assert verify(N=65) == -1 and verify(stride=8000) == -1 and verify(stride=8225) == -1 and verify(p=None) == -8 and verify(s=ctypes.c_void_p(4)) == -3
    assert lib.gdn_tree_accept(ONE, ONE, ONE, ONE, ONE, 1, 65, None) == -1 and lib.gdn_tree_accept(ONE, None, ONE, ONE, ONE, 1, 4, None) == -8
    commit = lambda layers=2, stride=8224, B=1, slots=ONE: lib.gdn_tree_commit(p2, stride, p2, p2, p2, p2, p2, layers, slots, ONE, ONE, ONE, ONE, 4, B, 4, 4, None)  # noqa: E731
    assert commit(stride=10) == -1 and commit(slots=None) == -8 and commit(layers=0) == 0 and commit(B=0) == 0 and commit(B=-1) == -1
    compact = lambda row=512, table=ONE, B=1: lib.gdn_rows_compact(p2, 2, 4, 2, 64, row, table, ONE, 3, ONE, ONE, ONE, B, 8, None)  # noqa: E731
    assert compact(row=3) == -1 and compact(table=None) == -8 and compact(B=0) == 0
    copy = lambda n=4, sub=64, pairs=2, lens=None: lib.gdn_entries_copy(p2, 2, n, 2, sub, i2, i2, lens, pairs, None)  # noqa: E731
    assert copy(n=1) == -4 and copy(sub=3) == -1 and copy(pairs=0) == 0
    assert copy(lens=(ctypes.c_longlong * 2)(64, 66)) == -1


def test_tree_attention_refuses_tables_beyond_32_bit_positions():
    lib = _lib.load()
    attn = lambda B, KV, page_size, max_pages, q=ONE: lib.gqa_tree_attn(q, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, ONE, 1 << 40, B, 64, 16 * KV, KV, page_size, max_pages, 1, None)  # noqa: E731
    assert attn(1, 1, 1 << 20, 2048) == -7 and b"too long" in lib.gdn_last_error_string()      # 2^31 rows: positions
    assert attn(256, 8, 1 << 14, 1 << 10) == -7                      # 2^24 rows: 256 sequences x 8 heads x 8 row tiles x 2^17 key tiles
    assert attn(256, 8, 1 << 14, 1 << 9, q=None) == -8 and attn(1, 1, 1 << 14, 1 << 16, q=None) == -8      # (accepted: the next check answers)


def _pool(n_pages, page_size=8):
    return PagePool(2, n_pages, page_size, 2, 16, device="cpu")


def test_fork_shares_full_pages_and_copies_the_last():
    pool = _pool(9)
    pages = [pool.alloc() for _ in range(3)]
    for X in pool.K + pool.V:
        X.copy_(torch.randn(X.shape).bfloat16())
    before = [X.clone() for X in pool.K + pool.V]
    forks = pool.fork(pages, 19, 3)                                  # two full pages and three rows
    assert all(f[:2] == pages[:2] and len(f) == 3 for f in forks) and len({f[2] for f in forks} | {pages[2]}) == 4
    assert pool.refs[pages[0]] == 4 and pool.refs[pages[2]] == 1 and all(pool.refs[f[2]] == 1 for f in forks)
    for X, X0 in zip(pool.K + pool.V, before):
        for f in forks:
            assert torch.equal(X[f[2], :, :3], X0[pages[2], :, :3]) and torch.equal(X[f[2], :, 3:], X0[f[2], :, 3:])
        assert torch.equal(X[pages], X0[pages])
    with pytest.raises(MemoryError):
        pool.fork(pages, 19, 3)                                      # two pages left
    assert pool.refs[pages[0]] == 4 and pool.available() == 2
    assert pool.fork(pages, 16, 2) == [pages[:2]] * 2 and pool.available() == 2, "nothing is copied behind a full page"
    assert pool.fork([], 0, 2) == [[], []]
    with pytest.raises(ValueError):
        pool.fork(pages, 25, 1)
    for f in forks:
        pool.release(f)
    assert pool.available() == 5


def test_trim_gives_back_pages_behind_the_last_token():
    pools = PagedPools(Cfg(layers=4), 3, 256, page_size=8, n_pages=40, device="cpu")
    pools.reserve(1, 60)
    assert len(pools.owned[1]) == 8
    pools.advance(1, 17)
    pools.trim(1)
    assert len(pools.owned[1]) == 3 and pools.table[1, :4].tolist() == pools.owned[1] + [0]
    free = pools.pages.available()
    pools.trim(1)
    assert pools.pages.available() == free
    with pytest.raises(ValueError):
        pools.fork(1, [1])
    with pytest.raises(ValueError):
        pools.fork(1, [0, 0])
    with pytest.raises(ValueError):
        pools.fork(1, [3])                                           # the trash slot


def test_operators_run_on_cuda_tensors_only():
    from qwen_tailor_b200 import batch, batch_spec
    i = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        batch_spec.accept_tree(i, i, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        batch.copy_entries([torch.zeros(4, 8)], [1], [0])
