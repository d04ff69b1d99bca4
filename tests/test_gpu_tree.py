"""GPU: operators for trees of drafted tokens and the cache copies around them, against the definitions in 64 bits (oracle/tree_oracle.py)."""
import numpy as np
import pytest
import torch

from conftest import bf16_dev, f32_dev, host, i32_dev
from oracle import tree_oracle as tree
from qwen_tailor_b200 import Cfg, _lib, synth
from qwen_tailor_b200.batch import attn_paged, attn_tree, compact_rows, copy_entries
from qwen_tailor_b200.batch_spec import accept_tree, deltanet_bm, deltanet_commit, deltanet_tree
from qwen_tailor_b200.paged_pools import PagedPools
from qwen_tailor_b200.prefix_cache import PagePool
from short_waits import compile_library, operators_use

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8                # a rounding to bf16, relative to the value
# attention before that rounding: scores are fp32 sums of 256 products (|q||k| / 16 <= ~24 here; 2^-21 of that at worst is < 2^-16 in the exponent), exp and
# weights that are exact to 2^-16: together below 2^-14 of the same sums taken over |V|
ATTN_ABS = 2.0 ** -14
# y of the tree rule before its rounding: every product is exact to 2^-16 of its factors' norms; a path sums at most 64 terms weighted by |q.k| <= 0.09
DELTA_ABS = 2.0 ** -12


def random_tree(rng, N, used=None, kind="random"):
    """parents [N]; nodes from `used` on are unused."""
    used = N if used is None else used
    p = np.full(N, -2, np.int32)
    for i in range(used):
        p[i] = {"chain": i - 1, "star": -1 if i == 0 else 0, "forest": -1 if i < 3 else rng.integers(0, i), "random": -1 if i == 0 else rng.integers(0, i)}[kind]
    return p


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def attn_case(rng, ctx, N, page, H=8, KV=2, scale=1.0):
    ctx = np.asarray(ctx, np.int64)
    need = -(-(ctx + N) // page)
    total = int(need.sum()) + 1
    order = rng.permutation(total - 1) + 1
    table = np.zeros((len(ctx), int(need.max()) + 1), np.int32)
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = order[o:o + n]
        o += n
    r = lambda *s: synth.bf16r(rng.standard_normal(s) * scale)  # noqa: E731
    B = len(ctx)
    return dict(q=r(B * N, H, 256), k_new=r(B * N, KV, 256), v_new=r(B * N, KV, 256), k_pages=r(total, KV, page, 256), v_pages=r(total, KV, page, 256), table=table,
                ctx=ctx.astype(np.int32))


def to_dev(c, dev):
    return {k: i32_dev(v, dev) if v.dtype == np.int32 else bf16_dev(v, dev) for k, v in c.items()}


def run_attn(d, parents):
    return attn_tree(d["q"], d["k_new"], d["v_new"], d["k_pages"], d["v_pages"], d["table"], d["ctx"], parents)


def context(c, b, X):
    n, P = int(c["ctx"][b]), X.shape[2]
    return np.concatenate([X[p] for p in c["table"][b]], axis=1)[:, :n] if n else np.zeros((X.shape[1], 0, 256), np.float32)


def check_attn(c, parents, out, K1, V1, skip=()):
    N, P = parents.shape[1], c["k_pages"].shape[2]
    want_K, want_V = c["k_pages"].copy(), c["v_pages"].copy()
    for b in range(len(c["ctx"])):
        r = slice(b * N, (b + 1) * N)
        ref, mag = tree.attn_tree(c["q"][r], c["k_new"][r], c["v_new"][r], context(c, b, c["k_pages"]), context(c, b, c["v_pages"]), parents[b])
        err = np.abs(out[r] - ref)
        assert (err <= HALF * np.abs(ref) + ATTN_ABS * mag + 1e-30).all(), (b, float((err - HALF * np.abs(ref)).max()), float(mag.max()))
        for i, line in enumerate(tree.lines(parents[b])):
            if line:
                at = int(c["ctx"][b]) + i
                want_K[c["table"][b, at // P], :, at % P], want_V[c["table"][b, at // P], :, at % P] = c["k_new"][b * N + i], c["v_new"][b * N + i]
    assert np.array_equal(K1, want_K) and np.array_equal(V1, want_V), "only the rows of used nodes are appended"


@pytest.mark.parametrize("ctx,N,page,kind,H,KV", [
    ([0], 1, 64, "chain", 8, 2), ([1, 0, 63, 64, 65], 1, 64, "chain", 8, 2), ([700], 8, 64, "random", 8, 2), ([130, 0, 5, 64, 257], 13, 64, "forest", 8, 2),
    ([511, 1025], 16, 128, "star", 8, 2), ([300, 77, 1], 33, 64, "random", 8, 2), ([64, 191, 1000], 64, 64, "chain", 8, 2), ([1300, 64], 64, 256, "random", 8, 2),
    ([100, 47, 48, 0], 13, 48, "random", 8, 2), ([37, 90], 7, 1, "random", 8, 2), ([530, 3], 20, 37, "random", 8, 2), ([200, 64], 21, 16, "random", 8, 2),
    ([150, 300], 31, 64, "random", 16, 2), ([150, 300], 11, 64, "random", 4, 4), ([129], 40, 64, "random", 24, 4), ([333, 10], 9, 64, "random", 32, 2),
    ([90, 200], 64, 32, "random", 3, 3), ([5000, 2], 5, 64, "random", 8, 2),
])
def test_attn_tree(dev, ctx, N, page, kind, H, KV):
    rng = np.random.default_rng(N * 1000 + page)
    c = attn_case(rng, ctx, N, page, H, KV)
    parents = np.stack([random_tree(rng, N, max(1, N - (3 * b) % 5), kind) for b in range(len(ctx))])
    d = to_dev(c, dev)
    out = run_attn(d, i32_dev(parents, dev))
    assert out.shape == d["q"].shape and out.dtype == torch.bfloat16
    check_attn(c, parents, host(out), host(d["k_pages"]), host(d["v_pages"]))
    assert _lib.device_status() == 0


def test_attn_tree_peaked_scores_and_many_sequences(dev):
    """Large scores (one key takes almost all the weight, found late in the context) and more sequences than blocks."""
    rng = np.random.default_rng(5)
    ctx = rng.integers(0, 200, 90)
    c = attn_case(rng, ctx, 3, 64, scale=3.0)
    parents = np.stack([random_tree(rng, 3) for _ in ctx])
    d = to_dev(c, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    for b in range(len(ctx)):
        r = slice(b * 3, b * 3 + 3)
        ref, mag = tree.attn_tree(c["q"][r], c["k_new"][r], c["v_new"][r], context(c, b, c["k_pages"]), context(c, b, c["v_pages"]), parents[b])
        # scores nine times as large: 9 x the exponent's error, 2^-13 + 2^-16 < 2^-12 of the sums over |V|
        assert (np.abs(out[r] - ref) <= HALF * np.abs(ref) + 2.0 ** -12 * mag).all()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("B,N,page", [(80, 40, 64), (300, 3, 16)])
def test_attn_tree_more_pairs_than_blocks(dev, B, N, page):
    """80 sequences with two row tiles each (pairs are joined by the block they start in), and more sequences than one launch takes."""
    rng = np.random.default_rng(B)
    ctx = rng.integers(0, 150, B)
    ctx[[0, B // 2, B - 1]] = [600, 0, 700]
    c = attn_case(rng, ctx, N, page)
    parents = np.stack([random_tree(rng, N, max(1, N - b % 3)) for b in range(B)])
    d = to_dev(c, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    check_attn(c, parents, out, host(d["k_pages"]), host(d["v_pages"]))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("H,KV,N", [(32, 2, 64), (10, 2, 64), (24, 2, 50), (7, 1, 64), (13, 1, 37)])
def test_attn_tree_row_tiles(dev, H, KV, N):
    """Eight, three, five, four and five row tiles of a range side by side (5, 12, 7 and 13 heads on one leave rows of the tile empty)."""
    rng = np.random.default_rng(H * N)
    ctx = [140, 0, 2200]
    c = attn_case(rng, ctx, N, 64, H, KV)
    parents = np.stack([random_tree(rng, N, N - b) for b in range(3)])
    d = to_dev(c, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    check_attn(c, parents, out, host(d["k_pages"]), host(d["v_pages"]))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N", [3, 40])
def test_attn_tree_nothing_leaks_from_masked_places(dev, N):
    """NaN and infinities behind the context in its last page, in unused pages, in unused nodes and in siblings change nothing where
    they are masked; where a node does see them it gets them."""
    rng = np.random.default_rng(6)
    ctx = [70, 5, 64, 0]
    c = attn_case(rng, ctx, N, 64)
    parents = np.stack([random_tree(rng, N, N - 1, "star") for _ in ctx])
    clean = to_dev(c, dev)
    ref = host(run_attn(clean, i32_dev(parents, dev)))
    for X in (c["k_pages"], c["v_pages"]):
        X[0] = np.nan
        for b, n in enumerate(ctx):
            seen = np.zeros((c["table"].shape[1], 64), bool)
            seen.reshape(-1)[:n] = True
            for p in range(-(-(n + N) // 64)):
                X[c["table"][b, p]][:, ~seen[p]] = [np.nan, np.inf, -np.inf][b % 3]
    for b in range(4):
        c["k_new"][b * N + 1], c["v_new"][b * N + 1] = np.nan, [np.inf, np.nan][b % 2]      # node 1: a leaf of the star
        c["k_new"][b * N + N - 1], c["v_new"][b * N + N - 1] = np.inf, np.nan                   # unused
        c["q"][b * N + N - 1] = np.nan
    d = to_dev(c, dev)
    got = host(run_attn(d, i32_dev(parents, dev)))
    for b in range(4):
        for i in range(N):
            if i != 1:
                assert np.array_equal(got[b * N + i], ref[b * N + i]), (b, i)
        assert np.isnan(got[b * N + 1]).all()
        assert not got[b * N + N - 1].any()
    # a finite key with a non-finite value: exactly the dimensions of the nodes that see it
    c["k_new"][1], c["v_new"][1] = c["k_new"][0], c["v_new"][0]
    c["v_new"][1][:, 7] = np.inf
    got = host(run_attn(to_dev(c, dev), i32_dev(parents, dev)))
    assert np.isposinf(got[1][:, 7]).all() and np.isfinite(np.delete(got[1], 7, 1)).all()
    assert np.array_equal(got[0], ref[0]) and np.array_equal(got[2:N], ref[2:N])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N,H,KV", [(13, 8, 2), (40, 8, 2), (9, 24, 2)])
def test_attn_tree_rows_of_a_warp_see_different_values(dev, N, H, KV):
    """Infinities and NaN in the values of several nodes of a random tree: the rows of one warp add different numbers of them between two loads from
    tensor memory, and some of its rows are no node's.  Every output is what the definition gives, infinities with their sign."""
    rng = np.random.default_rng(N + H)
    ctx = [70, 900, 0]
    c = attn_case(rng, ctx, N, 64, H, KV)
    parents = np.stack([random_tree(rng, N, N - b) for b in range(3)])
    for b in range(3):
        for i in range(1, N, 2):
            c["v_new"][b * N + i, :, rng.integers(0, 256, 6)] = rng.choice([np.inf, -np.inf, np.nan], (6, KV))
    d = to_dev(c, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    for b in range(3):
        r = slice(b * N, (b + 1) * N)
        with np.errstate(invalid="ignore"):
            ref, mag = tree.attn_tree(c["q"][r], c["k_new"][r], c["v_new"][r], context(c, b, c["k_pages"]), context(c, b, c["v_pages"]), parents[b])
        fin = np.isfinite(ref)
        assert fin.any() and not fin.all()
        assert np.array_equal(out[r][~fin], ref[~fin].astype(np.float32), equal_nan=True)
        assert (np.abs(out[r][fin] - ref[fin]) <= HALF * np.abs(ref[fin]) + ATTN_ABS * mag[fin] + 1e-30).all()
    assert _lib.device_status() == 0


def test_attn_tree_reports_and_skips_what_is_malformed(dev):
    rng = np.random.default_rng(7)
    ctx = [40, 50, 60, 70]
    c = attn_case(rng, ctx, 6, 64)
    parents = np.stack([random_tree(rng, 6, kind="chain") for _ in ctx])
    parents[1] = [-1, 0, 5, 1, 2, 0]                                 # node 2 hangs below a later node; 4 below 2
    d = to_dev(c, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    assert _lib.device_status() == 1
    check_attn(c, parents, out, host(d["k_pages"]), host(d["v_pages"]))
    assert not out[8].any() and not out[10].any()
    # a context that does not fit its table, and a negative one: those sequences give zeros and write nothing
    parents[1] = random_tree(rng, 6)
    for bad in (c["table"].shape[1] * 64 - 5, -1, 2 ** 31 - 1):
        c2 = dict(c, ctx=np.array([40, 50, bad, 70], np.int32))
        d = to_dev(c2, dev)
        out = host(run_attn(d, i32_dev(parents, dev)))
        assert _lib.device_status() == 1
        none = parents.copy()
        none[2] = -2
        check_attn(dict(c2, ctx=np.array([40, 50, 0, 70], np.int32)), none, out, host(d["k_pages"]), host(d["v_pages"]))
    # a page number outside the pool: reported, nothing faults, the other sequences are right
    c2 = dict(c, table=c["table"].copy())
    c2["table"][3, 0] = 10 ** 6
    d = to_dev(c2, dev)
    out = host(run_attn(d, i32_dev(parents, dev)))
    assert _lib.device_status() == 1
    for b in range(3):
        r = slice(6 * b, 6 * b + 6)
        ref, mag = tree.attn_tree(c["q"][r], c["k_new"][r], c["v_new"][r], context(c, b, c["k_pages"]), context(c, b, c["v_pages"]), parents[b])
        assert (np.abs(out[r] - ref) <= HALF * np.abs(ref) + ATTN_ABS * mag).all()


def test_attn_tree_refusals(dev):
    rng = np.random.default_rng(8)
    c = attn_case(rng, [10, 20], 4, 64)
    parents = np.stack([random_tree(rng, 4)] * 2)
    d = to_dev(c, dev)
    p = i32_dev(parents, dev)
    run_attn(d, p)
    for change in (dict(q=d["q"].float()), dict(q=d["q"][:, :7]), dict(q=d["q"][:7]), dict(k_new=d["k_new"][:, :1]), dict(table=d["table"].long()), dict(ctx=d["ctx"][:1]),
                   dict(v_pages=d["v_pages"][:2]), dict(q=d["q"][..., :128].contiguous()), dict(table=d["table"][:1])):
        with pytest.raises(ValueError):
            run_attn({**d, **change}, p)
    with pytest.raises(ValueError):
        run_attn(d, p.long())
    with pytest.raises(ValueError):
        run_attn(d, torch.full((2, 65), -1, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError):
        run_attn({**d, "q": d["q"].cpu()}, p)
    with pytest.raises(ValueError):
        attn_tree(d["q"], d["k_new"], d["v_new"], d["k_pages"], d["v_pages"], d["table"], d["ctx"], p, out=d["q"].float())
    empty = attn_tree(d["q"][:0], d["k_new"][:0], d["v_new"][:0], d["k_pages"], d["v_pages"], d["table"][:0], d["ctx"][:0], p[:0])
    assert empty.shape == (0, 8, 256)


def test_attn_tree_of_a_chain_is_attn_paged(dev):
    rng = np.random.default_rng(9)
    ctx = [700, 64, 0, 129]
    c = attn_case(rng, ctx, 4, 64)
    a, b = to_dev(c, dev), to_dev(c, dev)
    got = host(run_attn(a, i32_dev(np.tile(np.arange(4) - 1, (4, 1)), dev)))
    ref = host(attn_paged(b["q"], b["k_new"], b["v_new"], b["k_pages"], b["v_pages"], b["table"], b["ctx"], M=4))
    assert np.abs(got - ref).max() <= 2 * HALF * np.abs(ref).max()                # two roundings of values of one size
    assert torch.equal(a["k_pages"], b["k_pages"]) and torch.equal(a["v_pages"], b["v_pages"])


def test_attn_tree_captured_on_other_streams_and_repeatable(dev):
    """Two captured graphs replayed in turn, a second stream, and the same bits every time."""
    rng = np.random.default_rng(10)
    cases = [(attn_case(rng, [900, 1500], 12, 64), 12), (attn_case(rng, [3000], 40, 64), 40)]
    refs, graphs, outs, devs, ps = [], [], [], [], []
    for c, N in cases:
        d, p = to_dev(c, dev), i32_dev(np.stack([random_tree(rng, N) for _ in c["ctx"]]), dev)
        refs.append(run_attn(d, p).clone())
        devs.append(d), ps.append(p)
        out = torch.empty_like(d["q"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attn_tree(d["q"], d["k_new"], d["v_new"], d["k_pages"], d["v_pages"], d["table"], d["ctx"], p, out=out)
        graphs.append(g), outs.append(out)
    for _ in range(3):
        for g, out, ref in zip(graphs, outs, refs):
            out.fill_(7)
            g.replay()
            assert torch.equal(out, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [run_attn(d, p) for d, p in zip(devs, ps)]
    here = [run_attn(d, p) for d, p in zip(devs, ps)]                 # overlaps the other stream's calls (the appended rows are the same)
    torch.cuda.synchronize()
    for g, h, ref in zip(got, here, refs):
        assert torch.equal(g, ref) and torch.equal(h, ref)
    assert _lib.device_status() == 0


@pytest.fixture(scope="module")
def short_waits(tmp_path_factory):
    return compile_library(tmp_path_factory.mktemp("short_waits"))


def test_attn_tree_gives_up_in_order(dev, short_waits):
    """Waits that run out are reported (status 2), nothing is left in flight, and the next calls are right."""
    rng = np.random.default_rng(20)
    for ctx, N, H, page in (([3000, 70, 0], 12, 8, 64), ([2000], 40, 8, 48), ([900, 1500], 3, 24, 5)):
        c = attn_case(rng, ctx, N, page, H)
        d, p = to_dev(c, dev), i32_dev(np.stack([random_tree(rng, N) for _ in ctx]), dev)
        ref = run_attn(d, p)
        assert _lib.device_status() == 0
        with operators_use(short_waits):
            for _ in range(20):
                run_attn(d, p)
                assert _lib.device_status() == 2
        assert torch.equal(run_attn(d, p), ref) and _lib.device_status() == 0


# ---------------------------------------------------------------------------------------------------------------------
# the gated delta rule
# ---------------------------------------------------------------------------------------------------------------------
def delta_case(rng, B, N, n_slots, layers=1):
    A, dtb = zip(*(synth.layer_params(rng) for _ in range(layers)))
    return dict(proj=synth.bf16r(rng.standard_normal((layers, B * N, 8224))), conv=synth.bf16r(rng.standard_normal((layers, n_slots * 2, 3, 6144))),
                conv_w=np.stack([synth.conv_weights(rng) for _ in range(layers)]), A_log=np.stack(A), dt_bias=np.stack(dtb),
                ssm=(rng.standard_normal((layers, n_slots, 16, 128, 128)) * 0.1).astype(np.float32),
                slots=rng.permutation(n_slots)[:B].astype(np.int32), pos=rng.integers(0, 1000, B).astype(np.int32))


def delta_dev(c, dev):
    f32 = ("ssm", "A_log", "dt_bias")
    return {k: i32_dev(v, dev) if v.dtype == np.int32 else f32_dev(v, dev) if k in f32 else bf16_dev(v, dev) for k, v in c.items()}


def run_delta(d, parents, proj=None):
    return deltanet_tree(d["proj"][0] if proj is None else proj, d["conv"][0], d["conv_w"][0], d["A_log"][0], d["dt_bias"][0], d["ssm"][0], d["slots"], d["pos"], parents)


@pytest.mark.parametrize("B,N,kind", [(1, 1, "chain"), (3, 2, "chain"), (2, 8, "random"), (2, 13, "forest"), (2, 16, "star"), (1, 17, "random"), (2, 32, "random"), (1, 33, "chain"),
                                      (2, 64, "random"), (1, 64, "chain"), (1, 63, "star"), (20, 5, "random")])
def test_deltanet_tree(dev, B, N, kind):
    rng = np.random.default_rng(B * 100 + N)
    c = delta_case(rng, B, N, B + 2)
    parents = np.stack([random_tree(rng, N, max(1, N - (2 * b) % 3), kind) for b in range(B)])
    d = delta_dev(c, dev)
    wide = torch.full((B * N, 8256), float("nan"), dtype=torch.bfloat16, device=dev)      # rows of a wider buffer
    wide[:, :8224] = d["proj"][0]
    keep = d["ssm"].clone(), d["conv"].clone()
    for proj in (None, wide[:, :8224]):
        y = host(run_delta(d, i32_dev(parents, dev), proj))
        for b in range(min(B, 4)):
            s, par = int(c["slots"][b]), int(c["pos"][b]) & 1
            ref = tree.deltanet_tree(c["proj"][0, b * N:(b + 1) * N], c["conv"][0, 2 * s + par], c["conv_w"][0], c["A_log"][0], c["dt_bias"][0], c["ssm"][0, s], parents[b])
            got = y[b * N:(b + 1) * N]
            scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
            assert (np.abs(got - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all(), (b, float((np.abs(got - ref) - HALF * np.abs(ref)).max()), float(scale.min()))
            assert not got[[i for i, line in enumerate(tree.lines(parents[b])) if not line]].any()
    assert torch.equal(d["ssm"], keep[0]) and torch.equal(d["conv"], keep[1]), "a verify changes nothing in the pools"
    assert _lib.device_status() == 0


def test_deltanet_tree_malformed_trees_slots_and_masked_nans(dev):
    rng = np.random.default_rng(31)
    c = delta_case(rng, 4, 6, 5)
    parents = np.stack([random_tree(rng, 6, kind="star") for _ in range(4)])
    d = delta_dev(c, dev)
    good = host(run_delta(d, i32_dev(parents, dev))).reshape(4, 6, -1)
    assert _lib.device_status() == 0
    for field, bad in (("slots", 5), ("slots", -1), ("pos", -3)):
        x = c[field].copy()
        x[2] = bad
        y = host(run_delta({**d, field: i32_dev(x, dev)}, i32_dev(parents, dev))).reshape(4, 6, -1)
        assert _lib.device_status() == 1
        assert not y[2].any() and np.array_equal(np.delete(y, 2, 0), np.delete(good, 2, 0))
    p = parents.copy()
    p[1] = [-1, 4, 0, 1, 0, 0]                                       # node 1 below a later node, node 3 below node 1
    y = host(run_delta(d, i32_dev(p, dev))).reshape(4, 6, -1)
    assert _lib.device_status() == 1
    assert not y[1, [1, 3]].any() and np.allclose(y[1, [0, 2, 4, 5]], good[1, [0, 2, 4, 5]], atol=2 * HALF * np.abs(good[1]).max())
    x = c["proj"].copy()
    x[0, 0 * 6 + 3] = np.nan                                         # a leaf
    x[0, 1 * 6 + 5] = np.inf                                         # an unused node
    p = parents.copy()
    p[1, 5] = -2
    y = host(run_delta(d, i32_dev(p, dev), bf16_dev(x[0], dev))).reshape(4, 6, -1)
    assert np.isnan(y[0, 3]).any() and np.array_equal(np.delete(y[0], 3, 0), np.delete(good[0], 3, 0)) and np.array_equal(y[1, :5], good[1, :5]) and not y[1, 5].any()
    assert _lib.device_status() == 0
    with pytest.raises(ValueError):
        run_delta(d, i32_dev(parents, dev).long())
    with pytest.raises(ValueError):
        run_delta(d, torch.full((1, 65), -1, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        run_delta({**d, "slots": d["slots"][:3]}, i32_dev(parents, dev))
    with pytest.raises(ValueError):
        run_delta({**d, "ssm": d["ssm"][:, :3]}, i32_dev(parents, dev))
    assert run_delta({**d, "slots": d["slots"][:0], "pos": d["pos"][:0]}, i32_dev(parents[:0], dev), d["proj"][0][:0]).shape == (0, 2048)


def test_deltanet_tree_refuses_rows_of_another_form(dev):
    rng = np.random.default_rng(33)
    d = delta_dev(delta_case(rng, 2, 3, 2), dev)
    p = i32_dev(np.stack([random_tree(rng, 3)] * 2), dev)
    proj = d["proj"][0]
    wide = torch.zeros(6, 2 * 8224, dtype=torch.bfloat16, device=dev)
    odd = torch.zeros(6 * 8224 + 1, dtype=torch.bfloat16, device=dev)[1:].view(6, 8224)
    for bad in (proj.float(), proj[:, :8223], proj[:5], proj.view(-1), wide[:, ::2], odd, proj.view(2, 3, 8224), torch.zeros(6, 8226, dtype=torch.bfloat16, device=dev)):
        with pytest.raises(ValueError):
            run_delta(d, p, bad)
    run_delta(d, p, torch.zeros(6, 8228, dtype=torch.bfloat16, device=dev))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N", [12, 64])
def test_deltanet_tree_with_decays_from_none_to_all(dev, N):
    """Tokens that keep the state, that halve it and that wipe it out, mixed along every path: what lies between two nodes of a path counts, not
    the sum from its root (which leaves the range in which fp32 tells a difference of 0.01 apart)."""
    rng = np.random.default_rng(N)
    c = delta_case(rng, 2, N, 3)
    c["dt_bias"][:] = 0
    c["A_log"][:] = 0
    a = rng.choice([-6.0, -1.0, 20.0, 100.0, 30000.0], (2 * N, 16), p=[0.4, 0.3, 0.1, 0.1, 0.1])      # decays e^-log(1 + e^a): 0.998, 0.73, 2e-9, 0, 0
    c["proj"][0, :, 8208:8224] = a
    parents = np.stack([random_tree(rng, N, kind=kind) for kind in ("chain", "random")])
    d = delta_dev(c, dev)
    y = host(run_delta(d, i32_dev(parents, dev)))
    for b in range(2):
        s, par = int(c["slots"][b]), int(c["pos"][b]) & 1
        ref = tree.deltanet_tree(host(d["proj"])[0, b * N:(b + 1) * N], c["conv"][0, 2 * s + par], c["conv_w"][0], c["A_log"][0], c["dt_bias"][0], c["ssm"][0, s], parents[b])
        got = y[b * N:(b + 1) * N]
        scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
        assert (np.abs(got - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all(), float((np.abs(got - ref) - HALF * np.abs(ref) - DELTA_ABS * scale).max())
    assert _lib.device_status() == 0


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("N", [6, 16, 27, 32, 50, 64])
def test_deltanet_tree_with_a_node_that_is_not_finite(dev, N, value):
    """A q, k, v or gate of one head of an inner node is NaN or infinite: that head sums over ancestors one by one.  Element by element the result is
    finite where the rule's is, and right there: nodes that do not hang below it, those that hang below a q far enough, the other heads."""
    rng = np.random.default_rng(N)
    c = delta_case(rng, 5, N, 5)
    parents = np.stack([random_tree(rng, N, N - b % 2) for b in range(5)])
    heads = [0, 5, 15, 7, 2]
    for b, (channel, h) in enumerate(zip((128 * 0 + 3, 2048 + 127, 4096 + 64, 0, 0), heads)):
        at = channel + 128 * h if b < 3 else 8192 + h if b == 3 else 8208 + h      # q, k, v; beta; decay
        c["proj"][0, b * N + N // 3, at] = value if b < 3 else np.nan
    d = delta_dev(c, dev)
    y = host(run_delta(d, i32_dev(parents, dev))).reshape(5, N, -1)
    for b, h in enumerate(heads):
        s, par = int(c["slots"][b]), int(c["pos"][b]) & 1
        with np.errstate(invalid="ignore", over="ignore"):
            ref = tree.deltanet_tree(c["proj"][0, b * N:(b + 1) * N], c["conv"][0, 2 * s + par], c["conv_w"][0], c["A_log"][0], c["dt_bias"][0], c["ssm"][0, s], parents[b])
        fin = np.isfinite(ref)
        assert fin[:, :128 * h].all() and fin[:, 128 * h + 128:].all() and not fin[N // 3].all() and fin[0].all()
        assert np.array_equal(np.isfinite(y[b]), fin), b
        ref, got = np.where(fin, ref, 0), np.where(fin, y[b], 0)
        scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
        assert (np.abs(got - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all(), (b, float((np.abs(got - ref) - HALF * np.abs(ref)).max()))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N", [6, 16, 20, 32, 64])
def test_deltanet_tree_over_a_state_that_is_not_finite(dev, N):
    """NaN and infinities in some value rows of a slot's state, and everywhere in the trash slot's: rows of unused nodes are zero all the same, used
    nodes get NaN in those value rows, as the rule gives it (an infinite S k meets itself with the other sign in S + beta (v - S k) k^T), and no others."""
    rng = np.random.default_rng(N)
    c = delta_case(rng, 4, N, 5)
    c["slots"][:] = [2, 0, 3, 4]
    c["ssm"][0, 0, 3, 17, 5] = np.nan
    c["ssm"][0, 0, 3, 90, 127] = np.inf
    c["ssm"][0, 0, 11, 64, 0] = -np.inf
    c["ssm"][0, 4] = rng.choice([np.nan, np.inf, -np.inf], (16, 128, 128))
    parents = np.stack([random_tree(rng, N, N - 2 - b) for b in range(4)])
    parents[1, 1], parents[3] = -2, -2                               # an unused node between used ones (and what hangs below it); an idle row of the batch
    d = delta_dev(c, dev)
    y = host(run_delta(d, i32_dev(parents, dev))).reshape(4, N, -1)
    for b in range(3):
        s, par = int(c["slots"][b]), int(c["pos"][b]) & 1
        with np.errstate(invalid="ignore"):
            ref = tree.deltanet_tree(c["proj"][0, b * N:(b + 1) * N], c["conv"][0, 2 * s + par], c["conv_w"][0], c["A_log"][0], c["dt_bias"][0], c["ssm"][0, s], parents[b])
        used = np.array([bool(line) for line in tree.lines(parents[b])])
        assert not y[b, ~used].any() and (~used).sum() >= 2 + b
        assert np.array_equal(np.isnan(y[b]), np.isnan(ref)) and np.isnan(ref).sum() == (3 * used.sum() if b == 1 else 0)
        ref = np.nan_to_num(ref)
        scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
        assert (np.abs(np.nan_to_num(y[b]) - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all()
    assert not y[3].any(), "an idle row, whatever the trash slot holds"
    assert _lib.device_status() == (1 if any(p == 1 for p in parents[1]) else 0)      # (a used node below an unused one is malformed)


def test_deltanet_tree_gives_up_in_order(dev, short_waits):
    """Waits that run out are reported (status 2), nothing is left in flight, and the next calls are right."""
    rng = np.random.default_rng(21)
    for B, N in ((20, 5), (20, 27), (30, 64)):
        c = delta_case(rng, B, N, B)
        d, p = delta_dev(c, dev), i32_dev(np.stack([random_tree(rng, N) for _ in range(B)]), dev)
        ref = run_delta(d, p)
        assert _lib.device_status() == 0
        with operators_use(short_waits):
            for _ in range(20):
                run_delta(d, p)
                assert _lib.device_status() == 2
        assert torch.equal(run_delta(d, p), ref) and _lib.device_status() == 0


def test_deltanet_tree_of_a_chain_agrees_with_deltanet_bm(dev):
    rng = np.random.default_rng(32)
    c = delta_case(rng, 2, 4, 3)
    c["pos"][:] = [4, 7]
    d = delta_dev(c, dev)
    y = host(run_delta(d, i32_dev(np.tile(np.arange(4) - 1, (2, 1)), dev)))
    ssm = torch.zeros(2, 4, 16, 128, 128, device=dev)
    conv = torch.zeros(4, 4, 3, 6144, dtype=torch.bfloat16, device=dev)
    for b in range(2):
        s = int(c["slots"][b])
        ssm[b, 0], conv[2 * b, 0] = d["ssm"][0, s], d["conv"][0, 2 * s + int(c["pos"][b]) % 2]
    zero = i32_dev([0, 0], dev)
    ref = host(deltanet_bm(d["proj"][0], conv, d["conv_w"][0], d["A_log"][0], d["dt_bias"][0], ssm, i32_dev([0, 1], dev), zero, zero, 4))
    # the chained kernel rounds conv, silu, norm (twice) and gates to bf16: six roundings of 2^-9 each on factors of y
    assert np.linalg.norm(y - ref) <= 6 * HALF * np.linalg.norm(ref)


@pytest.mark.parametrize("B,N,lengths,layers", [(1, 1, [1], 1), (3, 8, [1, 4, 0], 3), (4, 40, [2, 40, 17, 16], 2), (2, 6, [2, 3], 34)])
def test_deltanet_commit(dev, B, N, lengths, layers):
    rng = np.random.default_rng(N + layers)
    c = delta_case(rng, B, N, 2 * B + 1, layers)
    path = np.full((B, N), -1, np.int32)
    for b, n in enumerate(lengths):
        path[b, :n] = np.sort(rng.permutation(N)[:n])
    free = np.setdiff1d(np.arange(2 * B + 1), c["slots"])[:B].astype(np.int32)
    for stacked, dst in ((True, None), (False, free), (True, np.where(np.arange(B) % 2, c["slots"], free).astype(np.int32))):
        d = delta_dev(c, dev)
        args = [d[k] if stacked else list(d[k]) for k in ("proj", "conv", "conv_w", "A_log", "dt_bias", "ssm")]
        deltanet_commit(*args, d["slots"], d["pos"], i32_dev(path, dev), i32_dev(lengths, dev), dst_slots=None if dst is None else i32_dev(dst, dev))
        ssm, conv = host(d["ssm"]), host(d["conv"])
        want_ssm, want_conv = c["ssm"].astype(np.float64), c["conv"].copy()
        for l in range(0, layers, 1 if layers < 5 else 11):
            for b, n in enumerate(lengths):
                s, t, pos = int(c["slots"][b]), int(c["slots"][b] if dst is None else dst[b]), int(c["pos"][b])
                S, win = tree.commit(c["proj"][l, b * N:(b + 1) * N], c["conv"][l, 2 * s + (pos & 1)], c["conv_w"][l], c["A_log"][l], c["dt_bias"][l], c["ssm"][l, s], path[b, :n])
                # fp32 sums of 128 products per step, at most 40 steps
                assert np.abs(ssm[l, t] - S).max() <= 2.0 ** -16 * np.abs(S).max()
                want_ssm[l, t], want_conv[l, 2 * t + ((pos + n) & 1)] = ssm[l, t], win
            assert np.array_equal(ssm[l], want_ssm[l].astype(np.float32)) and np.array_equal(conv[l], want_conv[l]), "other slots and buffers stay as they are"
    assert _lib.device_status() == 0


def test_deltanet_commit_skips_what_is_out_of_range(dev):
    rng = np.random.default_rng(41)
    c = delta_case(rng, 3, 4, 4)
    path, n = np.tile(np.arange(4, dtype=np.int32), (3, 1)), np.array([2, 2, 2], np.int32)
    d = delta_dev(c, dev)
    run = lambda d, path, n, **k: deltanet_commit(d["proj"], d["conv"], d["conv_w"], d["A_log"], d["dt_bias"], d["ssm"], d["slots"], d["pos"], i32_dev(path, dev), i32_dev(n, dev), **k)  # noqa: E731
    run(d, path, n)
    good = d["ssm"].clone(), d["conv"].clone()
    s = int(c["slots"][1])
    p_bad, n_bad = path.copy(), n.copy()
    p_bad[1, 1], n_bad[1] = 4, 5
    for change, kw in ((dict(path=p_bad), {}), (dict(n=n_bad), {}), ({}, dict(dst_slots=i32_dev([c["slots"][0], 9, c["slots"][2]], dev)))):
        d = delta_dev(c, dev)
        run(d, **{"path": path, "n": n, **change}, **kw)
        assert _lib.device_status() == 1
        ssm, conv = d["ssm"][0], d["conv"][0]
        other = [i for i in range(4) if i != s]
        assert torch.equal(ssm[other], good[0][0][other]) and np.array_equal(host(ssm)[s], c["ssm"][0, s]) and np.array_equal(host(conv)[2 * s:2 * s + 2], c["conv"][0, 2 * s:2 * s + 2])
    with pytest.raises(ValueError):
        deltanet_commit([], [], [], [], [], [], d["slots"], d["pos"], i32_dev(path, dev), i32_dev(n, dev))
    with pytest.raises(ValueError):
        run(d, path[:2], n)
    with pytest.raises(ValueError):
        run({**d, "conv_w": d["conv_w"].float()}, path, n)
    with pytest.raises(ValueError):
        run({**d, "proj": d["proj"][:, :11]}, path, n)


def test_deltanet_commit_gives_up_in_order(dev, short_waits):
    """A block whose wait for its state runs out reports it (status 2) and writes nothing, in place or elsewhere, with and without a path."""
    rng = np.random.default_rng(22)
    c = delta_case(rng, 24, 10, 49, 4)
    n = rng.integers(0, 11, 24).astype(np.int32)
    path = i32_dev(np.tile(np.arange(10), (24, 1)), dev)
    free = np.setdiff1d(np.arange(48), c["slots"])[:24].astype(np.int32)
    for dst in (None, i32_dev(free, dev)):
        d = delta_dev(c, dev)
        with operators_use(short_waits):
            for _ in range(20):
                deltanet_commit(*(d[k] for k in ("proj", "conv", "conv_w", "A_log", "dt_bias", "ssm")), d["slots"], d["pos"], path, i32_dev(n, dev), dst_slots=dst)
                assert _lib.device_status() == 2
        assert np.array_equal(host(d["ssm"]), c["ssm"]) and np.array_equal(host(d["conv"]), c["conv"])
    assert _lib.device_status() == 0


def test_deltanet_commit_refuses_slots_that_depend_on_order(dev):
    rng = np.random.default_rng(42)
    c = delta_case(rng, 4, 3, 10)
    path, n = np.tile(np.arange(3, dtype=np.int32), (4, 1)), np.array([2, 1, 3, 2], np.int32)

    def run(slots, dst, n):
        d = delta_dev(c, dev)
        deltanet_commit(d["proj"], d["conv"], d["conv_w"], d["A_log"], d["dt_bias"], d["ssm"], i32_dev(slots, dev), d["pos"], i32_dev(path, dev), i32_dev(n, dev),
                        dst_slots=i32_dev(dst, dev))
        return d, host(d["ssm"])[0], _lib.device_status()
    good, bad = [0, 1, 2, 3], 0
    _, want, status = run(good, good, n)
    assert status == 0
    # (slots, destinations, sequences that are skipped)
    for slots, dst, skipped in (([0, 1, 0, 3], [0, 1, 0, 3], [0, 2]), ([0, 1, 2, 3], [4, 1, 4, 3], [0, 2]), ([0, 1, 2, 3], [2, 1, 5, 3], [0, 2]),
                                ([0, 1, 2, 3], [1, 2, 3, 0], [0, 1, 2, 3])):
        _, ssm, status = run(slots, dst, n)
        assert status == 1
        for b in range(4):
            if b in skipped:
                assert np.array_equal(ssm[dst[b]], c["ssm"][0, dst[b]]), (slots, dst, b)
            else:
                assert np.array_equal(ssm[dst[b]], want[b])
    # one slot read by many, untouched sequences, and padding in the last slot are all right
    _, ssm, status = run([0, 1, 0, 3], [0 + 4, 1, 5, 3], n)
    assert status == 0 and np.array_equal(ssm[4], want[0]) and np.array_equal(ssm[1], want[1])
    _, ssm, status = run([0, 1, 1, 1], [0, 1, 1, 1], np.array([2, 1, 0, 0], np.int32))
    assert status == 0 and np.array_equal(ssm[:2], want[:2])
    _, ssm, status = run([0, 9, 9, 3], [0, 9, 9, 3], n)
    assert status == 0 and np.array_equal(ssm[0], want[0]) and np.array_equal(ssm[3], want[3]) and np.array_equal(ssm[4:9], c["ssm"][0, 4:9])
    d = delta_dev(c, dev)
    with pytest.raises(ValueError, match="two layers"):
        deltanet_commit(*[[d[k][0]] * 2 for k in ("proj", "conv", "conv_w", "A_log", "dt_bias", "ssm")], d["slots"], d["pos"], i32_dev(path, dev), i32_dev(n, dev))


def test_more_sequences_than_a_block_has_threads(dev):
    """300 sequences: commit's look at the others' slots, compaction and accept go past one block's threads; two of them clash."""
    rng = np.random.default_rng(43)
    B = 300
    c = delta_case(rng, B, 1, B + 1)
    slots = rng.permutation(B).astype(np.int32)
    dup = slots.copy()
    dup[299] = dup[3]
    n = np.ones(B, np.int32)
    states = []
    for s in (slots, dup):
        d = delta_dev(c, dev)
        parents = torch.full((B, 1), -1, dtype=torch.int32, device=dev)
        n_path, path = accept_tree(parents, torch.zeros_like(parents), torch.zeros_like(parents))
        assert n_path.tolist() == n.tolist() and not path.any()
        deltanet_commit(d["proj"], d["conv"], d["conv_w"], d["A_log"], d["dt_bias"], d["ssm"], i32_dev(s, dev), d["pos"], path, n_path)
        states.append(host(d["ssm"])[0])
        assert _lib.device_status() == (s is dup)
    changed = np.array([(x != x0).any() for x, x0 in zip(states[0], c["ssm"][0])])
    assert changed[:B].all() and not changed[B]
    differs = np.array([(x != y).any() for x, y in zip(*states)])
    assert sorted(np.flatnonzero(differs)) == sorted([int(slots[3]), int(slots[299])])


# ---------------------------------------------------------------------------------------------------------------------
# accepting and copying
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("field", ["conv", "ssm"])
def test_deltanet_commit_refuses_one_pool_for_two_layers(dev, field):
    rng = np.random.default_rng(44)
    c = delta_case(rng, 2, 3, 4, 2)
    d = delta_dev(c, dev)
    layers = {k: list(d[k]) for k in ("proj", "conv", "conv_w", "A_log", "dt_bias", "ssm")}
    layers[field][1] = layers[field][0]
    with pytest.raises(ValueError, match=f"one {field} pool for two layers"):
        deltanet_commit(*layers.values(), d["slots"], d["pos"], i32_dev([[0, 1, 2]] * 2, dev), i32_dev([2, 1], dev))
    assert np.array_equal(host(d["ssm"]), c["ssm"]) and np.array_equal(host(d["conv"]), c["conv"])
    shared = {k: (list(d[k]) if k in ("conv", "ssm") else [d[k][0]] * 2) for k in layers}      # weights and rows may be shared
    deltanet_commit(*shared.values(), d["slots"], d["pos"], i32_dev([[0, 1, 2]] * 2, dev), i32_dev([2, 1], dev))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("N,kind", [(1, "chain"), (7, "random"), (32, "star"), (33, "forest"), (64, "random"), (64, "chain")])
def test_accept_tree(dev, N, kind):
    rng = np.random.default_rng(N)
    B = 37
    parents = np.stack([random_tree(rng, N, int(rng.integers(0, N + 1)), kind) for _ in range(B)])
    toks, ids = rng.integers(0, 3, (B, N)), rng.integers(0, 3, (B, N))
    for b in range(0, B, 3):                                         # chains that are confirmed to the end
        toks[b] = ids[b][np.maximum(parents[b], 0)]
    n, path = accept_tree(i32_dev(parents, dev), i32_dev(toks, dev), i32_dev(ids, dev))
    n, path = host(n), host(path)
    for b in range(B):
        want = tree.accept(parents[b], toks[b], ids[b])
        assert n[b] == len(want) and path[b].tolist() == want + [-1] * (N - len(want))
    assert _lib.device_status() == 0


def test_accept_tree_malformed(dev):
    parents = np.array([[-1, 2, 0, 1], [-1, -2, 1, 0]], np.int32)
    z = i32_dev(np.zeros((2, 4)), dev)
    n, path = accept_tree(i32_dev(parents, dev), z, z)
    assert _lib.device_status() == 1
    assert host(path).tolist() == [[0, 2, -1, -1], [0, 3, -1, -1]] and host(n).tolist() == [2, 2]
    with pytest.raises(ValueError):
        accept_tree(z.long(), z, z)
    with pytest.raises(ValueError):
        accept_tree(z, z[:1], z)
    assert accept_tree(z[:0], z[:0], z[:0])[1].shape == (0, 4)


@pytest.mark.parametrize("page,dim,dtype,L,elsewhere", [(64, 256, torch.bfloat16, 8, False), (16, 256, torch.bfloat16, 100, False), (5, 6, torch.bfloat16, 40, False), (8, 40, torch.float32, 33, True),
                                                        (64, 256, torch.bfloat16, 70, True)])
def test_compact_rows(dev, page, dim, dtype, L, elsewhere):
    rng = np.random.default_rng(L)
    base = np.array([0, 3, 77, page, 2 * page - 1], np.int32)
    B, width = len(base), (77 + 2 * L) // page + 2
    order = rng.permutation(2 * B * width) + 1
    table, other = order[:B * width].reshape(B, width).astype(np.int32), order[B * width:].reshape(B, width).astype(np.int32)
    pools = [torch.randn(2 * B * width + 1, 3, page, dim, device=dev).to(dtype) for _ in range(3)]
    n_keep = np.array([L, 0, L // 2, 1, L - 1], np.int32)
    keep = np.stack([np.sort(rng.permutation(2 * L)[:L]) for _ in base]).astype(np.int32)
    keep[3] = np.arange(L)
    want = [host(p).copy() for p in pools]
    to = other if elsewhere else table
    for X in want:
        src = X.copy()
        for b in range(B):
            for j in range(n_keep[b]):
                f, t = int(base[b] + keep[b, j]), int(base[b]) + j
                X[to[b, t // page], :, t % page] = src[table[b, f // page], :, f % page]
    compact_rows(pools, i32_dev(table, dev), i32_dev(base, dev), i32_dev(keep, dev), i32_dev(n_keep, dev), dst_table=i32_dev(other, dev) if elsewhere else None)
    assert all(np.array_equal(host(p), X) for p, X in zip(pools, want))
    assert _lib.device_status() == 0


def test_compact_rows_stops_at_a_bad_entry(dev):
    table = np.array([[1, 2], [3, 4], [5, 99], [6, 7]], np.int32)
    pool = torch.arange(8 * 4 * 8, device=dev).float().view(8, 1, 4, 8)
    want = host(pool).copy()
    keep = np.array([[1, 3, 2], [1, 8, 9], [2, 4, 5], [2, 3, 5]], np.int32)      # out of order; beyond the table; a bad page; fine
    for b, rows in ((0, [(0, 1), (1, 3)]), (1, [(0, 1)]), (2, [(0, 2)]), (3, [(0, 2), (1, 3), (2, 5)])):
        for t, f in rows:
            want[table[b, t // 4], :, t % 4] = host(pool)[table[b, f // 4], :, f % 4]
    compact_rows([pool], i32_dev(table, dev), i32_dev([0] * 4, dev), i32_dev(keep, dev), i32_dev([3] * 4, dev))
    assert _lib.device_status() == 1 and np.array_equal(host(pool), want)
    for n, base in ((-1, 0), (4, 0), (3, -1)):
        compact_rows([pool], i32_dev(table, dev), i32_dev([0, 0, 0, base], dev), i32_dev(keep, dev), i32_dev([0, 0, 0, n], dev))
        assert _lib.device_status() == 1 and np.array_equal(host(pool), want)
    t = i32_dev(table, dev)
    z = i32_dev([0] * 4, dev)
    for args in (([pool.half()], t, z, i32_dev(keep, dev), z), ([pool], t.long(), z, i32_dev(keep, dev), z), ([pool], t[:3], z, i32_dev(keep, dev), z), ([pool, pool[:3]], t, z, i32_dev(keep, dev), z),
                 ([], t, z, i32_dev(keep, dev), z)):
        with pytest.raises(ValueError):
            compact_rows(*args)


@pytest.mark.parametrize("shape,dtype,rows,stacked", [((40, 2, 64, 256), torch.bfloat16, None, False), ((40, 2, 64, 256), torch.bfloat16, 37, True), ((400, 2, 8, 16), torch.bfloat16, "each", False),
                                                      ((9, 16, 128, 128), torch.float32, None, True), ((30, 3, 5, 3), torch.bfloat16, 2, False), ((30, 7), torch.float32, None, False), ((30, 3, 5, 3), torch.float32, 0, False)])
def test_copy_entries(dev, shape, dtype, rows, stacked):
    rng = np.random.default_rng(shape[0])
    n = shape[0] // 2 - 1
    order = rng.permutation(shape[0])
    dst, src = order[:n].tolist(), rng.choice(order[n:], n).tolist()        # sources repeat
    pools = [torch.randn((3, *shape) if stacked else shape, device=dev).to(dtype) for _ in range(2)]
    want = [p.clone() for p in pools]
    each = rng.integers(0, shape[2] + 1, n).tolist() if rows == "each" else [rows] * n
    for X in want:
        for Y in (X if stacked else [X]):
            for d, s, r in zip(dst, src, each):
                if r is None:
                    Y[d] = Y[s]
                else:
                    Y[d, :, :r] = Y[s, :, :r]
    copy_entries(pools, dst, src, rows=each if rows == "each" else rows, stacked=stacked)
    assert all(torch.equal(p, X) for p, X in zip(pools, want))


@pytest.mark.parametrize("entries,n,rows", [(1400, 600, "each"), (20000, 1030, 3)])
def test_copy_entries_beyond_one_launch(dev, entries, n, rows):
    rng = np.random.default_rng(n)
    order = rng.permutation(entries)
    dst, src = order[:n], order[n:2 * n]
    p = torch.randn(entries, 2, 4, 8, device=dev)
    each = rng.integers(0, 5, n) if rows == "each" else np.full(n, rows)
    want = p.cpu().clone()
    for d, s, r in zip(dst, src, each):
        want[d, :, :r] = want[s, :, :r]
    copy_entries([p], dst.tolist(), src.tolist(), rows=each.tolist() if rows == "each" else rows)
    assert torch.equal(p.cpu(), want)
    for d, s in ((dst.tolist() + [int(dst[5])], src.tolist() + [int(src[5])]), (dst.tolist() + [int(src[7])], src.tolist() + [int(order[-1])])):
        with pytest.raises(ValueError, match="entry"):
            copy_entries([p], d, s)
    assert torch.equal(p.cpu(), want)


def test_copy_entries_refusals(dev):
    p = torch.zeros(6, 2, 4, 8, device=dev)
    copy_entries([p], [], [])
    for dst, src, kw in (([1, 1], [0, 0], {}), ([1, 2], [0, 1], {}), ([6], [0], {}), ([0], [-1], {}), ([0, 1], [2], {}), ([1], [0], dict(rows=5)), ([1], [0], dict(rows=[1, 2])), ([1], [0], dict(rows=-1))):
        with pytest.raises(ValueError):
            copy_entries([p], dst, src, **kw)
    for pools in ([], [p.half()], [p, p[:3]], [p.transpose(2, 3)]):
        with pytest.raises(ValueError):
            copy_entries(pools, [1], [0])
    with pytest.raises(ValueError):
        copy_entries([p.view(6, 64)], [1], [0], rows=1)
    assert not p.any()


@pytest.mark.parametrize("dst,src,rows", [([2 ** 31], [0], None), ([0], [-2 ** 31 - 1], None), ([2 ** 40], [0], 1), ([1], [0], [2 ** 63])])
def test_copy_entries_refuses_numbers_beyond_32_bits(dev, dst, src, rows):
    p = torch.zeros(6, 2, 4, 8, device=dev)
    with pytest.raises(ValueError):
        copy_entries([p], dst, src, rows=rows)


def test_page_copies_onto_themselves_and_of_no_rows_change_nothing(dev):
    pool = PagePool(2, 6, 8, 2, 16, device=dev)
    for X in pool.K + pool.V:
        X.copy_(torch.randn(X.shape, device=dev))
    before = [X.clone() for X in pool.K + pool.V]
    pool.copy_rows(3, 3, 5)
    pool.copy_rows(3, 3, 8)
    pool.copy_rows(2, 1, 0)
    pool.copy_rows(2, 1, -1)
    pool.copy_pages([1, 4], [1, 4], 8)
    assert all(torch.equal(X, X0) for X, X0 in zip(pool.K + pool.V, before))
    pool.copy_pages([1, 4, 5], [1, 2, 5], 3)
    for X, X0 in zip(pool.K + pool.V, before):
        X0[4, :, :3] = X0[2, :, :3]
        assert torch.equal(X, X0)
    with pytest.raises(ValueError):
        pool.copy_pages([1, 2], [3], 8)


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
def test_rounds_of_tree_speculation_on_paged_pools(dev):
    """Fork a prompt into two slots; three rounds of verify, accept and commit over all layers; the caches hold exactly the accepted tokens:
    states and windows as the token-by-token rule leaves them, K/V rows in order, and the next round's attention sees them."""
    rng = np.random.default_rng(77)
    cfg = Cfg(layers=4)                                              # three GatedDeltaNet layers and a full-attention layer
    nl, N, ctx0 = cfg.n_linear, 10, 61
    pools = PagedPools(cfg, 4, 256, n_pages=30)
    c = delta_case(rng, 1, 1, 1, nl)
    kv = synth.bf16r(rng.standard_normal((2, 1, 2, ctx0, 256)))
    state = dict(kv=[(bf16_dev(kv[0], dev), bf16_dev(kv[1], dev))], conv=[bf16_dev(x[:1], dev) for x in c["conv"]], ssm=[f32_dev(x[:1], dev) for x in c["ssm"]])
    pools.admit(2, state, ctx0)
    pools.fork(2, [0, 3])
    seqs = [3, 2, 0]
    B = len(seqs)
    hist = [(kv[0, 0], kv[1, 0]) for _ in seqs]                      # K, V [2, n, 256] of every sequence
    S = [[x[0].astype(np.float64) for x in c["ssm"]] for _ in seqs]
    win = [[x[0].astype(np.float64) for x in c["conv"]] for _ in seqs]
    weights = bf16_dev(c["conv_w"], dev), f32_dev(c["A_log"], dev), f32_dev(c["dt_bias"], dev)
    slots = i32_dev(seqs, dev)
    for _ in range(3):
        lengths = [int(pools.length[s]) for s in seqs]
        for s, n in zip(seqs, lengths):
            pools.reserve(s, n + N)
        pos = i32_dev(lengths, dev)
        parents = np.stack([random_tree(rng, N, N - b) for b in range(B)])
        proj = synth.bf16r(rng.standard_normal((nl, B * N, 8224)))
        q, k, v = (synth.bf16r(rng.standard_normal((B * N, h, 256))) for h in (8, 2, 2))
        ids = rng.integers(0, 2, (B, N)).astype(np.int32)
        toks = rng.integers(0, 2, (B, N)).astype(np.int32)
        p = i32_dev(parents, dev)
        projs = [bf16_dev(x, dev) for x in proj]
        ys = [host(pools.deltanet_tree(l, projs[l], weights[0][l], weights[1][l], weights[2][l], slots, pos, p)) for l in range(nl)]
        o = host(pools.attn_tree(0, bf16_dev(q, dev), bf16_dev(k, dev), bf16_dev(v, dev), slots, pos, p))
        n_path, path = accept_tree(p, i32_dev(toks, dev), i32_dev(ids, dev))
        pools.commit_tree(projs, list(weights[0]), list(weights[1]), list(weights[2]), slots, pos, path, n_path)
        for b, s in enumerate(seqs):
            r = slice(b * N, (b + 1) * N)
            ref, mag = tree.attn_tree(q[r], k[r], v[r], *hist[b], parents[b])
            assert (np.abs(o[r] - ref) <= HALF * np.abs(ref) + ATTN_ABS * mag + 1e-30).all()
            want = tree.accept(parents[b], toks[b], ids[b])
            assert host(path)[b, :int(n_path[b])].tolist() == want
            hist[b] = tuple(np.concatenate([h, x[r][want].transpose(1, 0, 2)], 1) for h, x in zip(hist[b], (k, v)))
            pools.advance(s, len(want))
            pools.trim(s)
            n = int(pools.length[s])
            for X, h in zip((pools.pages.K[0], pools.pages.V[0]), hist[b]):
                rows = np.concatenate([host(X[pg]) for pg in pools.owned[s]], 1)
                assert np.array_equal(rows[:, :n], h), "the accepted rows lie behind the context in order"
            assert len(pools.owned[s]) == -(-n // 64)
            for l in range(nl):
                ref = tree.deltanet_tree(proj[l, r], win[b][l], c["conv_w"][l], c["A_log"][l], c["dt_bias"][l], S[b][l], parents[b])
                scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
                assert (np.abs(ys[l][r] - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all()
                S[b][l], win[b][l] = tree.commit(proj[l, r], win[b][l], c["conv_w"][l], c["A_log"][l], c["dt_bias"][l], S[b][l], want)
                assert np.abs(host(pools.ssm[l][s]) - S[b][l]).max() <= 2.0 ** -16 * np.abs(S[b][l]).max()
                assert np.array_equal(host(pools.conv[l][2 * s + n % 2]), win[b][l])
    for s in seqs:
        pools.release(s)
    assert pools.pages.available() == pools.pages.n_pages - 1
    assert _lib.device_status() == 0


def test_a_round_captured_replayed_and_padded(dev):
    """Verify, accept, commit and compaction in one captured graph, replayed on fresh contents: what eager calls give; idle rows of the batch (trash
    slot, no nodes) change nothing; two such rounds on two streams do not disturb each other."""
    rng = np.random.default_rng(91)
    cfg = Cfg(layers=4)
    nl, N, live, S = cfg.n_linear, 7, 3, 5
    c = delta_case(rng, live, 1, S + 1, nl)
    f = lambda *s: synth.bf16r(rng.standard_normal(s))  # noqa: E731
    weights = list(bf16_dev(c["conv_w"], dev)), list(f32_dev(c["A_log"], dev)), list(f32_dev(c["dt_bias"], dev))
    lengths = [61, 64, 3]

    def fresh():
        pools = PagedPools(cfg, S, 256, n_pages=20)
        for l in range(nl):
            pools.ssm[l].copy_(f32_dev(c["ssm"][l], dev))
            pools.conv[l].copy_(bf16_dev(c["conv"][l], dev))
        for X, Y in zip(pools.pages.K + pools.pages.V, kv):
            X.copy_(Y)
        for s in range(live):
            pools.reserve(s, lengths[s] + N)
        return pools

    kv = [bf16_dev(f(20, 2, 64, 256), dev) for _ in range(2)]
    rounds = []
    for _ in range(2):
        parents = np.stack([random_tree(rng, N, N - b) for b in range(live)])
        rounds.append(dict(parents=parents, proj=f(nl, live * N, 8224), q=f(live * N, 8, 256), k=f(live * N, 2, 256), v=f(live * N, 2, 256),
                           toks=rng.integers(0, 2, (live, N)), ids=rng.integers(0, 2, (live, N))))

    def inputs(r, B):
        pad = lambda x, n, fill: np.concatenate([x, np.full((n, *x.shape[1:]), fill, x.dtype)])  # noqa: E731
        rows, seqs = (B - live) * N, B - live
        return dict(parents=i32_dev(pad(r["parents"], seqs, -2), dev), toks=i32_dev(pad(r["toks"], seqs, 0), dev), ids=i32_dev(pad(r["ids"], seqs, 0), dev),
                    q=bf16_dev(pad(r["q"], rows, np.nan), dev), k=bf16_dev(pad(r["k"], rows, np.nan), dev), v=bf16_dev(pad(r["v"], rows, np.nan), dev),
                    projs=[bf16_dev(pad(x, rows, np.nan), dev) for x in r["proj"]], slots=i32_dev(list(range(live)) + [S] * seqs, dev), pos=i32_dev(lengths + [0] * seqs, dev))

    def step(pools, i):
        ys = [pools.deltanet_tree(l, i["projs"][l], weights[0][l], weights[1][l], weights[2][l], i["slots"], i["pos"], i["parents"]) for l in range(nl)]
        o = pools.attn_tree(0, i["q"], i["k"], i["v"], i["slots"], i["pos"], i["parents"])
        n_path, path = accept_tree(i["parents"], i["toks"], i["ids"])
        pools.commit_tree(i["projs"], *weights, i["slots"], i["pos"], path, n_path)
        return [*ys, o, n_path, path]

    caches = lambda pools: [*pools.ssm, *pools.conv, *pools.pages.K, *pools.pages.V]  # noqa: E731
    start = [x.clone() for x in caches(fresh())]
    want = []
    for r in rounds:
        pools = fresh()
        out = step(pools, inputs(r, live))
        want.append((out, [x.clone() for x in caches(pools)]))
    assert _lib.device_status() == 0

    B = live + 2
    per_round = []
    for r in rounds:                                                 # one graph per round, pools and inputs of its own
        pools, i = fresh(), inputs(r, B)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(pools, i)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(pools, i)
        per_round.append((g, pools, out, torch.cuda.Stream(), i))    # (a graph does not keep its inputs alive)
    for _ in range(3):
        for g, pools, _, _, _ in per_round:
            for x, x0 in zip(caches(pools), start):
                x.copy_(x0)
        torch.cuda.synchronize()
        for g, _, _, stream, _ in per_round:                            # both at once
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for (g, pools, out, _, _), (ref, after) in zip(per_round, want):
            for x, y in zip(out, ref):
                assert torch.equal(x[:len(y)], y) and not (x[len(y):].float() * (x[len(y):] != -1)).any(), "idle rows: zeros, and -1 in the path"
            for x, y in zip(caches(pools), after):
                assert torch.equal(x, y)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("max_len,page", [(128, 64), (100, 64), (70, 7)])
def test_a_round_at_the_end_of_a_sequence(dev, max_len, page):
    """The last round before max_len, as documented: room for what fits, the nodes behind it unused.  A tree that fits to the last row, one of which two nodes
    fit, and a full sequence."""
    rng = np.random.default_rng(max_len)
    cfg = Cfg(layers=4)
    N, lengths = 6, [max_len - 6, max_len - 2, max_len]
    pools = PagedPools(cfg, 3, max_len, n_pages=3 * -(-max_len // page) + 1, page_size=page)
    c = delta_case(rng, 3, N, 4, cfg.n_linear)
    for l in range(cfg.n_linear):
        pools.ssm[l].copy_(f32_dev(c["ssm"][l], dev))
        pools.conv[l].copy_(bf16_dev(c["conv"][l], dev))
    r = lambda *s: synth.bf16r(rng.standard_normal(s))  # noqa: E731
    kv = [r(2, 2, n, 256) for n in lengths]
    for s, n in enumerate(lengths):
        pools.reserve(s, n)
        pools.length[s] = n
        for X, x in zip((pools.pages.K[0], pools.pages.V[0]), kv[s]):
            for i, pg in enumerate(pools.owned[s]):
                rows = x[:, i * page:(i + 1) * page]
                X[pg, :, :rows.shape[1]] = bf16_dev(rows, dev)
        pools.reserve(s, min(n + N, pools.Lmax))
    parents = np.stack([random_tree(rng, N, min(N, max_len - n)) for n in lengths])
    q, k, v = (r(3 * N, h, 256) for h in (8, 2, 2))
    slots, pos, p = i32_dev([0, 1, 2], dev), i32_dev(lengths, dev), i32_dev(parents, dev)
    projs, w = [bf16_dev(x, dev) for x in c["proj"]], (list(bf16_dev(c["conv_w"], dev)), list(f32_dev(c["A_log"], dev)), list(f32_dev(c["dt_bias"], dev)))
    ys = [host(pools.deltanet_tree(l, projs[l], w[0][l], w[1][l], w[2][l], slots, pos, p)).reshape(3, N, -1) for l in range(cfg.n_linear)]
    o = host(pools.attn_tree(0, bf16_dev(q, dev), bf16_dev(k, dev), bf16_dev(v, dev), slots, pos, p)).reshape(3, N, 8, 256)
    ids = np.zeros((3, N), np.int32)
    n_path, path = accept_tree(p, i32_dev(ids, dev), i32_dev(ids, dev))
    pools.commit_tree(projs, *w, slots, pos, path, n_path)
    for s, n in enumerate(lengths):
        want = tree.accept(parents[s], ids[s], ids[s])
        assert len(want) == int(n_path[s]) and (len(want) > 0) == (s < 2)
        ref, mag = tree.attn_tree(q[s * N:(s + 1) * N], k[s * N:(s + 1) * N], v[s * N:(s + 1) * N], *kv[s], parents[s])
        assert (np.abs(o[s] - ref) <= HALF * np.abs(ref) + ATTN_ABS * mag + 1e-30).all()
        pools.advance(s, len(want))
        pools.trim(s)
        for X, x, new in zip((pools.pages.K[0], pools.pages.V[0]), kv[s], (k, v)):
            rows = np.concatenate([host(X[pg]) for pg in pools.owned[s]], 1)[:, :n + len(want)]
            assert np.array_equal(rows, np.concatenate([x, new[s * N:(s + 1) * N][want].transpose(1, 0, 2)], 1))
        for l in range(cfg.n_linear):
            win = c["conv"][l, 2 * s + (n & 1)]
            ref = tree.deltanet_tree(c["proj"][l, s * N:(s + 1) * N], win, c["conv_w"][l], c["A_log"][l], c["dt_bias"][l], c["ssm"][l, s], parents[s])
            scale = np.abs(ref).reshape(N, 16, 128).max((0, 2)).repeat(128)
            assert (np.abs(ys[l][s] - ref) <= HALF * np.abs(ref) + DELTA_ABS * scale).all()
            S, win = tree.commit(c["proj"][l, s * N:(s + 1) * N], win, c["conv_w"][l], c["A_log"][l], c["dt_bias"][l], c["ssm"][l, s], want)
            assert np.abs(host(pools.ssm[l][s]) - S).max() <= 2.0 ** -16 * np.abs(S).max()
            assert np.array_equal(host(pools.conv[l][2 * s + (n + len(want)) % 2]), win)
    assert _lib.device_status() == 0


def test_pools_beyond_32_bit_offsets(dev):
    """Pages and slots that lie more than 2^31 elements into their pools give what the same contents give at the front."""
    rng = np.random.default_rng(5)
    c = attn_case(rng, [300, 64], 20, 64)
    parents = i32_dev(np.stack([random_tree(rng, 20) for _ in range(2)]), dev)
    d = to_dev(c, dev)
    near = run_attn(d, parents)
    used = c["k_pages"].shape[0]
    total = 2 ** 31 // (2 * 64 * 256) + used + 1                     # the last `used` pages start behind element 2^31
    K, V = (torch.empty(total, 2, 64, 256, dtype=torch.bfloat16, device=dev) for _ in range(2))
    first = total - used
    for X, name in ((K, "k_pages"), (V, "v_pages")):
        X[first:] = bf16_dev(c[name], dev)
    table = d["table"] + first
    assert torch.equal(attn_tree(d["q"], d["k_new"], d["v_new"], K, V, table, d["ctx"], parents), near)
    assert torch.equal(K[first:], d["k_pages"]) and torch.equal(V[first:], d["v_pages"]), "the appended rows too"
    keep, n_keep = i32_dev([[0, 3, 7, 19], [1, 2, 5, 6]], dev), i32_dev([4, 3], dev)
    compact_rows([d["k_pages"], d["v_pages"]], d["table"], d["ctx"], keep, n_keep)
    compact_rows([K, V], table, d["ctx"], keep, n_keep)
    assert torch.equal(K[first:], d["k_pages"]) and torch.equal(V[first:], d["v_pages"])
    copy_entries([K, V], [0, total - 1], [first + 1, 1], rows=33)
    assert torch.equal(K[0, :, :33], K[first + 1, :, :33]) and torch.equal(V[total - 1, :, :33], V[1, :, :33])
    del K, V

    c = delta_case(rng, 2, 9, 2)
    c["slots"][:] = [0, 1]
    d = delta_dev(c, dev)
    parents = i32_dev(np.stack([random_tree(rng, 9) for _ in range(2)]), dev)
    path, n = i32_dev([[0, 1, 4], [0, 2, -1]], dev), i32_dev([3, 2], dev)
    far = 2 ** 31 // (16 * 128 * 128) + 1
    ssm = torch.empty(1, far + 5, 16, 128, 128, device=dev)
    conv = torch.empty(1, 2 * (far + 5), 3, 6144, dtype=torch.bfloat16, device=dev)
    ssm[:, far:far + 2], conv[:, 2 * far:2 * far + 4] = d["ssm"], d["conv"]
    e = {**d, "ssm": ssm, "conv": conv, "slots": d["slots"] + far}
    assert torch.equal(run_delta(e, parents), run_delta(d, parents))
    for x in (d, e):
        deltanet_commit(x["proj"], x["conv"], x["conv_w"], x["A_log"], x["dt_bias"], x["ssm"], x["slots"], x["pos"], path, n)
    assert torch.equal(ssm[:, far:far + 2], d["ssm"]) and torch.equal(conv[:, 2 * far:2 * far + 4], d["conv"])
    copy_entries([ssm], [far + 3], [far + 1], stacked=True)
    assert torch.equal(ssm[0, far + 3], ssm[0, far + 1])
    assert _lib.device_status() == 0
