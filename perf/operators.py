"""What is timed and compared for the operators of speculative decoding with a TREE of drafted tokens, and for the cache copies around it.

One round of tree speculation on the hybrid model: every sequence has up to 64 drafted tokens ("nodes"); node i hangs below the
node parents[i] < i, or (-1) below the last token in the caches; a smaller value marks an unused node.  Per layer the nodes are
verified at once,

* ``attn``   -- full-attention layers: each node attends the paged cache and its own ancestors; the rows are appended to the cache,
* ``delta``  -- GatedDeltaNet layers: each node starts from its parent's state (the slot's state for a root); no state is written,

then the round is settled over all layers,

* ``commit`` -- the accepted path is found from the target's tokens, the recurrent states advance along it and the K/V rows of the
  path move to the front of the appended rows (here into another slot and other pages, so that the source stays a checkpoint),

and, when sequences are forked (parallel samples of one prompt, checkpoints),

* ``copy``   -- entries of many pools at once: K/V pages (their first rows), recurrent states, conv windows.

Sizes are those of the model constants in qwen_tailor_b200/config.py: 18 GatedDeltaNet layers with 16 heads of 128 x 128 fp32 state
and 6144 mixed channels, 6 full-attention layers with head_dim 256 (8 query heads on 2 KV heads; other head counts are drawn too).
"""
import math

import numpy as np
import torch

own = False

HV, DK, KD, CD, PW, D = 16, 128, 2048, 6144, 8224, 256
N_LINEAR, N_FULL, PAGE = 18, 6, 64
STATE = HV * DK * DK * 4                                             # bytes of one recurrent state
WINDOW = 3 * CD * 2                                                  # bytes of one conv window


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a single user with a short prompt and a small tree: the latency of one layer
        dict(name="attn-one-short", op="attn", B=1, N=8, depth=4, lo=700, hi=700, page=64, H=8, KV=2, ragged=False),
        # the verify step of the benchmark (contexts from 1024 to 8192), 16 drafted tokens
        dict(name="attn-16x16", op="attn", B=16, N=16, depth=5, lo=1024, hi=8192, page=64, H=8, KV=2, ragged=False),
        # fresh and short sequences in odd numbers, pages that end inside a tile, unused nodes
        dict(name="attn-odd", op="attn", B=9, N=13, depth=6, lo=0, hi=1999, page=48, H=8, KV=2, ragged=True),
        # long documents and the largest tree
        dict(name="attn-long", op="attn", B=2, N=64, depth=8, lo=50001, hi=65536, page=64, H=8, KV=2, ragged=False),
        # one layer, one sequence, small tree
        dict(name="delta-one", op="delta", B=1, N=8, depth=4, ragged=False),
        # a medium batch, trees of different sizes
        dict(name="delta-16x27", op="delta", B=16, N=27, depth=6, ragged=True),
        # a full batch with the largest trees
        dict(name="delta-64x64", op="delta", B=64, N=64, depth=10, ragged=False),
        # settling a round for one sequence: all layers
        dict(name="commit-one", op="commit", B=1, N=8, depth=4, lo=700, hi=700),
        # settling a round for a batch: all layers
        dict(name="commit-24x32", op="commit", B=24, N=32, depth=7, lo=61, hi=900),
        # a prompt's slot forked for seven more samples: states, windows and the partly filled last page of every layer
        dict(name="fork-7", op="copy", what="fork", slots=8, n=7, pages=64, rows=37),
        # pages copied for many sequences at once (copy on write after a shared prefix)
        dict(name="pages-300", op="copy", what="pages", slots=0, n=300, pages=700, rows=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "delta", "commit", "copy"])
    if op == "attn":
        N, hi = _log(rng, 1, 64), _log(rng, 1, 65536)
        B = min(_log(rng, 1, 32), max(1, 115000 // (hi + N)))
        H, KV = rng.choice([(8, 2), (8, 2), (16, 2), (4, 4), (24, 4)])
        while B * KV * (hi + N) > 230000 or B * H * N * hi > 60000000:
            B, hi = max(1, B // 2), max(1, hi * 3 // 4)
        return dict(op="attn", B=B, N=N, depth=rng.randint(1, min(N, 12)), lo=rng.randint(0, hi), hi=hi, page=rng.choice([64, 64, 16, 48, 100, 256]),
                    H=H, KV=KV, ragged=rng.random() < 0.5)
    if op == "delta":
        N = _log(rng, 1, 64)
        return dict(op="delta", B=_log(rng, 1, 64), N=N, depth=rng.randint(1, min(N, 16)), ragged=rng.random() < 0.5)
    if op == "commit":
        N = _log(rng, 1, 64)
        return dict(op="commit", B=_log(rng, 1, 24), N=N, depth=rng.randint(1, min(N, 7)), lo=rng.randint(0, 500), hi=rng.randint(500, 900))
    if rng.random() < 0.5:
        return dict(op="copy", what="fork", slots=8, n=rng.randint(1, 7), pages=rng.randint(16, 64), rows=rng.randint(1, 64))
    n = _log(rng, 1, 300)
    return dict(op="copy", what="pages", slots=0, n=n, pages=2 * n + rng.randint(1, 100), rows=rng.choice([0, 0, 1, 33, 63]))


def _spread(lo, hi, B):
    """B lengths from lo to hi, in an order that mixes short and long ones."""
    v = [lo + (hi - lo) * i // max(1, B - 1) for i in range(B)] if B > 1 else [hi]
    return [v[(i * 7 + B // 2) % B] if math.gcd(7, B) == 1 else v[i] for i in range(B)]


def _used(c):
    """Nodes in use per sequence."""
    return [max(1, c["N"] - (b * 5) % 7) if c.get("ragged") else c["N"] for b in range(c["B"])]


def _accepted(c):
    """Nodes on the accepted path per sequence (the confirmed token included)."""
    return [1 + (b * 3 + c["depth"] - 1) % c["depth"] for b in range(c["B"])]


def work(c):
    if c["op"] == "attn":
        N, H, KV = c["N"], c["H"], c["KV"]
        ctx, used = _spread(c["lo"], c["hi"], c["B"]), _used(c)
        keys, nodes = sum(ctx), sum(used)
        # cached K and V once; the nodes' k and v once, and once more into the cache; q and the result
        nbytes = keys * KV * D * 4 + nodes * (KV * D * 8 + H * D * 4) + c["B"] * N * 4
        return dict(bytes=nbytes, flops=sum(4 * D * H * u * (t + c["depth"]) for t, u in zip(ctx, used)))
    if c["op"] == "delta":
        nodes = sum(_used(c))
        nbytes = c["B"] * (STATE + WINDOW) + nodes * ((CD + 32) * 2 + KD * 2) + CD * 8
        # S0 k, S0 q; k.k, q.k and two sums over the ancestors (depth of them)
        return dict(bytes=nbytes, flops=nodes * HV * (4 * DK * DK + 8 * DK * c["depth"] / 2))
    if c["op"] == "commit":
        steps = sum(_accepted(c))
        nbytes = N_LINEAR * (c["B"] * 2 * (STATE + WINDOW) + steps * (CD + 32) * 2) + N_FULL * steps * 2 * 2 * D * 2 * 2
        return dict(bytes=nbytes, flops=N_LINEAR * steps * HV * 6 * DK * DK)
    page = 2 * N_FULL * 2 * D * 2                                    # one row of every layer, K and V, two heads
    if c["what"] == "fork":
        return dict(bytes=(1 + c["n"]) * (N_LINEAR * (STATE + WINDOW) + page * c["rows"]), flops=0)
    return dict(bytes=2 * c["n"] * page * (c["rows"] or PAGE), flops=0)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _trees(rs, c):
    """parents int32 [B, N] and, per sequence, the nodes of a trunk `depth` long; the other nodes hang anywhere."""
    B, N, depth = c["B"], c["N"], c["depth"]
    parents, trunks = np.full((B, N), -2, np.int32), []
    for b, used in enumerate(_used(c)):
        trunk = [0] + sorted((1 + rs.permutation(used - 1)[:min(depth, used) - 1]).tolist())
        for i in range(used):
            if i == 0:
                parents[b, i] = -1
            elif i in trunk:
                parents[b, i] = trunk[trunk.index(i) - 1]
            else:
                parents[b, i] = rs.randint(0, min(i, 1 + 2 * len([t for t in trunk if t < i])))
        trunks.append(trunk)
    return parents, trunks


def _tables(rs, need, extra=0):
    """A block table over shuffled pages (page 0 pads it); need[b] pages for sequence b."""
    total = sum(need) + 1 + extra
    order = 1 + rs.permutation(total - 1)
    table = np.zeros((len(need), max(need)), np.int32)
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = order[o:o + n]
        o += n
    return table, total, order[o:]


def prepare(case, seed):
    c = case
    rs = np.random.RandomState((seed * 1000003 + 12345) % (1 << 31))
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 1)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    bf = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    s = dict(case=c, op=c["op"])
    if c["op"] == "attn":
        B, N, H, KV, P = c["B"], c["N"], c["H"], c["KV"], c["page"]
        ctx = _spread(c["lo"], c["hi"], B)
        table, total, _ = _tables(rs, [(t + N + P - 1) // P for t in ctx])
        s.update(q=bf(B * N, H, D), k_new=bf(B * N, KV, D), v_new=bf(B * N, KV, D), k_pages=bf(total, KV, P, D), v_pages=bf(total, KV, P, D),
                 table=i32(table), ctx=i32(ctx), parents=i32(_trees(rs, c)[0]))
        return s
    if c["op"] in ("delta", "commit"):
        B, N = c["B"], c["N"]
        layers = 1 if c["op"] == "delta" else N_LINEAR
        n_slots = (B if c["op"] == "delta" else 2 * B) + 2               # `commit` writes into a second set of slots
        slots = rs.permutation(n_slots - 1)
        parents, trunks = _trees(rs, c)
        s.update(proj=bf(layers, B * N, PW), conv=bf(layers, n_slots * 2, 3, CD), conv_w=(torch.randn(layers, CD * 4, generator=g, device="cuda") * 0.5).bfloat16(),
                 A_log=torch.rand(layers, HV, generator=g, device="cuda") * math.log(16.0), dt_bias=torch.randn(layers, HV, generator=g, device="cuda") * 0.1,
                 ssm=torch.randn(layers, n_slots, HV, DK, DK, generator=g, device="cuda") * 0.1,
                 slots=i32(slots[:B]), parents=i32(parents))
        if c["op"] == "delta":
            s["pos"] = i32(rs.randint(0, 5000, B))
            return s
        ctx = _spread(c["lo"], c["hi"], B)
        need = [(t + N + PAGE - 1) // PAGE for t in ctx]
        tails = [n - t // PAGE for n, t in zip(need, ctx)]
        table, total, spare = _tables(rs, need, sum(tails))
        dst, o = table.copy(), 0
        for b, n in enumerate(tails):                                # the destination shares the full pages and has tail pages of its own
            dst[b, need[b] - n:need[b]] = spare[o:o + n]
            o += n
        ids = rs.randint(0, 200000, (B, N))
        toks = rs.randint(0, 200000, (B, N))
        for b, (trunk, acc) in enumerate(zip(trunks, _accepted(c))):
            for i in range(1, N):                                    # nothing else is what the target says ...
                toks[b, i] = ids[b, parents[b, i]] + 1
            for k in range(1, min(acc, len(trunk))):                 # ... but the first nodes of the trunk
                toks[b, trunk[k]] = ids[b, trunk[k - 1]]
        s.update(pos=i32(ctx), dst_slots=i32(slots[B:2 * B]), toks=i32(toks), ids=i32(ids), table=i32(table), dst_table=i32(dst),
                 K=bf(N_FULL, total, 2, PAGE, D), V=bf(N_FULL, total, 2, PAGE, D))
        return s
    fork = c["what"] == "fork"
    order = rs.permutation(c["pages"])
    src, dst = ([int(order[0])] * c["n"] if fork else order[:c["n"]].tolist()), order[c["n"] if not fork else 1:][:c["n"]].tolist()
    s.update(K=bf(N_FULL, c["pages"], 2, PAGE, D), V=bf(N_FULL, c["pages"], 2, PAGE, D), src=src, dst=dst, src_t=i32(src).long(), dst_t=i32(dst).long(),
             rows=c["rows"] or None)
    if fork:
        order = rs.permutation(c["slots"])
        ss, ds = [int(order[0])] * c["n"], order[1:][:c["n"]].tolist()
        s.update(ssm=torch.randn(N_LINEAR, c["slots"], HV, DK, DK, generator=g, device="cuda") * 0.1, conv=bf(N_LINEAR, c["slots"], 2, 3, CD), s_src=ss, s_dst=ds,
                 s_src_t=i32(ss).long(), s_dst_t=i32(ds).long())
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _closure(parents):
    """anc [B, N, N] bool: node j is node i or one of its ancestors (rows of unused nodes are empty)."""
    N = parents.shape[1]
    i = torch.arange(N, device=parents.device)
    step = (parents[:, :, None] == i).float() + torch.eye(N, device=parents.device)
    return (torch.matrix_power(step, max(1, N)) > 0) & (parents >= -1)[:, :, None]


def _attn(s):
    c, q, K, V = s["case"], s["q"], s["k_pages"], s["v_pages"]
    B, N, H, KV, P = c["B"], c["N"], c["H"], c["KV"], c["page"]
    parents, ctx, table = s["parents"], s["ctx"].long(), s["table"].long()
    kn, vn = s["k_new"].float().view(B, N, KV, D), s["v_new"].float().view(B, N, KV, D)
    T = c["hi"]
    used = (T + P - 1) // P
    gather = lambda X: X[table[:, :used]].float().transpose(1, 2).reshape(B, KV, used * P, D)  # noqa: E731
    qg = q.float().view(B, N, KV, H // KV, D).permute(0, 2, 3, 1, 4) / 16                          # [B, KV, G, N, D]
    seen = (torch.arange(used * P, device=q.device) < ctx[:, None])[:, None, None, None, :]
    old = (qg @ gather(K)[:, :, None].transpose(-1, -2)).masked_fill(~seen, -math.inf)
    anc = _closure(parents)
    new = (qg @ kn.permute(0, 2, 3, 1)[:, :, None]).masked_fill(~anc[:, None, None], -math.inf)
    top = torch.maximum(old.amax(-1, keepdim=True) if used else torch.full_like(new[..., :1], -math.inf), new.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    po, pn = torch.exp(old - top), torch.exp(new - top)
    o = po @ torch.where(seen[:, :, 0].transpose(-1, -2), gather(V), 0.0)[:, :, None] + pn @ vn.permute(0, 2, 1, 3)[:, :, None]
    total = po.sum(-1, keepdim=True) + pn.sum(-1, keepdim=True)
    o = o / torch.where(total == 0, 1.0, total)
    out = o.permute(0, 3, 1, 2, 4).masked_fill((parents < -1)[:, :, None, None, None], 0.0).reshape(B * N, H, D).to(q.dtype)
    b, n = torch.nonzero(parents >= -1, as_tuple=True)
    at = ctx[b] + n
    page = table[b, at // P]
    K[page, :, at % P] = s["k_new"].view(B, N, KV, D)[b, n]
    V[page, :, at % P] = s["v_new"].view(B, N, KV, D)[b, n]
    return dict(out=out, k_pages=K, v_pages=V)


def _front(rows, w, a, b, A_log, dt_bias):
    """Four conv taps [.., 4, 6144] -> silu -> q, k, v [.., 16, 128] (q, k of unit length, q also / sqrt(128)), log-decay and beta [.., 16]."""
    x = (rows.float() * w.float()).sum(-2)
    x = x * torch.sigmoid(x)
    q, k, v = x.view(*x.shape[:-1], 3, HV, DK).unbind(-3)
    unit = lambda t: t * torch.rsqrt((t * t).sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    a = a.float() + dt_bias
    soft = torch.clamp(a, min=0) + torch.log1p(torch.exp(-a.abs()))
    return unit(q) * DK ** -0.5, unit(k), v, -torch.exp(A_log) * soft, torch.sigmoid(b.float())


def _rule(S0, q, k, v, lg, beta, anc):
    """The gated delta rule for the nodes of a tree, all at once.  S0 [.., H, v, k]; q, k, v [.., N, H, 128]; lg, beta [.., N, H];
    anc [B, 1, N, N]: self and ancestors.  With G the decay summed from the root and M = exp(G_i - G_a) for ancestors a:
    u = beta (v - e^G S0 k) - sum_a beta M (k.k_a) u_a,  y = e^G S0 q + sum_a M (q.k_a) u_a.  Returns y, u, k [.., H, N, 128] and G."""
    q, k, v = (t.transpose(-2, -3) for t in (q, k, v))
    lg, beta = lg.transpose(-1, -2), beta.transpose(-1, -2)
    G = (anc.float() * lg[..., None, :]).sum(-1)
    M = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~anc, -math.inf))
    eye = torch.eye(q.shape[-2], device=q.device)
    X = -(beta[..., None] * M * (k @ k.transpose(-1, -2))) * (1 - eye)
    T = eye + X                                                      # (1 - X)^-1 of a nilpotent X: the powers of X, doubled
    for _ in range(max(0, (q.shape[-2] - 1).bit_length() - 1)):
        X = X @ X
        T = T + T @ X
    grow = torch.exp(G)[..., None]
    u = T @ (beta[..., None] * (v - grow * (k @ S0.transpose(-1, -2))))
    y = grow * (q @ S0.transpose(-1, -2)) + (M * (q @ k.transpose(-1, -2))) @ u
    return y, u, k, G


def _delta(s):
    c, parents = s["case"], s["parents"].long()
    B, N = c["B"], c["N"]
    proj = s["proj"][0].view(B, N, PW)
    slots = s["slots"].long()
    window = s["conv"][0][slots * 2 + (s["pos"].long() & 1)]
    rows = torch.cat([window, proj[..., :CD]], 1)                    # the window's rows are the three tokens before a root
    up = torch.cat([torch.arange(-1, 2, device=proj.device).clamp(min=0).expand(B, 3), torch.where(parents >= 0, parents + 3, 2)], 1)
    p1 = up[:, 3:]
    p2 = up.gather(1, p1)
    p3 = up.gather(1, p2)
    b = torch.arange(B, device=proj.device)[:, None]
    taps = torch.stack([rows[b, p3], rows[b, p2], rows[b, p1], proj[..., :CD]], 2)
    q, k, v, lg, beta = _front(taps, s["conv_w"][0].view(CD, 4).t(), proj[..., PW - HV:], proj[..., PW - 2 * HV:PW - HV], s["A_log"][0], s["dt_bias"][0])
    y = _rule(s["ssm"][0][slots], q, k, v, lg, beta, _closure(s["parents"])[:, None])[0]
    y = y.transpose(-2, -3).masked_fill(~(parents >= -1)[:, :, None, None], 0.0)
    return y.reshape(B * N, KD).to(proj.dtype)


def _accept(parents, toks, ids):
    """Nodes of the path that the target confirms: the first root, then as long as there is one the first child whose token the target chose."""
    B, N = parents.shape
    up = parents.long().clamp(min=0)
    hit = (parents == -1) | ((parents >= 0) & (toks == ids.gather(1, up)))
    earlier = torch.ones(N, N, device=parents.device).tril(-1) > 0
    rival = (parents[:, :, None] == parents[:, None, :]) & hit[:, None, :] & earlier
    good = hit & ~rival.any(-1)
    on = (good[:, None, :] | ~_closure(parents)).all(-1) & (parents >= -1)
    path = torch.where(on, torch.arange(N, device=parents.device), N).sort(1)[0]
    return on.sum(1).int(), torch.where(path == N, -1, path).int()


def _commit(s):
    c = s["case"]
    B, N = c["B"], c["N"]
    n, path = _accept(s["parents"], s["toks"], s["ids"])
    dev = path.device
    slots, dst, pos = s["slots"].long(), s["dst_slots"].long(), s["pos"].long()
    L, E = N_LINEAR, c["depth"]                                      # no path is longer than the trunk
    node = path[:, :E].long().clamp(min=0)
    live = torch.arange(E, device=dev) < n[:, None]
    b = torch.arange(B, device=dev)[:, None]
    x = s["proj"].view(L, B, N, PW)[:, b, node]                      # [L, B, E, 8224]
    rows = torch.cat([s["conv"][:, slots * 2 + (pos & 1)], x[..., :CD]], 2)
    layer = lambda t: t[:, None, None]  # noqa: E731
    q, k, v, lg, beta = _front(rows.unfold(2, 4, 1).transpose(-1, -2), layer(s["conv_w"].view(L, CD, 4).transpose(1, 2)),
                               x[..., PW - HV:], x[..., PW - 2 * HV:PW - HV], layer(s["A_log"]), layer(s["dt_bias"]))
    lg, beta = lg * live[..., None], beta * live[..., None]          # steps behind the path change nothing
    S0 = s["ssm"][:, slots]
    _, u, k, G = _rule(S0, q, k, v, lg, beta, (torch.ones(E, E, device=dev).tril() > 0)[None, None])
    end = G[..., -1:]
    s["ssm"][:, dst] = torch.exp(end)[..., None] * S0 + (torch.exp(end - G)[..., None] * u).transpose(-1, -2) @ k
    s["conv"][:, dst * 2 + ((pos + n) & 1)] = rows[:, b, n[:, None] + torch.arange(3, device=dev)]
    bb, j = torch.nonzero(live, as_tuple=True)
    f, t = pos[bb] + node[bb, j], pos[bb] + j
    fp, tp = s["table"].long()[bb, f // PAGE], s["dst_table"].long()[bb, t // PAGE]
    s["K"][:, tp, :, t % PAGE] = s["K"][:, fp, :, f % PAGE]
    s["V"][:, tp, :, t % PAGE] = s["V"][:, fp, :, f % PAGE]
    return dict(n_path=n, path=path, ssm=s["ssm"], conv=s["conv"], K=s["K"], V=s["V"])


def _copy(s):
    rows = s["rows"] or PAGE
    s["K"][:, s["dst_t"], :, :rows] = s["K"][:, s["src_t"], :, :rows]
    s["V"][:, s["dst_t"], :, :rows] = s["V"][:, s["src_t"], :, :rows]
    if "ssm" not in s:
        return dict(K=s["K"], V=s["V"])
    s["ssm"][:, s["s_dst_t"]] = s["ssm"][:, s["s_src_t"]]
    s["conv"][:, s["s_dst_t"]] = s["conv"][:, s["s_src_t"]]
    return dict(K=s["K"], V=s["V"], ssm=s["ssm"], conv=s["conv"])


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return dict(attn=_attn, delta=_delta, commit=_commit, copy=_copy)[s["op"]](s)


def _own(s):
    from qwen_tailor_b200 import batch, batch_spec
    if s["op"] == "attn":
        out = batch.attn_tree(s["q"], s["k_new"], s["v_new"], s["k_pages"], s["v_pages"], s["table"], s["ctx"], s["parents"])
        return dict(out=out, k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["op"] == "delta":
        return batch_spec.deltanet_tree(s["proj"][0], s["conv"][0], s["conv_w"][0], s["A_log"][0], s["dt_bias"][0], s["ssm"][0], s["slots"], s["pos"], s["parents"])
    if s["op"] == "commit":
        n, path = batch_spec.accept_tree(s["parents"], s["toks"], s["ids"])
        batch_spec.deltanet_commit(s["proj"], s["conv"], s["conv_w"], s["A_log"], s["dt_bias"], s["ssm"], s["slots"], s["pos"], path, n, dst_slots=s["dst_slots"])
        batch.compact_rows([s["K"], s["V"]], s["table"], s["pos"], path, n, dst_table=s["dst_table"], stacked=True)
        return dict(n_path=n, path=path, ssm=s["ssm"], conv=s["conv"], K=s["K"], V=s["V"])
    batch.copy_entries([s["K"], s["V"]], s["dst"], s["src"], rows=s["rows"], stacked=True)
    if "ssm" not in s:
        return dict(K=s["K"], V=s["V"])
    batch.copy_entries([s["ssm"]], s["s_dst"], s["s_src"], stacked=True)
    batch.copy_entries([s["conv"]], s["s_dst"], s["s_src"], stacked=True)
    return dict(K=s["K"], V=s["V"], ssm=s["ssm"], conv=s["conv"])


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _token(rows, w, a, b, A_log, dt_bias):
    """One token: the raw rows t-3 .. t [.., 4, 6144] -> q, k, v [.., 16, 128], decay and beta [.., 16], in 64 bits."""
    x = torch.einsum("...tc,...ct->...c", rows.double(), w.double().unflatten(-1, (CD, 4)))
    x = x / (1 + torch.exp(-x))
    heads = lambda lo: x[..., lo:lo + KD].unflatten(-1, (HV, DK))  # noqa: E731
    q, k = heads(0), heads(KD)
    q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(DK)
    k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    rate = torch.logaddexp(a.double() + dt_bias.double(), torch.zeros((), dtype=torch.float64, device=a.device))
    return q, k, heads(2 * KD), torch.exp(-torch.exp(A_log.double()) * rate), 1 / (1 + torch.exp(-b.double()))


def _advance(S, k, v, g, beta):
    S = S * g[..., None, None]
    d = (v - (S * k[..., None, :]).sum(-1)) * beta[..., None]
    return S + d[..., :, None] * k[..., None, :]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attn":
        B, N, H, KV, P = c["B"], c["N"], c["H"], c["KV"], c["page"]
        parents, ctx = s["parents"].tolist(), s["ctx"].tolist()
        out = torch.zeros(B, N, H, D, dtype=torch.float64, device="cuda")
        kn, vn = s["k_new"].view(B, N, KV, D), s["v_new"].view(B, N, KV, D)
        for b in range(B):
            pages = s["table"][b].long()
            flat = lambda X, t: X[pages[:(t + P - 1) // P]].transpose(0, 1).reshape(KV, -1, D)[:, :t].double()  # noqa: E731
            K, V = flat(s["k_pages"], ctx[b]), flat(s["v_pages"], ctx[b])
            lines = []                                               # the line of every node: its ancestors and itself
            for i, p in enumerate(parents[b]):
                lines.append([] if p < -1 else (lines[p] if p >= 0 else []) + [i])
            mask = torch.zeros(N, N, dtype=torch.bool)
            for i, line in enumerate(lines):
                mask[i, line] = True
            mask = mask.cuda()
            q = s["q"].view(B, N, KV, H // KV, D)[b].double()
            for h in range(KV):
                qh = q[:, h].reshape(-1, D)
                lo, ln = qh @ K[h].t() / 16, qh @ kn[b, :, h].double().t() / 16
                ln = ln.masked_fill(~mask.repeat_interleave(H // KV, 0), -math.inf)
                p = torch.softmax(torch.cat([lo, ln], 1), 1)
                p = torch.where(torch.isnan(p), 0.0, p)              # an unused node of an empty cache sees nothing
                o = p[:, :ctx[b]] @ V[h] + p[:, ctx[b]:] @ vn[b, :, h].double()
                out[b, :, h * (H // KV):(h + 1) * (H // KV)] = o.view(N, H // KV, D)
            out[b, [i for i, line in enumerate(lines) if not line]] = 0                    # nor does it see the cache
            for i, line in enumerate(lines):
                if line:
                    page, row = int(pages[(ctx[b] + i) // P]), (ctx[b] + i) % P
                    s["k_pages"][page, :, row], s["v_pages"][page, :, row] = kn[b, i], vn[b, i]
        return dict(out=out.view(B * N, H, D), k_pages=s["k_pages"], v_pages=s["v_pages"])
    if c["op"] == "delta":
        B, N = c["B"], c["N"]
        parents = s["parents"].cpu()
        slots = s["slots"].long()
        proj = s["proj"][0].view(B, N, PW)
        state = s["ssm"][0][slots].double()[:, None]                 # column 0: before the tree, column 1 + i: after node i
        state = torch.cat([state, torch.zeros(B, N, HV, DK, DK, dtype=torch.float64, device="cuda")], 1)
        window = s["conv"][0][slots * 2 + s["pos"].long() % 2]
        last = torch.cat([window[:, None], torch.zeros(B, N, 3, CD, dtype=torch.bfloat16, device="cuda")], 1)
        y = torch.zeros(B, N, HV, DK, dtype=torch.float64, device="cuda")
        for i in range(N):
            b = torch.nonzero(parents[:, i] >= -1)[:, 0].cuda()
            if not len(b):
                continue
            up = parents[:, i].cuda().long()[b] + 1
            x = proj[b, i]
            rows = torch.cat([last[b, up], x[:, None, :CD]], 1)
            q, k, v, g, beta = _token(rows, s["conv_w"][0], x[:, PW - HV:], x[:, PW - 2 * HV:PW - HV], s["A_log"][0], s["dt_bias"][0])
            S = _advance(state[b, up], k, v, g, beta)
            state[b, i + 1], last[b, i + 1] = S, rows[:, 1:]
            y[b, i] = (S * q[..., None, :]).sum(-1)
        return y.view(B * N, KD)
    if c["op"] == "commit":
        B, N = c["B"], c["N"]
        parents, toks, ids = (s[k].tolist() for k in ("parents", "toks", "ids"))
        pos = s["pos"].tolist()
        proj = s["proj"].view(N_LINEAR, B, N, PW)
        paths, ssm = [], s["ssm"].double()
        for b in range(B):
            path = [parents[b].index(-1)]
            while True:
                here = [i for i in range(N) if parents[b][i] == path[-1] and toks[b][i] == ids[b][path[-1]]]
                if not here:
                    break
                path.append(here[0])
            paths.append(path + [-1] * (N - len(path)))
            a, z = int(s["slots"][b]), int(s["dst_slots"][b])
            S, rows = ssm[:, a], s["conv"][:, 2 * a + pos[b] % 2]
            for i in path:
                x = proj[:, b, i]
                rows = torch.cat([rows[:, -3:], x[:, None, :CD]], 1)
                _, k, v, g, beta = _token(rows, s["conv_w"], x[:, PW - HV:], x[:, PW - 2 * HV:PW - HV], s["A_log"], s["dt_bias"])
                S = _advance(S, k, v, g, beta)
            ssm[:, z], s["conv"][:, 2 * z + (pos[b] + len(path)) % 2] = S, rows[:, -3:]
            for j, i in enumerate(path):
                (fp, fr), (tp, tr) = divmod(pos[b] + i, PAGE), divmod(pos[b] + j, PAGE)
                for X in (s["K"], s["V"]):
                    X[:, int(s["dst_table"][b, tp]), :, tr] = X[:, int(s["table"][b, fp]), :, fr]
        return dict(n_path=torch.tensor([sum(i >= 0 for i in p) for p in paths], dtype=torch.int32), path=torch.tensor(paths, dtype=torch.int32), ssm=ssm,
                    conv=s["conv"], K=s["K"], V=s["V"])
    rows = s["rows"] or PAGE
    for X in (s["K"], s["V"]):
        for d, f in zip(s["dst"], s["src"]):
            X[:, d, :, :rows] = X[:, f, :, :rows]
    if "ssm" not in s:
        return dict(K=s["K"], V=s["V"])
    for X in (s["ssm"], s["conv"]):
        for d, f in zip(s["s_dst"], s["s_src"]):
            X[:, d] = X[:, f]
    return dict(K=s["K"], V=s["V"], ssm=s["ssm"].double(), conv=s["conv"])
