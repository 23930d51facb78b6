"""Tree-of-drafts operators on the GPU against a plain 64-bit implementation."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
HALF = torch.finfo(torch.bfloat16).eps / 2          # a bf16 rounding is off by at most this much of the value


def inv_freq():
    return 1e6 ** (-torch.arange(0, D, 2, device="cuda").float() / D)


def random_parents(B, T, g, absent=False, forest=False):
    par = torch.full((B, T), -2, dtype=torch.int32)
    for b in range(B):
        n = T if not absent else int(torch.randint(0, T + 1, (1,), generator=g))
        for t in range(n):
            lo = -1 if forest or t == 0 else 0
            par[b, t] = int(torch.randint(max(lo, t - 7), max(t, lo + 1), (1,), generator=g)) if t else -1
    return par


def paths_of(par):
    out = []
    for row in par.tolist():
        p = []
        for t, up in enumerate(row):
            p.append([t] if up == -1 else (p[up] + [t] if 0 <= up < t and p[up] else []))
        out.append(p)
    return out


def plan_words(paths, T):
    W = (T + 63) // 64
    depth = torch.tensor([[len(p) - 1 for p in row] for row in paths], dtype=torch.int32)
    mask = torch.zeros(len(paths), T, W, dtype=torch.int64)
    for b, row in enumerate(paths):
        for t, p in enumerate(row):
            for u in p:
                w = 1 << (u % 64)
                mask[b, t, u // 64] += w - (1 << 64) if w >= 1 << 63 else w
    return depth, mask


def attend_64(qb, qg, k, kg, v, paths, lens, w_0, scale):
    """(out, lse, sum of p |v|) in 64 bits; kg None: one class."""
    B, T, H, _ = qb.shape
    rep = H // k.shape[2]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=qb.device)
    absv = torch.zeros_like(out)
    lse = torch.full((B, H, T), -math.inf, dtype=torch.float64, device=qb.device)
    for b in range(B):
        L = lens[b]
        kpos = torch.tensor([*range(L), *(L + len(p) - 1 for p in paths[b])], device=qb.device)
        for t in range(T):
            if not paths[b][t]:
                continue
            rows = torch.tensor([*range(L), *(L + u for u in paths[b][t])], device=qb.device)
            far = L + len(paths[b][t]) - 1 - kpos[rows] > w_0
            kk, vv = k[b, rows].double(), v[b, rows].double()
            s = torch.einsum("grd,jgd->grj", qb[b, t].double().view(-1, rep, D), kk)
            if kg is not None:
                s2 = torch.einsum("grd,jgd->grj", qg[b, t].double().view(-1, rep, D), kg[b, rows].double())
                s = torch.where(far, s2, s)
            s = s * scale
            lse[b, :, t] = torch.logsumexp(s, -1).reshape(-1)
            p = torch.softmax(s, -1)
            out[b, t] = torch.einsum("grj,jgd->grd", p, vv).reshape(H, D)
            absv[b, t] = torch.einsum("grj,jgd->grd", p, vv.abs()).reshape(H, D)
    return out, lse, absv


def check_attention(out, lse, want, absv, want_lse):
    # the output is rounded once and so is every probability that multiplies a value: half a step of each; the rest (fp32
    # sums, exponentials to 1e-4) is below 2^-11 of the values' weighted sum
    bound = HALF * (want.abs() + absv) + 2.0 ** -11 * absv
    assert torch.isfinite(out.float()).all()
    assert ((out.double() - want).abs() <= bound).all(), ((out.double() - want).abs() / bound.clamp(min=1e-30)).max()
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    # a score of 128 products of about unit values is off by at most 128 * 2^-24 * (their absolute sum ~ 100) * scale ~ 7e-5
    assert (lse.double() - want_lse)[~empty].abs().max() <= 2e-4 if (~empty).any() else True


@pytest.mark.parametrize("B, T", [(1, 1), (2, 7), (1, 64), (3, 65), (2, 256)])
def test_draft_tree_equals_the_walk(B, T):
    from jetlm.kernels import draft_ops as d
    g = torch.Generator().manual_seed(B * 1000 + T)
    par = random_parents(B, T, g, absent=B > 1, forest=True)
    tree = d.draft_tree(par.cuda())
    depth, mask = plan_words(paths_of(par), T)
    assert torch.equal(tree.depth.cpu(), depth) and torch.equal(tree.mask.cpu(), mask)
    again = d.draft_tree(par.long().cuda())
    assert torch.equal(again.depth, tree.depth) and torch.equal(again.mask, tree.mask)


def test_draft_tree_takes_bad_links_as_absent_nodes():
    from jetlm.kernels import draft_ops as d
    par = torch.tensor([[-1, 0, 5, 2, -7, 4, 6, 1 << 30, 0]])          # later, own and negative links and what hangs on them
    for t in (par.int(), par.long(), par.long() - (par == -7) * (1 << 40)):
        tree = d.draft_tree(t.cuda())
        assert tree.depth.tolist() == [[0, 1, -1, -1, -1, -1, -1, -1, 1]]
        assert tree.mask.flatten().tolist() == [1, 3, 0, 0, 0, 0, 0, 0, 0b100000001]


CASES = [
    # B, T, H, Hk, lens, rows beyond, w_0, group?, parents kind
    (1, 1, 16, 8, [0], 0, 8, True, "tree"),                # one token, empty cache
    (1, 1, 8, 8, [1], 3, 0, True, "tree"),                 # everything but itself is far
    (1, 5, 32, 8, [127], 0, 64, True, "tree"),             # the tile ends inside the tree
    (1, 4, 16, 8, [128], 9, 1000, True, "tree"),           # nothing is far
    (2, 16, 32, 8, [700, 3], 5, 100, True, "absent"),
    (3, 33, 12, 4, [256, 129, 0], 2, 3, True, "absent"),   # paths longer than w_0: drafted keys in the far class
    (1, 64, 32, 8, [1000], 1, 256, True, "forest"),
    (1, 65, 8, 8, [515], 0, 512, False, "tree"),           # one class
    (2, 130, 16, 8, [385, 77], 7, 40, True, "absent"),
    (1, 256, 8, 1, [300], 0, 30, True, "chain"),           # 2048 query rows on one key head
    (5, 3, 14, 2, [1, 2, 64, 65, 2000], 0, 31, True, "absent"),
    (1, 9, 64, 8, [4099], 0, 2048, True, "tree"),
    (1, 3, 128, 1, [200], 3, 64, True, "tree"),            # one node a row tile
    (2, 40, 10, 2, [150, 300], 0, 90, True, "absent"),     # 25 nodes a row tile, three rows unused
    (40, 2, 8, 8, list(range(0, 400, 10)), 0, 20, True, "tree"),   # more (sample, head) pairs than parts
    # caches so large that the walk counts as a long one, whatever they hold
    (1, 12, 32, 8, [1030], 40000, 300, True, "absent"),
    (1, 70, 32, 8, [700], 40000, 200, True, "forest"),
    (2, 33, 16, 8, [0, 511], 20000, 5, True, "absent"),
    (1, 64, 32, 8, [900], 40000, 64, False, "tree"),
    # so many pairs that most are one segment, which writes the result itself, and some are cut
    (60, 9, 32, 8, list(range(1, 1200, 20)), 0, 200, True, "absent"),
    (48, 40, 16, 4, list(range(0, 960, 20)), 3, 64, True, "absent"),     # two row tiles
    (30, 100, 8, 2, list(range(0, 600, 20)), 0, 50, True, "forest"),     # four row tiles, two CTAs a part
    (300, 1, 2, 1, list(range(300)), 0, 33, True, "absent"),
]


def make(case, seed=0, poison=True):
    B, T, H, Hk, lens, more, w_0, two, kind = case
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gd, device="cuda").bfloat16()        # noqa: E731
    if kind == "chain":
        par = torch.arange(-1, T - 1, dtype=torch.int32)[None].repeat(B, 1)
    else:
        par = random_parents(B, T, g, absent=kind == "absent", forest=kind == "forest")
    rows = max(lens) + T + more
    k, kg, v = rn(B, rows, Hk, D), rn(B, rows, Hk, D), rn(B, rows, Hk, D)
    paths = paths_of(par)
    if poison:      # what a preallocated cache may hold in rows that no node names
        bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda").bfloat16()
        for b in range(B):
            dead = [lens[b] + t for t in range(T) if not paths[b][t]] + list(range(lens[b] + T, rows))
            for t in (k, kg, v):
                t[b, dead] = bad[torch.randint(0, 3, (len(dead), Hk, D), generator=gd, device="cuda")]
    return dict(par=par, paths=paths, lens=lens, qb=rn(B, T, H, D), qg=rn(B, T, H, D), k=k, kg=kg if two else None, v=v, w_0=w_0)


def call(s, **kw):
    from jetlm.kernels import draft_ops as d
    tree = d.draft_tree(s["par"].cuda())
    return d.tree_attention(s["qb"], s["qg"], s["k"], s["v"], tree, torch.tensor(s["lens"], dtype=torch.int32, device="cuda"),
                            w_0=s["w_0"], key_group_rows=s["kg"], **kw)


@pytest.mark.parametrize("case", CASES, ids=[f"B{c[0]}T{c[1]}H{c[2]}x{c[3]}w{c[6]}{c[8]}" for c in CASES])
def test_tree_attention(case):
    s = make(case)
    want, want_lse, absv = attend_64(s["qb"], s["qg"], s["k"], s["kg"], s["v"], s["paths"], s["lens"], s["w_0"], D ** -0.5)
    out, lse = call(s)
    check_attention(out, lse, want, absv, want_lse)


def test_tree_attention_empty_rows_and_any_mask():
    """A mask need not be a tree's: a node that names nothing over an empty cache is zero with lse -inf."""
    from jetlm.kernels import draft_ops as d
    s = make((2, 6, 8, 4, [0, 40], 0, 10, True, "tree"), poison=False)
    mask = torch.zeros(2, 6, 1, dtype=torch.int64)
    mask[:, 2] = 0b000100
    mask[:, 4] = 0b101010                                # not its own node
    depth = torch.tensor([[0, 0, 0, 1, 1, 1]] * 2, dtype=torch.int32)
    tree = d.DraftTree(depth.cuda(), mask.cuda())
    out, lse = d.tree_attention(s["qb"], s["qg"], s["k"], s["v"], tree, torch.tensor([0, 40], dtype=torch.int32, device="cuda"), w_0=10,
                                key_group_rows=s["kg"])
    for b, L in ((0, 0), (1, 40)):
        for t in range(6):
            seen = [*range(L), *(L + u for u in range(6) if (int(mask[b, t, 0]) >> u) & 1)]
            if not seen:
                assert (out[b, t] == 0).all() and (lse[b, :, t] == -math.inf).all()
                continue
            pos = [j if j < L else L + int(depth[b, j - L]) for j in seen]
            far = torch.tensor([L + int(depth[b, t]) - p > 10 for p in pos], device="cuda")
            for h in range(8):
                k, kg, v = (x[b, seen, h // 2].double() for x in (s["k"], s["kg"], s["v"]))
                z = torch.where(far, kg @ s["qg"][b, t, h].double(), k @ s["qb"][b, t, h].double()) * D ** -0.5
                p = torch.softmax(z, 0)
                want, av = p @ v, p @ v.abs()
                assert ((out[b, t, h].double() - want).abs() <= HALF * (want.abs() + av) + 2.0 ** -11 * av).all()
                assert abs(float(lse[b, h, t]) - float(torch.logsumexp(z, 0))) <= 2e-4


def test_tree_attention_large_scores_and_jumping_maximum():
    """Scores of some hundreds, larger and larger towards the end: the running maximum is raised again and again."""
    s = make((1, 8, 16, 8, [1500], 0, 700, True, "tree"), seed=3)
    ramp = torch.linspace(0.1, 30.0, s["k"].shape[1], device="cuda")[None, :, None, None]
    s["k"], s["kg"] = (s["k"].float() * ramp).bfloat16(), (s["kg"].float() * ramp).bfloat16()
    want, want_lse, absv = attend_64(s["qb"], s["qg"], s["k"], s["kg"], s["v"], s["paths"], s["lens"], s["w_0"], D ** -0.5)
    out, lse = call(s)
    # a score of up to 128 * 30 * 4 * 0.09 ~ 1400 in fp32 is off by at most 2^-23 of its terms' absolute sum (~ 1000): 1e-4 a term,
    # which moves a probability by as much again
    bound = HALF * (want.abs() + absv) + 2.0 ** -9 * absv
    assert ((out.double() - want).abs() <= bound).all()
    assert (lse.double() - want_lse).abs().max() <= 2e-3


def test_tree_attention_strides_out_and_devices_state():
    """(B, H, S, D) caches and queries passed as transposed views, a strided `out`, and neighbours left alone."""
    s = make((2, 10, 16, 4, [333, 20], 4, 50, True, "absent"), seed=5)
    ref, ref_lse = call(s)
    hm = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)       # noqa: E731
    t = dict(s, qb=hm(s["qb"]), qg=hm(s["qg"]), k=hm(s["k"]), kg=hm(s["kg"]), v=hm(s["v"]))
    big = torch.full((2, 10, 16, 3 * D), 7.0, device="cuda", dtype=torch.bfloat16)
    out, lse = call(t, out=big[..., D:2 * D])
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    assert (big[..., :D] == 7).all() and (big[..., 2 * D:] == 7).all()
    assert torch.equal(call(s, return_lse=False), ref)


def test_tree_attention_side_stream_graph_and_repeats():
    """Results do not vary from run to run, on another stream, or replayed from a graph whose lengths and tree change."""
    from jetlm.kernels import draft_ops as d
    s = make((2, 12, 32, 8, [900, 411], 60, 128, True, "absent"), seed=8)
    ref, ref_lse = call(s)
    for _ in range(3):
        again, again_lse = call(s)
        assert torch.equal(again, ref) and torch.equal(again_lse, ref_lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, _ = call(s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref)
    par, lens = s["par"].cuda(), torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree = d.draft_tree(par)
        g_out, g_lse = d.tree_attention(s["qb"], s["qg"], s["k"], s["v"], tree, lens, w_0=s["w_0"], key_group_rows=s["kg"])
    lens.copy_(torch.tensor(s["lens"], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g_out, ref) and torch.equal(g_lse, ref_lse)
    s2 = make((2, 12, 32, 8, [900, 411], 60, 128, True, "tree"), seed=8, poison=False)
    for name in ("qb", "qg", "k", "kg", "v"):
        s[name].copy_(s2[name])
    par.copy_(s2["par"])
    lens.copy_(torch.tensor([17, 960], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want, want_lse = call(dict(s2, lens=[17, 960]))
    assert torch.equal(g_out, want) and torch.equal(g_lse, want_lse)


def test_tree_attention_lengths_are_clamped_to_the_cache():
    s = make((1, 4, 8, 8, [60], 0, 16, True, "tree"), poison=False)
    ref, _ = call(s)
    s["lens"] = [10 ** 6]
    out, _ = call(s)
    assert torch.equal(out, ref)
    s["lens"] = [-5]
    a, _ = call(s)
    s["lens"] = [0]
    b, _ = call(s)
    assert torch.equal(a, b)


def test_single_node_equals_the_decode_operator():
    """A tree of one node is a decode step: the same result as decode_segments within both operators' own bounds."""
    from jetlm.kernels import jetlong_ops as ops
    s = make((1, 1, 32, 8, [5000], 0, 1024, True, "tree"), seed=2, poison=False)
    out, lse = call(s)
    L = 5001
    far = L - 1 - 1024
    segs = [ops.KvSegment(s["kg"][:, :far], s["v"][:, :far], q_class=1), ops.KvSegment(s["k"][:, far:L], s["v"][:, far:L], q_class=0)]
    ref, ref_lse = ops.decode_segments([s["qb"], s["qg"]], segs)
    assert (out.float() - ref.float()).abs().max() <= 4 * HALF * s["v"][:, :L].float().abs().max()
    assert (lse - ref_lse).abs().max() <= 4e-4


@pytest.mark.parametrize("B, T, H, Hk, lens, G", [(1, 1, 16, 8, [0], 4), (2, 9, 32, 8, [130000, 77], 4), (3, 64, 8, 4, [5, 4000, 90], 1),
                                                  (1, 200, 12, 4, [1000], 32)])
def test_tree_append_has_the_bits_of_norm_rope(B, T, H, Hk, lens, G):
    """Every node's query and key are what jl_norm_rope writes for a token at the node's position, and the other cache rows stay."""
    from jetlm.kernels import draft_ops as d, jetlong_ops as ops
    g = torch.Generator().manual_seed(T)
    gd = torch.Generator(device="cuda").manual_seed(T)
    rn = lambda *s: torch.randn(*s, generator=gd, device="cuda").bfloat16()        # noqa: E731
    par = random_parents(B, T, g, absent=B > 1, forest=True)
    paths = paths_of(par)
    rows = max(lens) + T + 2
    qkv = rn(B, T, H + 2 * Hk, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    qw, kw, inv = rn(D), rn(D), inv_freq()
    kc, vc, kgc = (rn(B, Hk, rows, D).transpose(1, 2) for _ in range(3))
    want_k, want_v, want_g = kc.clone(), vc.clone(), kgc.clone()
    tree = d.draft_tree(par.cuda())
    qb, qg = d.tree_append(q, k, v, qw, kw, inv, kc, vc, tree, torch.tensor(lens, dtype=torch.int32, device="cuda"), q_eps=1e-6, k_eps=1e-5,
                           group_size=G, key_group_rows=kgc if G > 1 else None)
    assert G > 1 or qg is qb
    for b in range(B):
        for t in range(T):
            if not paths[b][t]:
                assert (qb[b, t] == 0).all() and (qg[b, t] == 0).all()
                continue
            pos, at, row = lens[b] + len(paths[b][t]) - 1, (slice(b, b + 1), slice(t, t + 1)), lens[b] + t
            w_qb, w_qg = ops.norm_rope(q[at], qw, inv, eps=1e-6, pos0=pos, group_size=G)
            w_kb, w_kg = ops.norm_rope(k[at], kw, inv, eps=1e-5, pos0=pos, group_size=G)
            assert torch.equal(qb[at], w_qb) and torch.equal(qg[at], w_qg)
            want_k[b, row], want_v[b, row] = w_kb[0, 0], v[b, t]
            if G > 1:
                want_g[b, row] = w_kg[0, 0]
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v) and torch.equal(kgc, want_g)


def test_tree_append_writes_no_row_past_the_cache():
    from jetlm.kernels import draft_ops as d
    rn = lambda *s: torch.randn(*s, device="cuda").bfloat16()        # noqa: E731
    whole_k, whole_v = rn(1, 20, 2, D), rn(1, 20, 2, D)
    keep_k, keep_v = whole_k.clone(), whole_v.clone()
    tree = d.draft_tree(torch.tensor([[-1, 0, 1, 2]], dtype=torch.int32, device="cuda"))
    args = (rn(1, 4, 4, D), rn(1, 4, 2, D), rn(1, 4, 2, D), rn(D), rn(D), inv_freq(), whole_k[:, :12], whole_v[:, :12], tree)
    d.tree_append(*args, torch.tensor([10], dtype=torch.int32, device="cuda"), q_eps=1e-6, k_eps=1e-6)
    assert torch.equal(whole_k[:, 12:], keep_k[:, 12:]) and torch.equal(whole_v[:, 12:], keep_v[:, 12:])
    assert torch.equal(whole_k[:, :10], keep_k[:, :10]) and not torch.equal(whole_k[:, 10:12], keep_k[:, 10:12])
    whole_k.copy_(keep_k)
    d.tree_append(*args, torch.tensor([-3], dtype=torch.int32, device="cuda"), q_eps=1e-6, k_eps=1e-6)
    assert torch.equal(whole_k, keep_k)


@pytest.mark.parametrize("B, Hk, n, group", [(1, 1, 1, False), (1, 8, 5, True), (3, 4, 9, True), (4, 9, 256, False), (2, 2, 37, True)])
def test_tree_keep_moves_the_path_and_nothing_else(B, Hk, n, group):
    from jetlm.kernels import draft_ops as d
    g = torch.Generator().manual_seed(B * 1000 + n)
    rows, T = 600, 256
    bufs = [torch.randn(B, rows, Hk, 128, generator=g).cuda().bfloat16() for _ in range(2)]
    bufs.insert(1, torch.randn(B, Hk, rows, 128, generator=g).cuda().bfloat16().transpose(1, 2))      # values head-major
    lens = torch.tensor({1: [17], 2: [11, 300], 3: [5, 0, 344], 4: [1, 344, 77, 340]}[B], dtype=torch.int32)
    path = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):
        k = n if b == 0 else int(torch.randint(0, n + 1, (1,), generator=g))
        path[b, :k] = torch.randperm(T, generator=g)[:k].sort().values.int()
    want = [x.clone() for x in bufs]
    for b in range(B):
        keep = path[b][path[b] >= 0].long()
        for w, x in zip(want, bufs):
            w[b, int(lens[b]): int(lens[b]) + len(keep)] = x[b, (int(lens[b]) + keep).cuda()]
    d.tree_keep(bufs[0], bufs[1], path.cuda(), lens.cuda(), key_group_rows=bufs[2] if group else None)
    for i, (w, x) in enumerate(zip(want, bufs)):
        if i < 2 or group:
            assert torch.equal(x, w), i


def test_tree_keep_stops_at_the_end_of_a_path_or_cache():
    from jetlm.kernels import draft_ops as d
    x = torch.randn(4, 64, 2, 128, generator=torch.Generator().manual_seed(3)).cuda().bfloat16()
    y, before = x.clone(), x.clone()
    path = torch.tensor([[1, 3, 3, 5], [2, 4, 1, 7], [0, 2, 1 << 30, 2000000000], [-5, 1, 2, 3]], dtype=torch.int32).cuda()
    lens = torch.tensor([10, 20, 60, 5], dtype=torch.int32).cuda()
    d.tree_keep(x, y, path, lens)                       # an entry that repeats, falls, leaves the cache, or is none
    want = before.clone()
    want[0, 10], want[0, 11] = before[0, 11], before[0, 13]
    want[1, 20], want[1, 21] = before[1, 22], before[1, 24]
    want[2, 60], want[2, 61] = before[2, 60], before[2, 62]
    assert torch.equal(x, want) and torch.equal(y, want)
    d.tree_keep(x, y, path, torch.tensor([-3, 64, 63, 1 << 30], dtype=torch.int32).cuda())       # lengths outside the cache
    assert torch.equal(x, want) and torch.equal(y, want)


def test_tree_attention_whole_segments_into_strided_out():
    """Results that a segment writes itself: into a view, without an LSE, and the same bits with one; what lies beside stays."""
    case = (60, 9, 32, 8, list(range(1, 1200, 20)), 0, 200, True, "absent")
    s = make(case)
    ref, _ = call(s)
    wide = torch.full((60, 9, 40, 136), 7.0, device="cuda").bfloat16()
    out = wide[:, :, 4:36, :128]
    assert call(s, out=out, return_lse=False) is out
    assert torch.equal(out, ref)
    wide[:, :, 4:36, :128] = 7.0
    assert (wide == 7.0).all()
