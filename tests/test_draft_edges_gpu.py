"""Tree-of-drafts operators at the edges: at the end of a cache, with NaN in the queries, without samples."""
import math

import pytest
import torch

from test_draft_ops_gpu import D, HALF, attend_64, call, check_attention, inv_freq, make, paths_of

pytestmark = pytest.mark.gpu


def full_cache(rows, T, H, Hk, present, w_0, two, seed, spare):
    """Sample b has present[b] nodes of T places and a cache that they fill to the last row (to `spare` rows from it for the last sample)."""
    B = len(present)
    s = make((B, T, H, Hk, [rows - T] * B, 0, w_0, two, "tree"), seed=seed, poison=False)
    assert s["k"].shape[1] == rows
    for b, n in enumerate(present):
        s["par"][b, n:] = -2
    s["paths"] = paths_of(s["par"])
    s["lens"] = [rows - n for n in present]
    s["lens"][-1] -= spare
    for b, n in enumerate(present):                   # rows that hold nothing
        for t in (s["k"], s["kg"], s["v"]):
            if t is not None:
                t[b, s["lens"][b] + n:] = math.nan
    return s


@pytest.mark.parametrize("w_0", [0, 5, 100, 5000])
@pytest.mark.parametrize("rows, T, H, Hk, present, two", [
    (300, 40, 16, 8, [40, 10, 1, 0, 7], True), (256, 16, 32, 8, [16, 3, 0, 5], True), (384, 130, 8, 8, [130, 64, 2, 1], True),
    (129, 9, 8, 2, [1, 0, 9, 2], False), (64, 64, 12, 4, [0, 64, 1, 30], True), (1300, 70, 32, 8, [5, 70, 33, 3], True)])
def test_nodes_that_reach_the_last_row_of_the_cache(rows, T, H, Hk, present, two, w_0):
    """A padded batch whose places do not all fit, but whose nodes do: every sample is attended where its nodes are."""
    s = full_cache(rows, T, H, Hk, present, w_0, two, seed=rows + w_0, spare=2 if rows > T else 0)
    want, want_lse, absv = attend_64(s["qb"], s["qg"], s["k"], s["kg"], s["v"], s["paths"], s["lens"], w_0, D ** -0.5)
    out, lse = call(s)
    check_attention(out, lse, want, absv, want_lse)


def test_append_and_attention_agree_on_a_full_cache():
    """Nodes written by tree_append into the last rows are attended where they were written."""
    from jetlm.kernels import draft_ops as d
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()        # noqa: E731
    par = torch.full((2, 12), -2, dtype=torch.int32)
    par[0, :3], par[1, :12] = torch.tensor([-1, 0, 0]), torch.arange(-1, 11)
    lens = [97, 60]
    kc, vc, kg = rn(2, 100, 4, D), rn(2, 100, 4, D), rn(2, 100, 4, D)
    tree, dl = d.draft_tree(par.cuda()), torch.tensor(lens, dtype=torch.int32, device="cuda")
    qb, qg = d.tree_append(rn(2, 12, 8, D), rn(2, 12, 4, D), rn(2, 12, 4, D), rn(D), rn(D), inv_freq(), kc, vc, tree, dl, q_eps=1e-6, k_eps=1e-6,
                           group_size=3, key_group_rows=kg)
    want, want_lse, absv = attend_64(qb, qg, kc, kg, vc, paths_of(par), lens, 20, D ** -0.5)
    out, lse = d.tree_attention(qb, qg, kc, vc, tree, dl, w_0=20, key_group_rows=kg)
    check_attention(out, lse, want, absv, want_lse)


def test_a_node_whose_row_is_past_the_cache_is_an_absent_one():
    """Its key has no place: it sees nothing (zero, lse -inf), nobody sees it, and the nodes before it are as they are without it."""
    s = make((2, 6, 8, 4, [94, 94], 0, 30, True, "chain"), seed=4, poison=False)      # 100 rows
    s["lens"] = [97, 100]
    s["paths"] = [[p if t < 3 else [] for t, p in enumerate(s["paths"][0])], [[] for _ in s["paths"][1]]]
    want, want_lse, absv = attend_64(s["qb"], s["qg"], s["k"], s["kg"], s["v"], s["paths"], s["lens"], 30, D ** -0.5)
    out, lse = call(s)
    check_attention(out, lse, want, absv, want_lse)


@pytest.mark.parametrize("case", [
    (1, 5, 16, 8, [200], 0, 60, True, "chain"), (1, 12, 32, 8, [9000], 3, 3000, True, "chain"), (1, 64, 32, 8, [20000], 0, 700, True, "forest"),
    (40, 4, 8, 8, list(range(10, 410, 10)), 0, 33, True, "chain"), (1, 16, 32, 8, [3000], 60000, 900, True, "tree"), (2, 80, 32, 8, [5000, 77], 0, 50, False, "tree")],
    ids=["whole", "split", "two_tiles", "many", "long_form", "three_tiles"])
def test_a_query_of_nan_gives_nan(case):
    """As in the plain form; no other row notices."""
    s = make(case, seed=9)
    ref, ref_lse = call(s)
    b, t, h = case[0] - 1, 2, 1
    s["qb"][b, t, h], s["qg"][b, t, h] = math.nan, math.nan
    out, lse = call(s)
    assert torch.isnan(out[b, t, h]).all() and torch.isnan(lse[b, h, t])
    out[b, t, h], lse[b, h, t] = ref[b, t, h], ref_lse[b, h, t]
    assert torch.equal(out, ref) and torch.equal(lse, ref_lse)


def test_a_score_of_nan_in_one_class_only():
    """NaN in the far query alone: rows with far keys are NaN, the others are not."""
    s = make((1, 3, 8, 8, [50], 0, 30, True, "chain"), seed=3, poison=False)
    ref, ref_lse = call(s)
    s["qg"][0, 1] = math.nan
    out, lse = call(s)
    assert torch.isnan(out[0, 1]).all() and torch.isnan(lse[0, :, 1]).all()
    assert torch.equal(out[0, [0, 2]], ref[0, [0, 2]]) and torch.equal(lse[0, :, [0, 2]], ref_lse[0, :, [0, 2]])
    s["w_0"] = 1000
    assert torch.isfinite(call(s)[0]).all()


def test_no_samples():
    from jetlm.kernels import draft_ops as d
    z = lambda *s: torch.empty(*s, device="cuda", dtype=torch.bfloat16)        # noqa: E731
    lens = torch.empty(0, dtype=torch.int32, device="cuda")
    tree = d.draft_tree(torch.empty(0, 3, dtype=torch.int32, device="cuda"))
    k, v = z(0, 20, 2, D), z(0, 20, 2, D)
    qb, qg = d.tree_append(z(0, 3, 4, D), z(0, 3, 2, D), z(0, 3, 2, D), torch.ones(D, device="cuda").bfloat16(), torch.ones(D, device="cuda").bfloat16(),
                           inv_freq(), k, v, tree, lens, q_eps=1e-6, k_eps=1e-6, group_size=2)
    assert qb.shape == qg.shape == (0, 3, 4, D)
    out, lse = d.tree_attention(qb, qg, k, v, tree, lens, w_0=4)
    assert out.shape == (0, 3, 4, D) and lse.shape == (0, 4, 3)
    d.tree_keep(k, v, torch.empty(0, 3, dtype=torch.int32, device="cuda"), lens)
