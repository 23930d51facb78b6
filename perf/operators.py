"""What is timed of the drafted-token and vocabulary-head operators: their cases, inputs, plain forms and exact values.

Four operators, in the order in which a step that verifies drafted tokens on a long cache runs them:

  append   `draft_ops.draft_tree` + `draft_ops.tree_append`: ancestor masks and depths of a tree of drafted tokens from its
           parent links, then per-head RMSNorm and RoPE of the drafted queries and keys at their tree positions, the
           regrouped copies, and the writes into the cache rows behind the committed ones
  attend   `draft_ops.tree_attention`: every drafted token against the whole cache and its own ancestors, two position classes
  score    `head_ops.token_scores`: log-probability of a given next token and the most likely one for every row, without logits
  loss     `head_ops.linear_cross_entropy`: the mean loss over a large vocabulary and both its gradients, without logits

`own` chooses between the plain forms (elementary torch operations, 32 bits or more) and the framework's calls.
"""
import math

import torch

own = False

DEV = "cuda"
D = 128                     # head size of every model configuration here
VOCAB = 151936


def listed():
    return [
        # one short conversation on the 1.7B geometry, four drafted tokens: launch latency is all there is
        dict(name="attend_short", op="attend", batch=1, ctx=1037, nodes=4, heads=16, kv_heads=8, w_0=256, group=2, ragged=False),
        # the decode benchmark's context with a small tree of drafts: one pass over the cache
        dict(name="attend_131072_t16", op="attend", batch=1, ctx=131056, nodes=16, heads=32, kv_heads=8, w_0=32768, group=4, ragged=False),
        # the same with a wide tree: 256 query rows for every key head, the products weigh as much as the reads
        dict(name="attend_131072_t64", op="attend", batch=1, ctx=131008, nodes=64, heads=32, kv_heads=8, w_0=32768, group=4, ragged=False),
        # a served batch: other lengths and node counts for every sample, the small near window of the model configurations
        dict(name="attend_ragged_b8", op="attend", batch=8, ctx=32001, nodes=23, heads=32, kv_heads=8, w_0=2048, group=3, ragged=True),
        # one drafted chain step of one sample
        dict(name="append_t5", op="append", batch=1, ctx=1500, nodes=5, heads=16, kv_heads=8, w_0=256, group=2, ragged=False),
        # wide trees of a served batch, far positions
        dict(name="append_t64_b8", op="append", batch=8, ctx=4000, nodes=64, heads=32, kv_heads=8, w_0=2048, group=4, ragged=True),
        # the greedy choice after one decoded token: one row against the whole vocabulary
        dict(name="score_1", op="score", rows=1, hidden=2048, vocab=VOCAB, ignored=0.0, top=True),
        # the rows of a drafted tree
        dict(name="score_49", op="score", rows=49, hidden=4096, vocab=VOCAB, ignored=0.0, top=True),
        # the log-likelihood of a window of a book
        dict(name="score_8191", op="score", rows=8191, hidden=4096, vocab=VOCAB, ignored=0.0, top=False),
        # a small training step with an odd vocabulary
        dict(name="loss_127", op="loss", rows=127, hidden=2048, vocab=50257, ignored=0.0),
        # a window of which the prompt's tokens are left out of the loss
        dict(name="loss_1000_masked", op="loss", rows=1000, hidden=4096, vocab=VOCAB, ignored=0.4),
        # a training step on the 4B head
        dict(name="loss_4096", op="loss", rows=4096, hidden=2560, vocab=VOCAB, ignored=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "score", "loss"])
    if op in ("attend", "append"):
        heads, kv = rng.choice([(16, 8), (32, 8), (32, 8), (8, 8), (12, 4), (64, 8)])
        batch = rng.choice([1, 1, 1, 2, 3, 8])
        nodes = _log(rng, 1, 128)
        ctx = _log(rng, 1, 131008) if op == "attend" else _log(rng, 1, 4000)
        if op == "attend":
            ctx = max(1, min(ctx, int(131008 * 64 * 32 / (batch * nodes * heads)), 262144 // batch))
        return dict(op=op, batch=batch, ctx=ctx, nodes=nodes, heads=heads, kv_heads=kv, w_0=_log(rng, 1, 32768),
                    group=rng.choice([1, 2, 3, 4, 8]), ragged=batch > 1 and rng.random() < 0.7)
    hidden = rng.choice([512, 1024, 2048, 2560, 4096, 1032, 2056])
    vocab = rng.choice([VOCAB, VOCAB, 32000, 50257, _log(rng, 1000, 150000)])
    if op == "score":
        rows = min(_log(rng, 1, 8191), int(8191 * 4096 * VOCAB / (hidden * vocab)))
        return dict(op=op, rows=rows, hidden=hidden, vocab=vocab, ignored=rng.choice([0.0, 0.1]), top=rows <= 128)
    rows = min(_log(rng, 1, 4096), int(4096 * 2560 * VOCAB / (hidden * vocab)))
    return dict(op=op, rows=rows, hidden=hidden, vocab=vocab, ignored=rng.choice([0.0, 0.1, 0.5]))


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------

def _tree(case, g):
    """Random parent links (B, T): node 0 is the last accepted token (its parent is the committed context, -1), every other
    node hangs on an earlier one; -2 marks the places behind a sample's last node."""
    B, T = case["batch"], case["nodes"]
    lo = torch.rand(B, T, generator=g) * torch.arange(T)
    par = torch.maximum(lo.floor(), torch.arange(T) - 9.0).long().clamp(min=0)
    par = torch.minimum(par, (torch.arange(T) - 1).clamp(min=0))
    par[:, 0] = -1
    if case["ragged"]:
        n = torch.randint(max(1, T // 2), T + 1, (B, 1), generator=g)
        par = torch.where(torch.arange(T)[None] < n, par, torch.tensor(-2))
    return par


def _closure(par):
    """(depth (B,T), sees (B,T,T) bool) of parent links: sees[i, j] where j is i or an ancestor of i."""
    B, T = par.shape
    step = torch.eye(T, dtype=torch.float64, device=par.device)[None] + (par[:, :, None] == torch.arange(T, device=par.device))
    sees = (torch.linalg.matrix_power(step, max(T, 1)) > 0.5) & (par > -2)[:, :, None]
    return sees.sum(-1) - 1, sees


def _words(sees):
    """The rows of `sees` as little-endian 64-bit words."""
    B, T, _ = sees.shape
    W = (T + 63) // 64
    bits = torch.zeros(B, T, W * 64, dtype=torch.int64, device=sees.device)
    bits[:, :, :T] = sees.long()
    return (bits.view(B, T, W, 64) << torch.arange(64, device=sees.device)).sum(-1)


def prepare(case, seed):
    g = torch.Generator().manual_seed(int(seed))
    gd = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=gd, device=DEV)  # noqa: E731
    s = dict(case=case)
    if case["op"] in ("attend", "append"):
        B, T, H, Hk = case["batch"], case["nodes"], case["heads"], case["kv_heads"]
        lens = torch.full((B,), case["ctx"])
        if case["ragged"]:
            lens = (lens * (0.25 + 0.75 * torch.rand(B, generator=g))).long().clamp(min=1)
            lens[0] = case["ctx"]
        rows = case["ctx"] + T + 3                     # a preallocated cache has rows to spare
        par = _tree(case, g)
        depth, sees = _closure(par)
        s.update(lens=lens.int().to(DEV), parents=par.int().to(DEV), inv_freq=1e6 ** (-torch.arange(0, D, 2, device=DEV).float() / D))
        # the cache buffers of one layer, token-major; their rows hold keys that were rotated when they were written
        s["k_cache"], s["v_cache"] = randn(B, rows, Hk, D).bfloat16(), randn(B, rows, Hk, D).bfloat16()
        s["kg_cache"] = randn(B, rows, Hk, D).bfloat16() if case["group"] > 1 else None
        if case["op"] == "attend":
            s.update(depth=depth.int().to(DEV), mask=_words(sees).to(DEV))
            s["q_base"] = randn(B, T, H, D).bfloat16()
            s["q_group"] = randn(B, T, H, D).bfloat16() if case["group"] > 1 else s["q_base"]
        else:                                          # rows of one fused projection, so head rows of q, k, v are strided views
            qkv = randn(B, T, H + 2 * Hk, D).bfloat16()
            s["q"], s["k"], s["v"] = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
            s["q_weight"], s["k_weight"] = (1 + 0.1 * randn(D)).bfloat16(), (1 + 0.1 * randn(D)).bfloat16()
        return s
    N, Hd, V = case["rows"], case["hidden"], case["vocab"]
    w = (0.02 * randn(V, Hd)).bfloat16()
    labels = torch.randint(0, V, (N,), generator=g)
    # final hidden states: between no idea of the next token and near certainty of it
    sure = (torch.rand(N, 1, generator=g) * 0.25).to(DEV)
    h = (randn(N, Hd) + sure * math.sqrt(4096 / Hd) * 50.0 * w[labels.to(DEV)].float()).bfloat16()
    if case["ignored"] > 0:
        labels[torch.rand(N, generator=g) < case["ignored"]] = -100
        labels[-1] = 0                                 # a loss over nothing has no mean
    s.update(hidden=h, weight=w, labels=labels.to(DEV))
    if case["op"] == "loss":
        s["hidden"].requires_grad_(True)
        s["weight"].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------------------------

def _key_rows(s):
    """Per cache row: its position, whether it holds a drafted node and which, for every sample (B, R)."""
    B, R = s["k_cache"].shape[:2]
    T = s["case"]["nodes"]
    row = torch.arange(R, device=DEV)[None].expand(B, R)
    node = row - s["lens"].long()[:, None]
    return row, node, (node >= 0) & (node < T)


def _attend(s):
    c = s["case"]
    B, T, H, Hk = c["batch"], c["nodes"], c["heads"], c["kv_heads"]
    row, node, drafted = _key_rows(s)
    node = node.clamp(0, T - 1)
    depth = s["depth"].long()
    kpos = torch.where(drafted, s["lens"].long()[:, None] + depth.gather(1, node), row)                       # (B, R)
    qpos = s["lens"].long()[:, None] + depth                                                                  # (B, T)
    word = s["mask"].gather(2, (node // 64)[:, None].expand(B, T, -1))
    bit = ((word >> (node % 64)[:, None]) & 1).bool()                                                         # (B, T, R)
    sees = torch.where(drafted[:, None], bit, (row < s["lens"].long()[:, None])[:, None]) & (depth >= 0)[:, :, None]
    far = qpos[:, :, None] - kpos[:, None] > c["w_0"]

    def scores(q, k):
        q = q.float().view(B, T, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
        return (q @ k.float().permute(0, 2, 3, 1)).view(B, Hk, H // Hk, T, -1) * D ** -0.5

    sc = scores(s["q_base"], s["k_cache"])
    if s["kg_cache"] is not None:
        sc = torch.where(far[:, None, None], scores(s["q_group"], s["kg_cache"]), sc)
    sc = sc.masked_fill(~sees[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = (sc - top).exp_()
    total = p.sum(-1, keepdim=True)
    out = p.view(B, Hk, -1, p.shape[-1]) @ s["v_cache"].float().permute(0, 2, 1, 3)
    out = out.view(B, Hk, H // Hk, T, D) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + total.log()).squeeze(-1).reshape(B, H, T)
    return dict(out=out.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).bfloat16(), lse=lse)


def _rotated(x, pos, inv_freq):
    """x (B, T, heads, D) in 32 bits at integer positions pos (B, T); angles of far positions need 64 bits."""
    ang = pos.double()[:, :, None, None] * inv_freq.double()
    cos, sin = ang.cos().float(), ang.sin().float()
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _normed(x, weight, eps):
    """The model's norm: its result has the storage type, and so has the value that its weight multiplies."""
    x = x.float()
    unit = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return (weight.float() * unit.to(weight.dtype).float()).to(weight.dtype).float()


def _append(s):
    c = s["case"]
    B, T = c["batch"], c["nodes"]
    depth, sees = _closure(s["parents"].long())
    pos = s["lens"].long()[:, None] + depth
    present = depth >= 0
    q, k = _normed(s["q"], s["q_weight"], 1e-6), _normed(s["k"], s["k_weight"], 1e-6)
    keep = present[:, :, None, None]
    out = dict(depth=depth.int(), mask=_words(sees))
    out["q_base"] = torch.where(keep, _rotated(q, pos, s["inv_freq"]), 0.0).bfloat16()
    b, t = present.nonzero(as_tuple=True)
    at = (b, s["lens"].long()[b] + t)
    s["k_cache"][at] = _rotated(k, pos, s["inv_freq"]).bfloat16()[b, t]
    s["v_cache"][at] = s["v"][b, t]
    if s["kg_cache"] is not None:
        grouped = torch.div(pos, c["group"], rounding_mode="floor")
        out["q_group"] = torch.where(keep, _rotated(q, grouped, s["inv_freq"]), 0.0).bfloat16()
        s["kg_cache"][at] = _rotated(k, grouped, s["inv_freq"]).bfloat16()[b, t]
        out["kg_cache"] = s["kg_cache"]
    return dict(out, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _nll(s):
    """(loss per row with 0 at ignored ones, logsumexp, logits, labels that count) in 32 bits."""
    logits = s["hidden"].detach().float() @ s["weight"].detach().float().T
    top = logits.amax(-1, keepdim=True)
    lse = (top + (logits - top).exp().sum(-1, keepdim=True).log()).squeeze(-1)
    counts = s["labels"] >= 0
    picked = logits.gather(1, s["labels"].clamp(min=0)[:, None]).squeeze(1)
    return torch.where(counts, lse - picked, torch.zeros_like(lse)), lse, logits, counts


def _score(s):
    nll, lse, _, _ = _nll(s)
    out = dict(nll=nll, lse=lse)
    if s["case"]["top"]:                               # two logits may be closer than 32 bits tell apart
        out["top"] = (s["hidden"].double() @ s["weight"].double().T).argmax(-1)
    return out


def _loss(s):
    nll, lse, logits, counts = _nll(s)
    n = counts.sum()
    p = logits.sub_(lse[:, None]).exp_()
    p.scatter_add_(1, s["labels"].clamp(min=0)[:, None], -torch.ones_like(lse)[:, None])
    p *= (counts.float() / n)[:, None]
    dh, dw = p @ s["weight"].detach().float(), p.T @ s["hidden"].detach().float()
    return dict(loss=nll.sum() / n, d_hidden=dh.bfloat16(), d_weight=dw.bfloat16())


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------

def _framework():
    import os
    import sys
    package = os.path.join(os.getcwd(), "jet-long_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from jetlm.kernels import draft_ops, head_ops
    return draft_ops, head_ops


def run(state):
    s, c = state, state["case"]
    if own:
        draft_ops, head_ops = _framework()
        if c["op"] == "attend":
            out, lse = draft_ops.tree_attention(s["q_base"], s["q_group"], s["k_cache"], s["v_cache"],
                                                draft_ops.DraftTree(s["depth"], s["mask"]), s["lens"], w_0=c["w_0"],
                                                key_group_rows=s["kg_cache"])
            return dict(out=out, lse=lse)
        if c["op"] == "append":
            tree = draft_ops.draft_tree(s["parents"])
            q_base, q_group = draft_ops.tree_append(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["inv_freq"],
                                                    s["k_cache"], s["v_cache"], tree, s["lens"], q_eps=1e-6, k_eps=1e-6,
                                                    group_size=c["group"], key_group_rows=s["kg_cache"])
            out = dict(depth=tree.depth, mask=tree.mask, q_base=q_base, k_cache=s["k_cache"], v_cache=s["v_cache"])
            return dict(out, q_group=q_group, kg_cache=s["kg_cache"]) if c["group"] > 1 else out
        if c["op"] == "score":
            got = head_ops.token_scores(s["hidden"], s["weight"], s["labels"], top=c["top"])
            out = dict(nll=got.nll, lse=got.lse)
            return dict(out, top=got.top) if c["top"] else out
        loss = head_ops.linear_cross_entropy(s["hidden"], s["weight"], s["labels"])
        dh, dw = torch.autograd.grad(loss, [s["hidden"], s["weight"]])
        return dict(loss=loss.detach(), d_hidden=dh, d_weight=dw)
    with torch.no_grad():
        return dict(attend=_attend, append=_append, score=_score, loss=_loss)[c["op"]](s)


def work(case):
    c = case
    if c["op"] in ("attend", "append"):
        B, T, H, Hk = c["batch"], c["nodes"], c["heads"], c["kv_heads"]
        two = 2 if c["group"] > 1 else 1
        if c["op"] == "append":                        # q, k, v in; q (and its regrouped copy) out; the cache rows out
            return dict(bytes=B * T * D * 2.0 * ((H + 2 * Hk) + two * H + (1 + two) * Hk) + B * T * 16.0, flops=0)
        mean = c["ctx"] * (0.625 if c["ragged"] else 1.0)        # of 0.25 .. 1 of the longest
        keys = B * (mean + T)
        return dict(bytes=keys * Hk * D * 4.0 + B * T * H * (D * 2.0 * (two + 1) + 4), flops=4.0 * D * H * T * keys)
    N, Hd, V = c["rows"], c["hidden"], c["vocab"]
    product = 2.0 * N * Hd * V
    if c["op"] == "score":
        return dict(bytes=(N + V) * Hd * 2.0 + N * 16.0, flops=product)
    return dict(bytes=2 * (N + V) * Hd * 2.0 + N * 8.0, flops=3 * product)


# ------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------------------------

def _exact_attend(s):
    c = s["case"]
    B, T, H, Hk = c["batch"], c["nodes"], c["heads"], c["kv_heads"]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, H, T), -math.inf, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist()
    for b in range(B):
        L = int(s["lens"][b])
        paths = []
        for i, p in enumerate(parents[b]):             # a node's path from the root, itself included
            paths.append([] if p == -2 else [i] if p == -1 else paths[p] + [i])
        real = [i for i in range(T) if paths[i]]
        sees = torch.ones(len(real), L + T, dtype=torch.bool, device=DEV)
        sees[:, L:] = torch.tensor([[j in paths[i] for j in range(T)] for i in real], device=DEV)
        kpos = torch.cat([torch.arange(L), L + torch.tensor([len(p) - 1 for p in paths])]).to(DEV)
        qpos = torch.tensor([L + len(paths[i]) - 1 for i in real], device=DEV)
        near = qpos[:, None] - kpos[None] <= c["w_0"]
        for h in range(H):
            k = s["k_cache"][b, :L + T, h // (H // Hk)].double()
            a = s["q_base"][b, real, h].double() @ k.T
            if s["kg_cache"] is not None:
                kg = s["kg_cache"][b, :L + T, h // (H // Hk)].double()
                a = torch.where(near, a, s["q_group"][b, real, h].double() @ kg.T)
            a = torch.where(sees, a / math.sqrt(D), -math.inf)
            lse[b, h, real] = torch.logsumexp(a, -1)
            out[b, real, h] = torch.softmax(a, -1) @ s["v_cache"][b, :L + T, h // (H // Hk)].double()
    return dict(out=out, lse=lse)


def _exact_append(s):
    c = s["case"]
    B, T, half = c["batch"], c["nodes"], D // 2
    parents, freq = s["parents"].tolist(), s["inv_freq"].double()
    out = {n: s[n].double() for n in ("k_cache", "v_cache")}
    out["q_base"] = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    if s["kg_cache"] is not None:
        out["kg_cache"], out["q_group"] = s["kg_cache"].double(), torch.zeros_like(out["q_base"])
    out["depth"], out["mask"] = None, None

    def turned(x, w, p):
        x = x.double()
        y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / D + 1e-6)
        y = (y.bfloat16().double() * w.double()).bfloat16().double()          # the norm's own two roundings
        z = torch.complex(y[..., :half], y[..., half:]) * torch.polar(torch.ones_like(freq), p * freq)
        return torch.cat([z.real, z.imag], -1)

    for b in range(B):
        deep = []
        for t in range(T):
            par = parents[b][t]
            deep.append(-1 if par == -2 else 0 if par == -1 else deep[par] + 1)
            if deep[t] < 0:
                continue
            row, p = int(s["lens"][b]) + t, int(s["lens"][b]) + deep[t]
            out["q_base"][b, t] = turned(s["q"][b, t], s["q_weight"], p)
            out["k_cache"][b, row] = turned(s["k"][b, t], s["k_weight"], p)
            out["v_cache"][b, row] = s["v"][b, t].double()
            if s["kg_cache"] is not None:
                out["q_group"][b, t] = turned(s["q"][b, t], s["q_weight"], p // c["group"])
                out["kg_cache"][b, row] = turned(s["k"][b, t], s["k_weight"], p // c["group"])
    return out


def _exact_head(s):
    c = s["case"]
    h, w = s["hidden"].detach().double(), s["weight"].detach()
    N, V = c["rows"], c["vocab"]
    lab = s["labels"].clone()
    used = lab != -100
    lse, nll = torch.empty(N, dtype=torch.float64, device=DEV), torch.empty(N, dtype=torch.float64, device=DEV)
    dh = torch.empty_like(h) if c["op"] == "loss" else None
    dw = torch.zeros(V, c["hidden"], dtype=torch.float64, device=DEV) if c["op"] == "loss" else None
    wd = w.double()
    n = int(used.sum())
    for lo in range(0, N, 1024):                       # rows are independent of one another
        hi = min(N, lo + 1024)
        z = torch.mm(h[lo:hi], wd.t())
        lse[lo:hi] = torch.logsumexp(z, 1)
        y = torch.where(used[lo:hi], lab[lo:hi], 0)
        nll[lo:hi] = (lse[lo:hi] - z[torch.arange(hi - lo, device=DEV), y]) * used[lo:hi]
        if c["op"] == "loss":
            gr = torch.softmax(z, 1)
            gr[torch.arange(hi - lo, device=DEV), y] -= 1.0
            gr = gr * used[lo:hi, None] / n
            dh[lo:hi] = torch.mm(gr, wd)
            dw.addmm_(gr.t(), h[lo:hi])
    if c["op"] == "loss":
        return dict(loss=nll.sum() / n, d_hidden=dh, d_weight=dw)
    return dict(nll=nll, lse=lse, **(dict(top=None) if c["top"] else {}))


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return dict(attend=_exact_attend, append=_exact_append, score=_exact_head, loss=_exact_head)[case["op"]](s)
