"""Vocabulary-head operators on the GPU against a plain 64-bit implementation."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = torch.finfo(torch.bfloat16).eps / 2          # a bf16 rounding is off by at most this much of the value
F32 = torch.finfo(torch.float32).eps / 2

# rows, hidden, vocab
SIZES = [(1, 8, 1), (1, 64, 7), (3, 72, 130), (64, 128, 128), (65, 136, 257), (127, 512, 1000), (128, 64, 4096), (129, 264, 8193), (300, 1024, 777),
         (513, 192, 20011), (2, 2048, 50257)]


def make(N, H, V, seed=0, ignored=0.25, scale=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed + N + H + V)
    h = torch.randn(N, H, generator=g, device="cuda").bfloat16()
    w = (scale * torch.randn(V, H, generator=g, device="cuda")).bfloat16()
    y = torch.randint(0, V, (N,), generator=g, device="cuda")
    if ignored and N > 1:
        y[torch.rand(N, generator=g, device="cuda") < ignored] = -100
        y[0] = V - 1
    return h, w, y


def exact(h, w, y, coef=None):
    """lse, nll, z error bound; with per-row coefficients also the gradients and their bounds."""
    z = h.double() @ w.double().T
    lse = torch.logsumexp(z, 1)
    used = y >= 0
    nll = torch.where(used, lse - z.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    # an fp32 sum of K products is off by at most K half-steps of the products' absolute sum
    dz = h.shape[1] * F32 * (h.double().abs() @ w.double().abs().T).amax(1) + 1e-6
    if coef is None:
        return lse, nll, dz, z
    p = torch.softmax(z, 1)
    gr = p.clone()
    gr[torch.arange(len(y), device="cuda"), y.clamp(min=0)] -= 1
    c = torch.where(used, coef.double(), 0.0)[:, None]
    gr, p = gr * c, p * c.abs()
    # d logits: rounded to bf16 once, p itself off by the errors of z and lse and of the exponential (2^-20)
    err = HALF * gr.abs() + p * (4 * dz[:, None] + 2.0 ** -20)
    dh, dw = gr @ w.double(), gr.T @ h.double()
    acc = lambda k: k * F32                                       # noqa: E731
    b_h = err @ w.double().abs() + acc(w.shape[0]) * (gr.abs() @ w.double().abs()) + HALF * dh.abs() * (1 + HALF) + 1e-30
    b_w = err.T @ h.double().abs() + acc(len(y)) * (gr.abs().T @ h.double().abs()) + HALF * dw.abs() * (1 + HALF) + 1e-30
    b_h, b_w = b_h * (1 + HALF), b_w * (1 + HALF)
    return lse, nll, dz, z, dh, dw, b_h, b_w


@pytest.mark.parametrize("N, H, V", SIZES)
def test_token_scores(N, H, V):
    from jetlm.kernels import head_ops
    h, w, y = make(N, H, V)
    got = head_ops.token_scores(h, w, y, top=True)
    lse, nll, dz, z = exact(h, w, y)
    tol = 2 * dz + 2.0 ** -20 * (1 + lse.abs())                   # z and the sum of exponentials
    assert ((got.lse.double() - lse).abs() <= tol).all() and ((got.nll.double() - nll).abs() <= 2 * tol).all()
    assert (got.nll[y < 0] == 0).all()
    best = z.amax(1)
    assert (z.gather(1, got.top[:, None])[:, 0] >= best - 2 * dz).all()
    clear = z.topk(2, 1).values.diff(dim=1).abs()[:, 0] > 2 * dz if V > 1 else torch.ones(N, dtype=torch.bool, device="cuda")
    assert torch.equal(got.top[clear], z.argmax(1)[clear])
    assert got.nll.dtype == got.lse.dtype == torch.float32 and got.top.dtype == torch.int64
    only = head_ops.token_scores(h, w)
    assert only.nll is None and only.top is None and torch.equal(only.lse, got.lse)


@pytest.mark.parametrize("N, H, V", [(1, 520, 18945), (15, 72, 20000), (16, 2056, 9001), (17, 1032, 19000), (31, 64, 5), (32, 4096, 30011), (33, 256, 30011)])
def test_token_scores_of_few_rows(N, H, V):
    """Up to 32 rows the weight's rows are the rows of the product: one and several tiles a CTA, a last tile that is short or empty."""
    test_token_scores(N, H, V)


@pytest.mark.parametrize("N", [3, 32])
def test_few_rows_in_masked_and_strided_places(N):
    from jetlm.kernels import head_ops
    h, w, y = make(N, 264, 5003, ignored=0)
    big = torch.full((2 * N, 272), math.nan, device="cuda").bfloat16()       # rows and columns that do not belong to the operand
    big[::2, :264] = h
    wide = torch.full((5003, 280), math.inf, device="cuda").bfloat16()
    wide[:, :264] = w
    want = head_ops.token_scores(h, w, y, top=True)
    got = head_ops.token_scores(big[::2, :264], wide[:, :264], y, top=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h[1, 3] = math.nan
    got = head_ops.token_scores(h, w, y, top=True)
    keep = [i for i in range(N) if i != 1]
    assert torch.equal(got.lse[keep], want.lse[keep]) and torch.equal(got.top[keep], want.top[keep]) and torch.isnan(got.lse[1])


def test_equal_logits_give_the_lowest_index():
    from jetlm.kernels import head_ops
    h = torch.ones(5, 64, device="cuda").bfloat16()
    w = torch.zeros(3000, 64, device="cuda").bfloat16()
    assert (head_ops.token_scores(h, w, top=True).top == 0).all()
    w[[700, 701, 1400, 2999]] = 1
    got = head_ops.token_scores(h, w, top=True)
    assert (got.top == 700).all()
    assert torch.allclose(got.lse, torch.tensor(64 + math.log(4 + 2996 * math.exp(-64.0)), device="cuda").expand(5), atol=1e-5)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("N, H, V", SIZES)
def test_loss_and_gradients(N, H, V, reduction):
    from jetlm.kernels import head_ops
    h, w, y = make(N, H, V)
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = head_ops.linear_cross_entropy(h, w, y, reduction=reduction)
    up = torch.randn(loss.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    dh, dw = torch.autograd.grad(loss, [h, w], up)
    n = int((y >= 0).sum())
    coef = up if reduction == "none" else (up / n if reduction == "mean" else up).expand(N)
    lse, nll, dz, z, wdh, wdw, b_h, b_w = exact(h.detach(), w.detach(), y, coef)
    want = nll if reduction == "none" else nll.sum() / (n if reduction == "mean" else 1)
    tol = 4 * dz + 2.0 ** -19 * (1 + lse.abs())
    tol = tol if reduction == "none" else (tol * (y >= 0)).sum() / (n if reduction == "mean" else 1) + (N + 4) * F32 * want.abs()
    assert loss.dtype == torch.float32 and ((loss.double() - want).abs() <= tol).all()
    assert dh.dtype == dw.dtype == torch.bfloat16
    assert ((dh.double() - wdh).abs() <= b_h).all(), ((dh.double() - wdh).abs() / b_h).max()
    assert ((dw.double() - wdw).abs() <= b_w).all(), ((dw.double() - wdw).abs() / b_w).max()
    assert (dh[y < 0] == 0).all()


@pytest.mark.parametrize("counted", [0, 1, 63, 64, 65, 255, 256, 257, 511, 512, 513, 700])
@pytest.mark.parametrize("ignore", [-100, 7])
def test_rows_that_do_not_count_are_left_out(counted, ignore):
    """700 rows, of which `counted` at random places count; the others hold NaN.  They have no loss and no gradient."""
    from jetlm.kernels import head_ops
    N, H, V = 700, 136, 3001
    h, w, y = make(N, H, V, ignored=0)
    y = torch.where(y == ignore, ignore + 1, y)
    perm = torch.randperm(N, generator=torch.Generator().manual_seed(counted)).cuda()
    used, rest = perm[:counted].sort().values, perm[counted:]
    y[rest] = ignore
    dirty = h.clone()
    dirty[rest] = math.nan
    dirty.requires_grad_(True)
    w.requires_grad_(True)
    nll = head_ops.linear_cross_entropy(dirty, w, y, ignore_index=ignore, reduction="none")
    loss = head_ops.linear_cross_entropy(dirty, w, y, ignore_index=ignore, reduction="sum")
    up = torch.randn(N, generator=torch.Generator().manual_seed(5)).cuda()
    dh, dw = torch.autograd.grad(nll, [dirty, w], up)
    _, _, dz, _, wdh, wdw, b_h, b_w = exact(h[used], w.detach(), y[used] if ignore < 0 else y[used].clone(), up[used])
    lse, want, dz, _ = exact(h[used], w.detach(), y[used])
    tol = 4 * dz + 2.0 ** -19 * (1 + lse.abs())
    assert (nll[rest] == 0).all() and (dh[rest] == 0).all()
    assert ((nll[used].double() - want).abs() <= tol).all()
    assert abs(float(loss.detach()) - float(want.sum())) <= float(tol.sum()) + (N + 4) * F32 * float(want.abs().sum())
    assert ((dh[used].double() - wdh).abs() <= b_h).all() and ((dw.double() - wdw).abs() <= b_w).all()
    mean = head_ops.linear_cross_entropy(dirty, w, y, ignore_index=ignore)
    assert torch.isnan(mean) if counted == 0 else abs(float(mean.detach()) * counted - float(loss.detach())) <= 4 * F32 * abs(float(loss.detach())) + 1e-30


def test_gradient_agrees_with_differences():
    """d loss / d direction from the gradients against the loss itself moved by bf16-exact steps."""
    from jetlm.kernels import head_ops
    g = torch.Generator(device="cuda").manual_seed(4)
    pick = lambda *s: torch.randint(-8, 9, s, generator=g, device="cuda").float() / 8       # noqa: E731
    h, w, y = pick(40, 64), pick(333, 64) / 4, torch.randint(0, 333, (40,), generator=g, device="cuda")
    eh, ew = pick(40, 64) / 64, pick(333, 64) / 256      # steps that keep every value within bf16's 8 bits
    f = lambda s: head_ops.linear_cross_entropy((h + s * eh).bfloat16(), (w + s * ew).bfloat16(), y, reduction="sum").double()   # noqa: E731
    slope = (f(1) - f(-1)) / 2
    hb, wb = h.bfloat16().requires_grad_(True), w.bfloat16().requires_grad_(True)
    dh, dw = torch.autograd.grad(head_ops.linear_cross_entropy(hb, wb, y, reduction="sum"), [hb, wb])
    real = lambda s: ((h + s * eh).bfloat16().double(), (w + s * ew).bfloat16().double())                                        # noqa: E731
    (h1, w1), (h0, w0) = real(1), real(-1)
    dot = ((h1 - h0) / 2 * dh.double()).sum() + ((w1 - w0) / 2 * dw.double()).sum()
    # third-order term of the central difference, evaluated on the exact loss, plus half a step of every gradient element used
    ce = lambda s: torch.nn.functional.cross_entropy(real(s)[0] @ real(s)[1].T, y, reduction="sum")                               # noqa: E731
    h64, w64 = h.bfloat16().double().requires_grad_(True), w.bfloat16().double().requires_grad_(True)
    g_h, g_w = torch.autograd.grad(torch.nn.functional.cross_entropy(h64 @ w64.T, y, reduction="sum"), [h64, w64])
    curved = abs(float((ce(1) - ce(-1)) / 2 - (((h1 - h0) / 2 * g_h).sum() + ((w1 - w0) / 2 * g_w).sum())))
    rounding = 2 * HALF * float(((h1 - h0).abs() / 2 * dh.double().abs()).sum() + ((w1 - w0).abs() / 2 * dw.double().abs()).sum())
    assert abs(float(slope - dot)) <= curved + rounding + 1e-3


def test_only_one_gradient_and_leading_dimensions():
    from jetlm.kernels import head_ops
    h, w, y = make(60, 128, 900)
    h3 = h.view(3, 20, 128)
    full = torch.autograd.grad(head_ops.linear_cross_entropy(h.requires_grad_(True), w.requires_grad_(True), y), [h, w])
    hb = h3.detach().requires_grad_(True)
    dh, = torch.autograd.grad(head_ops.linear_cross_entropy(hb, w.detach(), y.view(3, 20)), [hb])
    assert dh.shape == hb.shape and torch.equal(dh.view(60, 128), full[0])
    dw, = torch.autograd.grad(head_ops.linear_cross_entropy(h3.detach(), w, y.view(3, 20)), [w])
    assert torch.equal(dw, full[1])
    # every second row of a wider buffer, and a slice whose leading dimensions do not collapse
    wide = torch.zeros(60, 256, device="cuda", dtype=torch.bfloat16)
    wide[:, :128] = h.detach()
    a = head_ops.token_scores(wide[:, :128], w.detach(), y)
    assert torch.equal(a.nll, head_ops.token_scores(h.detach(), w.detach(), y).nll)
    b = head_ops.token_scores(h3.detach()[:, :-1], w.detach(), y.view(3, 20)[:, :-1])
    assert b.nll.shape == (3, 19) and torch.equal(b.nll, a.nll.view(3, 20)[:, :-1])
    with pytest.raises(ValueError, match="contiguous"):
        head_ops.token_scores(wide[:, 1:129], w.detach(), y)
    with pytest.raises(ValueError, match="contiguous"):
        head_ops.token_scores(h.detach(), torch.zeros(900, 132, device="cuda", dtype=torch.bfloat16)[:, :128], y)
    with pytest.raises(ValueError, match="labels"):
        head_ops.token_scores(h.detach(), w.detach(), y.int())


def test_nothing_counted_no_rows_and_labels_out_of_range():
    from jetlm.kernels import head_ops
    h, w, y = make(9, 64, 100, ignored=0)
    none = torch.full_like(y, -100)
    hb, wb = h.requires_grad_(True), w.requires_grad_(True)
    loss = head_ops.linear_cross_entropy(hb, wb, none)
    assert math.isnan(float(loss))
    dh, dw = torch.autograd.grad(loss, [hb, wb])
    assert (dh == 0).all() and (dw == 0).all()
    assert float(head_ops.linear_cross_entropy(hb, wb, none, reduction="sum")) == 0
    e = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ey = torch.empty(0, device="cuda", dtype=torch.int64)
    s = head_ops.token_scores(e, w.detach(), ey, top=True)
    assert s.nll.shape == s.lse.shape == s.top.shape == (0,)
    loss = head_ops.linear_cross_entropy(e, wb, ey, reduction="sum")
    assert float(loss) == 0
    de, dw = torch.autograd.grad(loss, [e, wb])
    assert de.shape == (0, 64) and (dw == 0).all()
    for bad in (100, -1, 1 << 40, -(1 << 62)):
        z = y.clone()
        z[3] = bad
        s = head_ops.token_scores(h.detach(), w.detach(), z)
        assert math.isnan(float(s.nll[3])) and torch.isfinite(s.nll[[0, 1, 2, 4, 5, 6, 7, 8]]).all()
        loss = head_ops.linear_cross_entropy(hb, wb, z)
        assert math.isnan(float(loss))
        assert torch.isnan(torch.autograd.grad(loss, hb)[0][3]).all()
    z = y.clone()
    z[3] = 7
    other = y.clone()
    other[3] = 55
    assert torch.equal(head_ops.linear_cross_entropy(h.detach(), w.detach(), z, ignore_index=7, reduction="none")[[0, 3]] == 0,
                       torch.tensor([False, True], device="cuda"))


def test_infinite_and_nan_logits_stay_in_their_rows():
    from jetlm.kernels import head_ops
    h, w, y = make(6, 64, 300, ignored=0)
    good = head_ops.token_scores(h, w, y)
    h = h.clone()
    h[2, 5] = math.nan
    h[4, 0] = math.inf
    got = head_ops.token_scores(h, w, y)
    keep = [0, 1, 3, 5]
    assert torch.equal(got.nll[keep], good.nll[keep]) and torch.equal(got.lse[keep], good.lse[keep])
    assert not torch.isfinite(got.lse[[2, 4]]).any()


def test_large_logits_do_not_overflow():
    from jetlm.kernels import head_ops
    h, w, y = make(70, 256, 1500, scale=20.0, ignored=0)
    lse, nll, dz, _ = exact(h, w, y)
    got = head_ops.token_scores(h, w, y)
    assert lse.abs().max() > 500
    assert ((got.lse.double() - lse).abs() <= 2 * dz + 2.0 ** -20 * (1 + lse.abs())).all()
    assert ((got.nll.double() - nll).abs() <= 4 * dz + 2.0 ** -19 * (1 + lse.abs())).all()


def test_repeats_streams_and_graphs():
    from jetlm.kernels import head_ops
    h, w, y = make(200, 256, 9001)
    h.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        loss = head_ops.linear_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, [h, w]))

    ref = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graphs, outs = [], []
    for _ in range(2):                                            # two captured steps share no scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    h2, w2, y2 = make(200, 256, 9001, seed=77)
    with torch.no_grad():
        h.copy_(h2)
        w.copy_(w2)
        y.copy_(y2)
    want = step()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    assert not torch.equal(want[1], ref[1])


def test_labels_straight_from_the_scores():
    """The labels of one call are what the kernels of the call before it wrote, with nothing in between."""
    from jetlm.kernels import head_ops
    h, w, _ = make(700, 128, 20000)
    want = head_ops.token_scores(h, w, top=True).top.clone()
    ref = head_ops.linear_cross_entropy(h, w, want)
    none = torch.full_like(want, -100)
    for _ in range(20):
        assert float(head_ops.linear_cross_entropy(h, w, none, reduction="sum")) == 0
        assert torch.equal(head_ops.linear_cross_entropy(h, w, head_ops.token_scores(h, w, top=True).top), ref)


def test_more_rows_than_one_launch_of_the_scores_takes():
    """Rows are scored 16384 at a time; the last group here is one row, which alone would take the path of few rows."""
    from jetlm.kernels import head_ops
    h, w, y = make(2 * 16384 + 1, 64, 300)
    lse, nll, dz, z = exact(h, w, y)
    got = head_ops.token_scores(h, w, y, top=True)
    tol = 2 * dz + 2.0 ** -20 * (1 + lse.abs())
    assert ((got.lse.double() - lse).abs() <= tol).all() and ((got.nll.double() - nll).abs() <= 2 * tol).all()
    assert (z.gather(1, got.top[:, None])[:, 0] >= z.amax(1) - 2 * dz).all()
    n = int((y >= 0).sum())
    loss = head_ops.linear_cross_entropy(h, w, y)
    # 1024 threads add 33 values each, then 10 additions join them; one division
    assert abs(float(loss) - float(nll.sum()) / n) <= float((2 * tol + 44 * F32 * nll.abs()).sum()) / n + 2 * F32 * float(nll.abs().sum()) / n


@pytest.mark.parametrize("N, H, V", [(17000, 64, 9001), (120, 8, 1200001), (300, 136, 460000)])
def test_gradients_over_several_pieces_of_the_vocabulary(N, H, V):
    """More than 256 MB of d logits: the row gradients are added up over two pieces, of which the second is the shorter."""
    from jetlm.kernels import head_ops
    h, w, y = make(N, H, V)
    h.requires_grad_(True)
    w.requires_grad_(True)
    dh, dw = torch.autograd.grad(head_ops.linear_cross_entropy(h, w, y, reduction="sum"), [h, w])
    hd, wd = h.detach(), w.detach()
    step = max(1, (1 << 24) // V)                                 # the oracle takes the rows in chunks: its matrices are (rows, V) in 64 bits
    e_w, b_w = torch.zeros(V, H, dtype=torch.float64, device="cuda"), torch.zeros(V, H, dtype=torch.float64, device="cuda")
    for lo in range(0, N, step):
        sl = slice(lo, lo + step)
        *_, eh, ew, bh, bw = exact(hd[sl], wd, y[sl], torch.ones(y[sl].shape, device="cuda"))
        assert ((dh[sl].double() - eh).abs() <= bh).all(), lo
        e_w += ew
        b_w += bw
    # A chunk's bound counts fp32 additions of its own rows only; over all N rows they may take N * F32 * sum |dz| |h|, and a
    # chunk's bound holds HALF * sum |dz| |h| for the rounding of dz: a factor N * F32 / HALF of what is there.
    assert ((dw.double() - e_w).abs() <= b_w * (1 + N * F32 / HALF)).all()


def test_the_number_of_counted_rows_may_change_between_replays():
    """A captured step takes the rows that count from the labels it meets, none or all of them too."""
    from jetlm.kernels import head_ops
    h, w, y = make(600, 136, 3001, ignored=0)
    h.requires_grad_(True)
    w.requires_grad_(True)

    def step():
        loss = head_ops.linear_cross_entropy(h, w, y, reduction="sum")
        return (loss.detach(), *torch.autograd.grad(loss, [h, w]))

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    full = y.clone()
    for keep in (600, 0, 1, 257, 599, 300):
        y.copy_(full)
        y[torch.randperm(600, generator=torch.Generator().manual_seed(keep)).cuda()[keep:]] = -100
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), keep


def test_one_gradient_of_many_rows_and_calls_without_any():
    from jetlm.kernels import head_ops
    h, w, y = make(900, 136, 5003)
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = head_ops.linear_cross_entropy(h, w, y)
    dh, dw = torch.autograd.grad(loss, [h, w])
    assert torch.equal(torch.autograd.grad(head_ops.linear_cross_entropy(h, w.detach(), y), h)[0], dh)
    assert torch.equal(torch.autograd.grad(head_ops.linear_cross_entropy(h.detach(), w, y), w)[0], dw)
    with torch.no_grad():
        quiet = head_ops.linear_cross_entropy(h, w, y)
    assert torch.equal(quiet, loss.detach()) and not quiet.requires_grad
    with torch.inference_mode():
        assert torch.equal(head_ops.linear_cross_entropy(h, w, y), loss.detach())
    kept = [t.clone() for t in (h.detach(), w.detach(), y)]
    assert all(torch.equal(a, b) for a, b in zip(kept, (h.detach(), w.detach(), y)))
