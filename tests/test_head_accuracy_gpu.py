"""Vocabulary-head operators on rows whose label is predicted with confidence: the digits that the sums over K in parts, the
loss of a sure row and its gradient p - 1 have to keep."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = torch.finfo(torch.bfloat16).eps / 2          # a bf16 rounding is off by at most this much of the value
V = 20011


def sure_rows(N, H, lo, hi, seed=0, weight=0.02):
    """Rows, a head of usual scale and distinct labels with 1 - p(label) spread over [lo, hi] on a logarithmic scale: hidden states
    are noise plus as much of the label's weight row as that takes (found by bisection; rounding h moves 1 - p by some percent)."""
    g = torch.Generator(device="cuda").manual_seed(seed + N + H)
    w = (weight * torch.randn(V, H, generator=g, device="cuda")).bfloat16()
    y = torch.randperm(V, generator=g, device="cuda")[:N]
    noise = torch.randn(N, H, generator=g, device="cuda").double()
    want = torch.logspace(0, 1, N, device="cuda", dtype=torch.float64).log10() * (torch.tensor(hi / lo).log10()) if N > 1 else torch.zeros(1, device="cuda").double()
    want = lo * 10.0 ** want
    wy = w[y].double()
    zn, zw = noise @ w.double().T, wy @ w.double().T
    zn -= zn.gather(1, y[:, None])
    zw -= zw.gather(1, y[:, None])
    a, b = torch.zeros(N, 1, device="cuda").double(), torch.full((N, 1), 4 * 25 / (H * weight ** 2), device="cuda").double()
    for _ in range(40):
        c = (a + b) / 2
        q = ((zn + c * zw).exp().sum(1, keepdim=True) - 1).clamp(min=0)
        more = q / (1 + q) > want[:, None]
        a, b = torch.where(more, c, a), torch.where(more, b, c)
    return (noise + c * wy).bfloat16(), w, y


def exact(h, w, y):
    """In 64 bits, without cancelling: z of the labels, lse, the rest q = sum over the others of e^(z - z_y), and d nll / d z."""
    z = h.double() @ w.double().T
    zy = z.gather(1, y[:, None])
    e = (z - zy).exp().scatter(1, y[:, None], 0.0)
    q = e.sum(1, keepdim=True)
    dz = (e / (1 + q)).scatter(1, y[:, None], -q / (1 + q))
    return zy[:, 0], (zy + q.log1p())[:, 0], q[:, 0], dz


def part_of(N):
    """Products that one accumulator takes before it is added in an fp32 register."""
    return 64 if N <= 16 else 128 if N <= 32 else 256 if N <= 128 else 512


@pytest.mark.parametrize("H", [2048, 4096])
@pytest.mark.parametrize("N", [1, 16, 17, 49, 128, 300])
def test_scores_of_sure_rows_keep_their_digits(N, H):
    from jetlm.kernels import head_ops
    h, w, y = sure_rows(N, H, 1e-6, 1e-2)
    got = head_ops.token_scores(h, w, y, top=True)
    zy, lse, q, _ = exact(h, w, y)
    assert torch.equal(got.top, y)
    # lse is the label's logit and little more.  An accumulator cuts every sum of 16 products off, by at most an ulp (2^-23) of what
    # it holds then; the parts are added with half an ulp each.  The steps' sums are taken from the data.
    P = part_of(N)
    prod = (h.double() * w[y].double()).view(N, H // P, P // 16, 16).sum(-1)
    inside, total = prod.cumsum(-1).abs().sum((1, 2)), prod.sum(-1).cumsum(-1).abs().sum(-1)
    bound = 2.0 ** -23 * inside + 2.0 ** -24 * (total + lse.abs()) + 2.0 ** -22
    err = got.lse.double() - lse
    assert (err.abs() <= bound).all(), (err / bound, err)
    # nll = log(1 + q): q is off by the errors of two logits' difference (less than 1e-4 at these sizes), the exponential (2^-22)
    # and a sum in 32 bits, all relative to q itself
    want = q.log1p()
    rel = (got.nll.double() - want).abs() / want
    assert (rel <= 2.0 ** -11).all(), (rel.max(), want[rel.argmax()])
    plain = head_ops.linear_cross_entropy(h, w, y, reduction="none")
    assert ((plain.double() - want).abs() <= 2.0 ** -11 * want).all()


@pytest.mark.parametrize("lo, hi", [(1e-6, 1e-2), (0.05, 0.95)])
@pytest.mark.parametrize("reduction", ["sum", "none", "mean"])
@pytest.mark.parametrize("N, H", [(1, 4096), (17, 2048), (49, 4096), (128, 2048), (200, 4096), (300, 2048), (300, 4096)])
def test_gradient_of_sure_rows(N, H, reduction, lo, hi):
    """1 - p from 1e-2 down to 1e-6, and of usual rows: every row's gradient is right relative to the row itself, not to gradients of
    size one."""
    from jetlm.kernels import head_ops
    h, w, y = sure_rows(N, H, lo, hi, seed=5)
    if N > 256:                                       # rows that do not count in between: the others are packed
        y[3::7] = -100
    used = y >= 0
    hu, yu = h[used], y[used]
    _, _, q, dz = exact(hu, w, yu)
    n = len(yu)
    up = torch.linspace(0.5, 2.0, N, device="cuda") if reduction == "none" else torch.tensor(1.5, device="cuda")
    c = (up[used] if reduction == "none" else (up / n if reduction == "mean" else up).expand(n)).double()[:, None]
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dh, dw = torch.autograd.grad(head_ops.linear_cross_entropy(hg, wg, y, reduction=reduction), [hg, wg], up)
    dz = dz * c
    want_h, want_w = dz @ w.double(), dz.T @ hu.double()
    # d logits are rounded once (HALF of each), probabilities are off by less than 2^-11 (z cut off 256 times at 2^-23 of up to 8, lse,
    # exponential) and fp32 sums over V / 16 steps lose less than 2^-12; the result is rounded once
    each = HALF + 2.0 ** -10
    bound = each * (dz.abs() @ w.double().norm(dim=1)) + HALF * (1 + HALF) * want_h.norm(dim=1)
    err = (dh[used].double() - want_h).norm(dim=1)
    assert (err <= bound).all(), ((err / bound).max(), (q / (1 + q))[(err / bound).argmax()])
    assert (dh[~used] == 0).all()
    bound_w = each * (dz.abs().T @ hu.double().abs()) + HALF * (1 + HALF) * want_w.abs() + 1e-30
    assert ((dw.double() - want_w).abs() <= bound_w).all()


def test_losses_may_be_overwritten_before_the_backward_pass():
    from jetlm.kernels import head_ops
    h, w, y = sure_rows(40, 256, 1e-3, 1e-1)
    h.requires_grad_(True)
    m = torch.linspace(0, 1, 40, device="cuda")
    want, = torch.autograd.grad((head_ops.linear_cross_entropy(h, w, y, reduction="none") * m).sum(), h)
    loss = head_ops.linear_cross_entropy(h, w, y, reduction="none")
    loss *= m
    assert torch.equal(torch.autograd.grad(loss.sum(), h)[0], want)
