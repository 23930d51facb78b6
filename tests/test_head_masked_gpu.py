"""Rows that do not count, whatever they hold, at every number of rows."""
import math

import pytest
import torch

from test_head_ops_gpu import exact, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("N, H, V", [(2, 64, 300), (9, 72, 1000), (64, 136, 3001), (65, 128, 777), (128, 264, 8193), (129, 64, 5000), (200, 136, 3001),
                                     (256, 512, 1000), (120, 8, 1200001), (300, 136, 3001)])
def test_ignored_rows_take_no_part(N, H, V, bad):
    from jetlm.kernels import head_ops
    h, w, y = make(N, H, V, ignored=0)
    y[::2] = -100
    dirty = h.clone()
    dirty[::2] = bad
    wide = torch.full((N, H + 16), 3.0, device="cuda").bfloat16()            # rows further apart than they are long
    wide[:, :H] = dirty
    used = y >= 0
    up = torch.linspace(-1, 1, N, device="cuda")
    for rows in (dirty, wide[:, :H]):
        a, b = rows.detach().requires_grad_(True), w.clone().requires_grad_(True)
        nll = head_ops.linear_cross_entropy(a, b, y, reduction="none")
        dh, dw = torch.autograd.grad(nll, [a, b], up)
        assert (nll[~used] == 0).all() and (dh[~used] == 0).all()
        step = max(1, (1 << 24) // V)
        e_w = torch.zeros(V, H, dtype=torch.float64, device="cuda")
        b_w = torch.zeros_like(e_w)
        hu, yu, gu = h[used], y[used], up[used]
        for lo in range(0, len(yu), step):
            sl = slice(lo, lo + step)
            *_, eh, ew, bh, bw = exact(hu[sl], w, yu[sl], gu[sl])
            assert ((dh[used][sl].double() - eh).abs() <= bh).all()
            e_w += ew
            b_w += bw
        assert ((dw.double() - e_w).abs() <= b_w * (1 + 2.0 ** -10)).all()     # (each chunk's bound counts its own rows' additions in 32 bits)
    # the same from a clean copy of the rows, bit for bit
    clean = torch.where(used[:, None], h, torch.zeros_like(h)).requires_grad_(True)
    c = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(head_ops.linear_cross_entropy(clean, c, y, reduction="none"), c, up)[0], dw)
