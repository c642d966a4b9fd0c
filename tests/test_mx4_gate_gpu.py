"""Gate and up far from 1 on the GPU: silu(x gate) * (x up) where one factor is out of the
range that the result is in."""
import itertools

import pytest
import torch

import mx4_util as U
import spindle_b200 as sg

pytestmark = pytest.mark.gpu

# what 4 bits hold as it is: one value a row of the matrix, one of x, so that both sums are exact
GATES = [s * g for g in (0.0, 2.0 ** -30, 0.5, 2.0, 6.0, 16.0, 24.0, 64.0, 96.0, 2.0 ** 70) for s in (1, -1)]
UPS = [s * u for u in (2.0 ** -100, 1.0, 1.5 * 2.0 ** 60, 2.0 ** 120, 1.5 * 2.0 ** 126) for s in (1, -1)]


# one row: columns over a cluster, and not; several rows of the kernel for few; the kernel for many
@pytest.mark.parametrize("rows,cols,feats", [(1, 4096, 200), (3, 256, 200), (40, 320, 200), (2600, 288, 1025)])
def test_far_gates(dev, rows, cols, feats):
    pairs = list(itertools.product(GATES, UPS))
    g, u = (torch.tensor([pairs[i % len(pairs)][j] for i in range(feats)], device=dev) for j in (0, 1))
    w, v, x = torch.zeros(feats, cols, device=dev), torch.zeros(feats, cols, device=dev), torch.zeros(rows, cols, device=dev)
    w[:, 37], v[:, 37] = g, u
    x[:, 37] = torch.tensor([1.0, -1.0, 0.5], device=dev)[torch.arange(rows, device=dev) % 3]
    a, b = (x[:, 37:38].double() * t.double() for t in (g, u))
    want = a * torch.sigmoid(a) * b
    # ex2 is off by 2^-22 of it, the reciprocal by 2^-23, three sums and products of the exponential's and three of the result by a
    # half step each: 4 + 2 + 6 of 2^-24; the exponent's constant by 1.34e-8 for each of |a|.  Under -87.3 the result is 0.
    bound = want.abs() * (12 * 2.0 ** -24 + 1.34e-8 * a.abs().clamp(max=200) * (a < 0))
    bound = torch.where(a < -87, want.abs(), bound)
    W, V = sg.mx4_quantize(w), sg.mx4_quantize(v)
    for dtype in (torch.float32, torch.bfloat16):
        got = sg.mx4_matmul(x, W, up=V, dtype=dtype)
        over = want.abs() > 3.5e38
        assert torch.equal(got[over].double(), want[over].sign() * float("inf"))
        assert U.close(got[~over], want[~over], bound[~over])
    sg.device_status()


def test_far_gates_of_experts(dev):
    e, n, dim, ff = 3, 50, 64, 200
    pairs = list(itertools.product(GATES, UPS))
    w, v = torch.zeros(e, ff, dim, device=dev), torch.zeros(e, ff, dim, device=dev)
    w[:, :, 5], v[:, :, 5] = (torch.tensor([pairs[i % len(pairs)][j] for i in range(ff)], device=dev) for j in (0, 1))
    x = torch.zeros(n, dim, device=dev)
    x[:, 5] = 1.0
    p = sg.moe_route(torch.zeros(n, e, device=dev), sg.MoePlan(n, 2, e, device=dev))
    got = sg.mx4_experts(x, sg.mx4_quantize(w), p, up=sg.mx4_quantize(v)).double()
    a, b = w[0, :, 5].double(), v[0, :, 5].double()
    want = a * torch.sigmoid(a) * b
    assert not got.isnan().any()
    small = (want.abs() < 3.4e38) & (a > -87)
    assert ((got - want)[:, small].abs() <= want[small].abs() * (13 * 2.0 ** -24 + 1.34e-8 * 96) + 2.0 ** -149).all()
