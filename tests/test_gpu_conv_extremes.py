"""The convolution where its preactivations are far from zero, and where inputs or the filter are not finite: packed sequences on every path (boxes
through tensor maps, one channel a thread, the backward's ring) and rectangles, against the formula in 64 bits.

Tolerances, u = 2^-24.  The filter passes the input on as it is (taps 0, 0, 0, 1), so the preactivation v is exact.  Of a sigmoid the exponent -v log2(e) is
off by a rounding of the product and one of the constant, 2 u |v log2(e)|, which is 2 u |v| of the exponential; that is as much of the sigmoid for v far below
zero, and at most 0.28 x 2 u for v above.  Exponential, sum and reciprocal are good to 2^-22, u and 2^-23, 7 u, two products more if a pair shares a
reciprocal, and the product with v one: (2 |v| + 10) u for negative v, 11 u for others.  The derivative has that
once for its sigmoid and once for 1 + v (1 - sigmoid), which is away from zero for the values taken; there a sigmoid near 1 that is off by 2 u or rounded to u makes
2 v u, but none above v = 17.4, where exp(-v) is less than u / 2, the sum is 1 and so is its reciprocal: so (2 t + 10) u with t = -v or min(v, 18).
Twice as much is allowed, and twice that for the derivative.  What is below 2^-125 may be zero (subnormal reciprocals): |v| 2^-125 more.  bfloat16: 2^-8
of the value for its rounding.  dw and db: 1e-5 of the sum of their terms' sizes."""
import math

import pytest
import torch

from tests.test_gpu_packed import DEV, cu_of

pytestmark = pytest.mark.gpu

VALUES = [-1e30, -1e20, -1e6, -1e4, -200.0, -104.0, -88.5, -87.0, -60.5, -43.0, -41.0, -30.0, -5.0, 0.0, 0.5, 3.0, 43.0, 1e4, 1e30]


def plain(x, w, b):
    """y of one sequence from its taps; zero times infinity is a NaN, as in the sum that the formula has."""
    line = torch.cat([torch.zeros(3, x.shape[1], dtype=x.dtype, device=x.device), x])
    pre = b + sum(line[k:k + x.shape[0]] * w[:, 0, k] for k in range(4))
    return pre * torch.sigmoid(pre)


def makes(T, W, dtype, values, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.tensor(values)[torch.randint(len(values), (T, W), generator=g)].to(dtype).to(DEV)
    w = torch.zeros(W, 1, 4, device=DEV)
    w[:, 0, 3] = 1
    return x, w, torch.zeros(W, device=DEV), torch.randn(T, W, generator=g).to(dtype).to(DEV)


def within(got, want, v, dtype, factor=1.0):
    got, want, v = got.detach().double(), want.detach().double(), v.detach().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    t = torch.where(v < 0, -v, v.clamp(max=18))
    bound = 2 * factor * (2 * t + 10) * 2.0 ** -24 * want.abs() + v.abs() * 2.0 ** -125 + 2.0 ** -125
    if dtype == torch.bfloat16:
        bound += 2.0 ** -8 * want.abs() * 1.001
    ok = torch.isnan(want) | (got == want) | ((got - want).abs() <= bound)
    bad = torch.nonzero(~ok)
    assert not len(bad), [(v[tuple(i)].item(), got[tuple(i)].item(), want[tuple(i)].item()) for i in bad[:4]]


# on the 16-byte grid, off it, and (the last two) more values than the backward takes with one channel a thread
SIZES = [(70, 128, torch.float32), (70, 128, torch.bfloat16), (70, 37, torch.float32), (70, 37, torch.bfloat16), (70, 130, torch.bfloat16),
         (5000, 1024, torch.float32), (8000, 1024, torch.bfloat16)]


@pytest.mark.parametrize("T,W,dtype", SIZES)
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("values", ["near and above", "near and below", "all"])
def test_far_preactivations(T, W, dtype, dense, values):
    import mamba_b200
    x, w, b, dy = makes(T, W, dtype, {"near and above": [v for v in VALUES if v >= -5], "near and below": [v for v in VALUES if v <= 3], "all": VALUES}[values], T + W)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    if dense:
        y = mamba_b200.causal_conv1d_silu(leaves[0][None], *leaves[1:])[0]
    else:
        y = mamba_b200.causal_conv1d_silu_packed(*leaves, cu_seqlens=cu_of([T]))
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    v, g = x.double(), dy.double()
    s = torch.sigmoid(v)
    within(y, v * s, v, dtype)
    slope = g * s * (1 + v * (1 - s))
    within(dx, slope, v, dtype, 2)
    line = torch.cat([torch.zeros(3, W, dtype=torch.float64, device=DEV), v])
    for k in range(4):
        terms = slope * line[k:k + T]
        assert ((dw[:, 0, k].double() - terms.sum(0)).abs() <= 1e-5 * terms.abs().sum(0) + 1e-30).all(), k
    assert ((db.double() - slope.sum(0)).abs() <= 1e-5 * slope.abs().sum(0) + 1e-30).all()


@pytest.mark.parametrize("T,W,dtype", SIZES)
@pytest.mark.parametrize("dense", [False, True])
def test_infinities_and_nan(T, W, dtype, dense):
    """A channel that is not finite is NaN where the formula says so, and its neighbours are as without it."""
    import mamba_b200
    x, w, b, dy = makes(T, W, dtype, [-5.0, 0.5, 3.0, -30.0], T)
    x[T // 2, ::5], x[T // 3, 1::5], x[T // 4, 2::5] = -math.inf, math.inf, math.nan
    b[4] = -math.inf
    leaf = x.clone().requires_grad_()
    run = (lambda u: mamba_b200.causal_conv1d_silu(u[None], w, b)[0]) if dense else (lambda u: mamba_b200.causal_conv1d_silu_packed(u, w, b, cu_seqlens=cu_of([T])))
    y = run(leaf)
    dx, = torch.autograd.grad(y, leaf, dy)
    exact = x.double().requires_grad_()
    want = plain(exact, w.double(), b.double())
    within(y, want, torch.nan_to_num(x, 0, 0, 0), dtype)
    # the derivative, from the formula: s (1 + v (1 - s)), and through the taps that are zero
    pre = b.double() + sum(torch.cat([torch.zeros(3, W, dtype=torch.float64, device=DEV), x.double()])[k:k + T] * w.double()[:, 0, k] for k in range(4))
    s = torch.sigmoid(pre)
    slope = torch.cat([dy.double() * s * (1 + pre * (1 - s)), torch.zeros(3, W, dtype=torch.float64, device=DEV)])
    within(dx, sum(slope[3 - k:3 - k + T] * w.double()[:, 0, k] for k in range(4)), torch.nan_to_num(x, 0, 0, 0), dtype, 2)


@pytest.mark.parametrize("T,W,dtype", SIZES)
def test_rows_behind_the_last_sequence(T, W, dtype):
    """Zeros, whatever the filter holds."""
    import mamba_b200
    x, w, b, dy = makes(T, W, dtype, [-5.0, 0.5, 3.0], T)
    w[:, 0, 0], w[::2, 0, 3], b[1::3] = math.inf, math.nan, -math.inf
    for lengths in ([T // 2], [T - 1], [7, 2, T - 12], []):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        y = mamba_b200.causal_conv1d_silu_packed(*leaves, cu_seqlens=cu_of(lengths))
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        assert (y[sum(lengths):] == 0).all() and (dx[sum(lengths):] == 0).all(), lengths
    assert (dw == 0).all() and (db == 0).all()              # (of no sequence at all)
