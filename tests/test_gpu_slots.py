"""Single tokens on pools of slots, beam selection and reordering, against plain implementations in 64 bits.

The step: exponential, its argument, the softplus and two products, 32 u = 2e-6 of the tensor's largest value counted (u = 2^-24), 1e-5 allowed
as for the scan.  Selection: scores are one rounding of a value in 64 bits plus the error of the sum of exponentials (each within 4 u, added in pairs
of at most 32): 2^-24 of the value and 1e-6 allowed; tokens and parents are equal.  Reordering copies."""
import math

import pytest
import torch
import torch.nn.functional as F

from tests.test_gpu_packed import close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("B,W,N,dtype", [(1, 8, 16, torch.float32), (5, 72, 16, torch.bfloat16), (9, 33, 16, torch.float32),
                                         (33, 64, 8, torch.bfloat16), (4, 20, 32, torch.float32), (3, 12, 64, torch.float32)])
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("params", [torch.float32, torch.bfloat16])
def test_steps_on_slots(B, W, N, dtype, full, params):
    import mamba_b200
    g = torch.Generator().manual_seed(B + W + N)
    r = lambda *s: torch.randn(*s, generator=g)
    x, delta, z, Bm, Cm = (v.to(dtype).to(DEV) for v in (r(B, W), r(B, W), r(B, W), r(B, N), r(B, N)))
    A, D, bias = (v.to(params).to(DEV) for v in (-torch.exp(r(W, N) * 0.5), r(W), r(W) - 3))
    S = B + 3
    states, windows = r(S, W, N).to(DEV), r(S, W, 3).to(dtype).to(DEV)
    w, b = r(W, 1, 4).to(params).to(DEV), r(W).to(params).to(DEV)
    slots = torch.randperm(S, generator=g)[:B]
    if B > 2:
        slots[1], slots[2] = -1, S                          # padding of a captured batch
    d = lambda v: v.double().cpu()
    hs, ws = d(states).clone(), d(windows).clone()
    ys, cs = torch.zeros(B, W).double(), torch.zeros(B, W).double()
    for i, s in enumerate(slots.tolist()):
        if not 0 <= s < S:
            continue
        line = torch.cat([ws[s], d(x)[i][:, None]], 1)
        cs[i] = F.silu((line * d(w)[:, 0]).sum(1) + d(b))
        ws[s] = line[:, 1:]
        dt = F.softplus(d(delta)[i] + d(bias), threshold=1e9) if full else F.softplus(d(delta)[i]).to(dtype).double()
        hs[s] = torch.exp(dt[:, None] * d(A)) * hs[s] + (dt * d(x)[i])[:, None] * d(Bm)[i]
        ys[i] = hs[s] @ d(Cm)[i]
        if full:
            ys[i] = (ys[i] + d(D) * d(x)[i]) * F.silu(d(z)[i])
    given = dict(D=D, z=z, delta_bias=bias) if full else {}
    dl = delta if full else F.softplus(delta.double()).to(dtype)
    c, same = mamba_b200.conv_step_fn(x, windows, w, b, slots=slots.to(DEV))
    assert same is windows
    y, same = mamba_b200.ssm_step_fn(x, states, dl, A, Bm, Cm, **given, slots=slots.int().to(DEV))
    assert same is states
    close(c, cs, dtype, "conv")
    close(y, ys, dtype, "y")
    close(states, hs, what="states")
    assert torch.equal(d(windows), ws)
    idle = [s for s in range(S) if s not in slots.tolist()]
    assert torch.equal(d(states)[idle], hs[idle])


def plain_select(logits, scores, num, finished=None, end=None):
    G, K, V = logits.shape
    value = scores.double()[..., None] + torch.log_softmax(logits.double(), -1)
    none = ~torch.isfinite(scores) | torch.isnan(logits).any(-1) | (logits == math.inf).any(-1) | (logits == -math.inf).all(-1)
    value[none] = -math.inf
    if finished is not None:
        for g, k in torch.nonzero(finished).tolist():
            value[g, k] = -math.inf
            if torch.isfinite(scores[g, k]):
                value[g, k, end] = scores[g, k].double()
    best = torch.sort(value.view(G, -1), dim=-1, descending=True, stable=True)
    return best.values[:, :num], best.indices[:, :num] % V, best.indices[:, :num] // V


def check_select(logits, scores, num, finished=None, end=None):
    import mamba_b200
    s, t, p = mamba_b200.beam_select(logits, scores, num, finished=finished, end_token=end)
    ws, wt, wp = plain_select(logits.cpu(), scores.cpu(), num, None if finished is None else finished.cpu(), end)
    assert t.dtype == p.dtype == torch.int64 and s.dtype == torch.float32 and s.shape == (scores.shape[0], num)
    assert torch.equal(t.cpu(), wt) and torch.equal(p.cpu(), wp)
    s = s.cpu().double()
    same = s == ws
    assert (same | ((s - ws).abs() <= 1e-6 + 2.0 ** -24 * ws.abs())).all()


@pytest.mark.parametrize("G,K,V,num", [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 4), (3, 4, 33, 8), (1, 5, 8192, 10), (2, 2, 8193, 64), (1, 64, 3, 64),
                                       (2, 16, 20011, 32), (4, 4, 50280, 4), (1, 3, 128256, 6), (65, 2, 100, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select(G, K, V, num, dtype):
    g = torch.Generator().manual_seed(G + K + V)
    logits = (3 * torch.randn(G, K, V, generator=g)).to(dtype).to(DEV)          # bfloat16: full of equal logits
    scores = (-20 * torch.rand(G, K, generator=g)).to(DEV)
    check_select(logits, scores, num)
    finished = (torch.rand(G, K, generator=g) < 0.4).to(DEV)
    check_select(logits, scores, num, finished, V // 2)
    check_select(logits, scores, num, torch.ones_like(finished), 0)


def test_select_where_little_is_left():
    """-inf scores, masked logits, NaN, +inf, identical beams: what is no candidate comes last, lowest first."""
    G, K, V = 6, 4, 3000
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(G, K, V, generator=g)
    scores = -torch.rand(G, K, generator=g)
    scores[0, 1:] = -math.inf                               # the first step of a search
    logits[1, :, 3:] = -math.inf                            # three tokens a beam
    logits[2] = -math.inf                                   # nothing at all
    logits[3, 0, 17], logits[3, 1, 5], logits[3, 2] = math.nan, math.inf, -math.inf
    logits[4], scores[4] = logits[4, :1], scores[4, 0]      # beams alike
    logits[5, 1:, 1:] = torch.finfo(torch.float32).min      # a mask of the lowest value
    logits[5, 0, :] = 1.0
    for num in (1, 4, 16, 64):
        check_select(logits.to(DEV), scores.to(DEV), num)
        check_select(logits.to(DEV), scores.to(DEV), num, torch.tensor([[True, False, False, False]] * G, device=DEV), 1)
    scores[0, 0] = math.nan
    check_select(logits.to(DEV), scores.to(DEV), 9)


def test_select_masks_and_infinities():
    """A beam all of whose logits are the type's lowest value (uniform), very large ones, a NaN in a slice of -inf."""
    G, K, V = 5, 3, 9000
    g = torch.Generator().manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16):
        logits, scores = torch.randn(G, K, V, generator=g).to(dtype), -torch.rand(G, K, generator=g)
        logits[0] = torch.finfo(dtype).min
        logits[1, 0] = torch.finfo(dtype).max / 2
        logits[1, 1] = torch.finfo(dtype).max / 2 * (torch.rand(V, generator=g) - 0.5).to(dtype)
        logits[2, 0, 8192:] = -math.inf
        logits[2, 0, 8500] = math.nan
        logits[3, :, 8192:] = -math.inf
        logits[4, :] = 0.0                                  # everything equal
        for num in (1, 5, 33, 64):
            check_select(logits.to(DEV), scores.to(DEV), num)


def test_select_where_beams_are_alike():
    """Beams whose logits differ by a constant have the same candidates but for rounding: only 64 bits tell their order."""
    g = torch.Generator().manual_seed(2)
    base = torch.randn(4, 1, 20000, generator=g)
    check_select((base + torch.randn(4, 5, 1, generator=g)).to(DEV), torch.zeros(4, 5, device=DEV), 20)
    check_select((base + torch.randn(4, 5, 1, generator=g)).to(DEV), -torch.rand(4, 1, generator=g).repeat(1, 5).to(DEV), 40)


@pytest.mark.parametrize("K,V,num", [(64, 50280, 64), (40, 60000, 10), (64, 30000, 1), (33, 40000, 33)])
def test_select_of_more_slices_than_threads(K, V, num):
    """One group whose beams' slices are more than the joining CTA has threads; the second time with beams that only 64 bits tell apart."""
    g = torch.Generator().manual_seed(K)
    check_select(torch.randn(1, K, V, generator=g).to(DEV), -torch.rand(1, K, generator=g).to(DEV), num)
    alike = torch.randn(1, 1, V, generator=g) + torch.randn(1, K, 1, generator=g)
    check_select(alike.to(DEV), torch.zeros(1, K, device=DEV), num)
    check_select(alike.to(DEV).bfloat16(), torch.zeros(1, K, device=DEV), num, (torch.rand(1, K, generator=g) < 0.3).to(DEV), V - 1)


def test_select_strides_and_order():
    """Ascending logits (every thread's highest is its last), descending ones, views with other strides, an offset of one element."""
    g = torch.Generator().manual_seed(0)
    up = torch.arange(20000.).view(1, 2, 10000) / 1000
    check_select(up.to(DEV), torch.zeros(1, 2, device=DEV), 64)
    check_select(up.flip(-1).to(DEV), torch.zeros(1, 2, device=DEV), 64)
    big = torch.randn(3, 2, 4, 1001, generator=g).to(DEV)
    check_select(big[:, 1], torch.zeros(3, 4, device=DEV), 8)
    check_select(big[:, 0].transpose(0, 1), torch.zeros(4, 3, device=DEV), 8)
    check_select(big[..., 1:].reshape(-1)[1:1 + 2 * 3 * 999].view(2, 3, 999), torch.zeros(2, 3, device=DEV), 8)
    flat = torch.randn(6, 333, generator=g).to(DEV)
    import mamba_b200
    a, b = mamba_b200.beam_select(flat, torch.zeros(2, 3, device=DEV)), mamba_b200.beam_select(flat.view(2, 3, 333), torch.zeros(2, 3, device=DEV))
    assert all(torch.equal(u, v) for u, v in zip(a, b)) and a[0].shape == (2, 3)


def plain_reorder(slots, parents, pools):
    new, before = [], [p.clone() for p in pools]
    n = pools[0].shape[0] if pools else 0
    for own, par in zip(slots.tolist(), parents.tolist()):
        K = len(own)
        spare, seen, out = [own[k] for k in range(K) if k not in par], set(), []
        for p in par:
            if 0 <= p < K and p not in seen:
                seen.add(p)
                out.append(own[p])
                continue
            to = spare.pop(0)
            out.append(to)
            if 0 <= p < K and 0 <= own[p] < n and 0 <= to < n:
                for pool, old in zip(pools, before):
                    pool[to] = old[own[p]]
        new.append(out)
    return torch.tensor(new)


@pytest.mark.parametrize("G,K", [(1, 1), (1, 4), (3, 2), (2, 12), (64, 64), (5, 7)])
def test_reorder(G, K):
    import mamba_b200
    g = torch.Generator().manual_seed(G * K)
    S = G * K + 5
    pools = [torch.randn(S, 40, 16, generator=g), torch.randn(S, 40, 3, generator=g).bfloat16(), torch.randn(S, 7, 3, generator=g).bfloat16(),
             torch.randn(S, 9000, generator=g), torch.randint(0, 255, (S, 5), generator=g, dtype=torch.uint8), torch.zeros(S, 0)]
    slots = torch.randperm(S, generator=g)[: G * K].view(G, K)
    for case in range(4):
        parents = [torch.randint(0, K, (G, K), generator=g), torch.arange(K).repeat(G, 1), torch.zeros(G, K).long(),
                   torch.randint(-1, K + 1, (G, K), generator=g)][case]
        if case == 3:
            slots = slots.clone()
            slots[0, 0] = -1
        dev = [p.to(DEV) for p in pools]
        new = mamba_b200.beam_reorder(slots.to(DEV), parents.int().to(DEV), dev)
        want = [p.clone() for p in pools]
        assert torch.equal(new.cpu(), plain_reorder(slots, parents, want))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))


def test_reorder_by_many_ctas():
    """Enough to copy for every SM, and enough beams for several warps to work on the list: each CTA's share is of the same list."""
    import mamba_b200
    g = torch.Generator().manual_seed(0)
    G, K, S = 40, 16, 40 * 16
    pools = [torch.randn(S, 5000, generator=g), torch.randn(S, 12000, generator=g)]
    slots, parents = torch.randperm(S, generator=g).view(G, K), torch.randint(0, K, (G, K), generator=g)
    want = [p.clone() for p in pools]
    plain = plain_reorder(slots, parents, want)
    for _ in range(5):
        dev = [p.to(DEV) for p in pools]
        new = mamba_b200.beam_reorder(slots.to(DEV), parents.to(DEV), dev)
        assert torch.equal(new.cpu(), plain) and all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))


def test_reorder_of_many_pools_and_of_none():
    import mamba_b200
    g = torch.Generator().manual_seed(0)
    pools = [torch.randn(9, 3 + i, generator=g) for i in range(300)]
    slots, parents = torch.tensor([[0, 2, 4, 6]]), torch.tensor([[3, 3, 0, 3]])
    dev = [p.to(DEV) for p in pools]
    new = mamba_b200.beam_reorder(slots.to(DEV), parents.to(DEV), dev)
    want = [p.clone() for p in pools]
    assert torch.equal(new.cpu(), plain_reorder(slots, parents, want)) and all(torch.equal(a.cpu(), b) for a, b in zip(dev, want))
    assert torch.equal(mamba_b200.beam_reorder(slots.to(DEV), parents.to(DEV), []).cpu(), new.cpu())
