"""Sequences of different lengths laid end to end: scan and convolution with states in slots, and their gradients, against plain
implementations in 64 bits that take one sequence after the other.

Tolerances.  u = 2^-24 (float32), v = 2^-8 (bfloat16, half a step).  A scan's decay is off by a few u for the exponential and its argument's
rounding (|delta A| <= 8 here: 8 u), its input by the softplus (3e-7 = 5 u) and two products; through the recurrence the relative errors of all
steps are weighted by what is left of them, whose sum is the state's own scale: 32 u of that scale are counted, 2e-6.  The contraction adds 16 terms, and the
gate a sigmoid of 2 u.  Sums over rows (dA, dD, d bias) and channels (dB, dC) of n terms in float32 in any order: u sqrt(n) of the terms' scale more.
So float32 outputs are held to 1e-5 of the tensor's largest value, and bfloat16 ones to that and v of the value."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
V = 2.0 ** -8


def close(got, want, dtype=torch.float32, what=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, what
    if want.numel() == 0:
        return
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    bound = 1e-5 * want.abs().max() + (V * want.abs() * 1.001 if dtype == torch.bfloat16 else 0)
    off = (got - want).abs() - bound
    assert off.max() <= 1e-30, f"{what}: {off.max().item():.3g} over, largest {want.abs().max().item():.3g}"


def cu_of(lengths, dtype=torch.int32):
    return torch.tensor([0] + lengths).cumsum(0).to(dtype).to(DEV)


def inputs(seed, T, W, N=16, dtype=torch.float32, gate=True, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    t = {"x": r(T, W), "delta": r(T, W) * 0.5 - (0 if bias else 5), "A": -torch.exp(torch.log(torch.arange(1., N + 1)).repeat(W, 1) + 0.2 * r(W, N)),
         "B": r(T, N), "C": r(T, N), "D": 1 + 0.1 * r(W), "z": r(T, W) if gate else None, "delta_bias": r(W) * 0.5 - 3 if bias else None}
    if not bias:
        t["delta"] = F.softplus(t["delta"])
    for k in ("x", "delta", "B", "C", "z"):
        if t[k] is not None:
            t[k] = t[k].to(dtype)
    return {k: None if v is None else v.to(DEV) for k, v in t.items()}


def plain_scan(t, lengths, states=None, slots=None, resume=None):
    """One sequence after the other, one row after the other, in 64 bits on the CPU."""
    d = {k: None if v is None else v.double().cpu() if not v.requires_grad else v.double().cpu() for k, v in t.items()}
    T, W = d["x"].shape
    states = None if states is None else states.double().cpu().clone()
    ys, lo = [], 0
    for r, n in enumerate(lengths):
        s = slice(lo, lo + n)
        dt = d["delta"][s] if d["delta_bias"] is None else F.softplus(d["delta"][s] + d["delta_bias"], threshold=1e9)
        slot = int(slots[r]) if slots is not None else -1
        known = states is not None and 0 <= slot < len(states)
        h = states[slot].clone() if known and resume is not None and bool(resume[r]) else torch.zeros(W, d["A"].shape[1], dtype=torch.float64)
        for i in range(n):
            h = torch.exp(dt[i][:, None] * d["A"]) * h + (dt[i] * d["x"][lo + i])[:, None] * d["B"][lo + i]
            y = h @ d["C"][lo + i]
            if d["D"] is not None:
                y = y + d["D"] * d["x"][lo + i]
            ys.append(y if d["z"] is None else y * F.silu(d["z"][lo + i]))
        if known and n:
            states[slot] = h
        lo += n
    ys += [torch.zeros(W, dtype=torch.float64)] * (T - lo)
    return torch.stack(ys) if ys else torch.zeros(0, W, dtype=torch.float64), states


LENGTHS = [[1], [17], [16, 1, 31, 2], [0, 5, 0, 0, 40, 1, 1, 3, 0], [100, 7], [8, 8, 8], [33, 65, 15, 0], [3] * 30]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("W,N,dtype", [(32, 16, torch.float32), (40, 16, torch.bfloat16), (36, 16, torch.float32), (20, 8, torch.bfloat16),
                                       (5, 32, torch.float32), (72, 64, torch.float32), (96, 8, torch.float32)])
def test_scan_with_slots(lengths, W, N, dtype):
    import mamba_b200
    T = sum(lengths) + 3                                    # rows behind the last sequence
    t = inputs(T + W, T, W, N, dtype)
    R = len(lengths)
    g = torch.Generator().manual_seed(R)
    slots = torch.randperm(R + 2, generator=g)[:R]
    if R > 2:
        slots[2] = -1
    resume = torch.arange(R) % 2 == 0
    states = torch.randn(R + 2, W, N, generator=g).to(DEV)
    want, after = plain_scan(t, lengths, states, slots, resume)
    before = states.clone()
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of(lengths), states=states, slots=slots.to(DEV), resume=resume.to(DEV))
    assert y.dtype == dtype
    close(y, want, dtype, "y")
    close(states, after, what="states")
    untouched = [s for s in range(R + 2) if s not in [int(v) for v, n in zip(slots, lengths) if n]]
    assert torch.equal(states[untouched], before[untouched]) and (y[sum(lengths):] == 0).all()


@pytest.mark.parametrize("lengths", [[1], [16, 1, 31, 2], [0, 5, 0, 40, 1, 3, 0], [100, 7]])
@pytest.mark.parametrize("W,N,dtype", [(32, 16, torch.float32), (40, 16, torch.bfloat16), (36, 16, torch.float32), (20, 8, torch.bfloat16),
                                       (5, 32, torch.float32)])
@pytest.mark.parametrize("gate,bias", [(True, True), (False, False)])
def test_scan_gradients(lengths, W, N, dtype, gate, bias):
    import mamba_b200
    T = sum(lengths) + 2
    t = inputs(T + W, T, W, N, dtype, gate, bias)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items() if v is not None}
    y = mamba_b200.selective_scan_packed(**{**t, **leaves}, cu_seqlens=cu_of(lengths, torch.int64))
    dy = torch.randn(T, W, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    exact = {k: v.double().cpu().requires_grad_() for k, v in t.items() if v is not None}
    want, _ = plain_scan({**t, **exact}, lengths)
    close(y, want, dtype, "y")
    for k, a, b in zip(leaves, got, torch.autograd.grad(want, list(exact.values()), dy.double().cpu())):
        assert a.dtype == t[k].dtype
        close(a, b, a.dtype, "d" + k)


@pytest.mark.parametrize("lengths", [[200], [33, 160, 1, 64, 0, 49], [16, 32, 48], [5, 300]])
@pytest.mark.parametrize("piece", [16, 48, 64])
@pytest.mark.parametrize("W,dtype", [(32, torch.float32), (40, torch.bfloat16), (100, torch.float32)])
def test_pieces(lengths, piece, W, dtype):
    """Sequences cut into pieces: the same as uncut, with states and gradients."""
    import mamba_b200
    T = sum(lengths) + 37
    t = inputs(T + W, T, W, 16, dtype)
    R = len(lengths)
    slots, resume = torch.arange(R).flip(0), torch.arange(R) % 2 == 0
    pool = torch.randn(R + 1, W, 16, generator=torch.Generator().manual_seed(5)).to(DEV)
    want, after = plain_scan(t, lengths, pool, slots, resume)
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of(lengths), states=pool, slots=slots.to(DEV), resume=resume.to(DEV),
                                             piece_length=piece)
    close(y, want, dtype, "y")
    close(pool, after, what="states")
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn(T, W, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu_of(lengths), piece_length=piece)
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    exact = {k: v.double().cpu().requires_grad_() for k, v in t.items()}
    want, _ = plain_scan(exact, lengths)
    close(y, want, dtype, "y")
    for k, a, b in zip(leaves, got, torch.autograd.grad(want, list(exact.values()), dy.double().cpu())):
        close(a, b, a.dtype, "d" + k)


@pytest.mark.parametrize("lengths", [[700, 33, 200, 0, 97, 1], [1000], [192, 193, 191], [97, 96, 95] * 3])
@pytest.mark.parametrize("piece", [96, 192, 256])
@pytest.mark.parametrize("W,dtype", [(32, torch.float32), (40, torch.bfloat16)])
def test_pieces_in_parts(lengths, piece, W, dtype):
    """Pieces long enough for their carries to come in 2 to 4 parts."""
    test_pieces(lengths, piece, W, dtype)


def test_many_cut_sequences():
    """More sequences than a CTA has threads, some of them cut."""
    lengths = [3, 0, 1, 40, 2] * 80 + [130, 1, 70]
    test_pieces(lengths, 32, 32, torch.float32)


@pytest.mark.parametrize("piece", [0, 16])
def test_nothing_crosses_a_border(piece):
    """A sequence of NaN and infinities, and garbage behind the last one, leave the others as they are, bit for bit."""
    import mamba_b200
    lengths, T, W = [21, 13, 40], 80, 64
    t = inputs(3, T, W)
    cu = cu_of(lengths)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn(T, W, generator=torch.Generator().manual_seed(1)).to(DEV)
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu, piece_length=piece)
    clean = torch.autograd.grad(y, [leaves[k] for k in ("x", "delta", "z")], dy)
    bad, dbad = {k: v.clone() for k, v in t.items()}, dy.clone()
    for v in [bad[k] for k in ("x", "delta", "B", "C", "z")] + [dbad]:
        v[21:34:2] = float("nan")
        v[22:34:2] = float("inf")
        v[74:] = float("nan")
    other = {k: v.requires_grad_() for k, v in bad.items()}
    y2 = mamba_b200.selective_scan_packed(**other, cu_seqlens=cu, piece_length=piece)
    grads = torch.autograd.grad(y2, [other[k] for k in ("x", "delta", "z")], dbad)
    keep = torch.tensor(list(range(21)) + list(range(34, 74)), device=DEV)
    assert torch.equal(y[keep], y2[keep]) and (y2[74:] == 0).all()
    for a, b in zip(clean, grads):
        assert torch.equal(a[keep], b[keep]) and (b[74:] == 0).all()


def plain_conv(x, w, b, lengths, windows=None, slots=None, resume=None):
    x, w, b = x.double().cpu(), w.double().cpu(), None if b is None else b.double().cpu()
    windows = None if windows is None else windows.double().cpu().clone()
    W, lo, ys = x.shape[1], 0, []
    for r, n in enumerate(lengths):
        slot = int(slots[r]) if slots is not None else -1
        known = windows is not None and 0 <= slot < len(windows)
        head = windows[slot].t().clone() if known and resume is not None and bool(resume[r]) else torch.zeros(3, W, dtype=torch.float64)
        line = torch.cat([head, x[lo:lo + n]])
        if n:
            ys.append(F.silu(F.conv1d(line.t()[None], w, b, groups=W)[0].t()))
            if known:
                windows[slot] = line[-3:].t()
        lo += n
    ys.append(torch.zeros(x.shape[0] - lo, W, dtype=torch.float64))
    return torch.cat(ys), windows


# lengths that put first rows one and two rows in front of the borders of chunks (32 rows) and of CTAs (256)
CONV_LENGTHS = LENGTHS + [[31, 1, 1, 40], [30, 40], [31, 2, 40], [30, 1, 1, 1, 30], [255, 300], [254, 1, 1, 1, 200], [254, 2, 1, 100], [1] * 70,
                          [2] * 300]


@pytest.mark.parametrize("lengths", CONV_LENGTHS)
@pytest.mark.parametrize("W,dtype", [(32, torch.float32), (40, torch.bfloat16), (5, torch.float32), (130, torch.bfloat16)])
def test_conv_with_slots(lengths, W, dtype):
    import mamba_b200
    T, R = sum(lengths) + 3, len(lengths)
    g = torch.Generator().manual_seed(T + W)
    x, w, b = torch.randn(T, W, generator=g).to(dtype).to(DEV), torch.randn(W, 1, 4, generator=g).to(DEV), torch.randn(W, generator=g).to(DEV)
    slots = torch.randperm(R + 2, generator=g)[:R]
    if R > 2:
        slots[2] = R + 7
    resume = torch.rand(R, generator=g) < 0.7
    windows = torch.randn(R + 2, W, 3, generator=g).to(dtype).to(DEV)
    want, after = plain_conv(x, w, b, lengths, windows, slots, resume)
    with torch.no_grad():
        y = mamba_b200.causal_conv1d_silu_packed(x, w, b, cu_seqlens=cu_of(lengths), windows=windows, slots=slots.to(DEV), resume=resume.to(DEV))
    close(y, want, dtype, "y")
    assert torch.equal(windows.double().cpu(), after) and (y[sum(lengths):] == 0).all()


@pytest.mark.parametrize("lengths", CONV_LENGTHS + [[129, 127, 1, 128]])
@pytest.mark.parametrize("W,dtype,with_bias", [(32, torch.float32, True), (40, torch.bfloat16, True), (5, torch.float32, False)])
def test_conv_gradients(lengths, W, dtype, with_bias):
    import mamba_b200
    T = sum(lengths) + 5
    g = torch.Generator().manual_seed(T + W)
    t = [torch.randn(T, W, generator=g).to(dtype).to(DEV), torch.randn(W, 1, 4, generator=g).to(DEV)]
    if with_bias:
        t.append(torch.randn(W, generator=g).to(DEV))
    dy = torch.randn(T, W, generator=g).to(dtype).to(DEV)
    leaves, exact = [v.clone().requires_grad_() for v in t], [v.double().cpu().requires_grad_() for v in t]
    y = mamba_b200.causal_conv1d_silu_packed(*leaves, cu_seqlens=cu_of(lengths))
    want, _ = plain_conv(*exact, *([None] if not with_bias else []), lengths)
    close(y, want, dtype, "y")
    got, ref = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, exact, dy.double().cpu())
    for k, a, b in zip(("dx", "dw", "db"), got, ref):
        close(a, b, a.dtype, k)


def _many_lengths(total, seed):
    """Lengths of all kinds, so that first rows fall on every place of a box and of a warp's rows; the rest in one long sequence."""
    g = torch.Generator().manual_seed(seed)
    lengths = [1] * 20 + [2, 3, 0, 5] * 10 + torch.randint(1, 70, (60,), generator=g).tolist() + [0, 0, 255, 256, 257, 31, 32, 33]
    return lengths + [total - sum(lengths)]


def _fast_plain_conv(x, w, b, lengths, windows, slots, resume):
    """In 64 bits on the GPU, all sequences at once: each row's taps from a line of heads and rows."""
    W, R = x.shape[1], len(lengths)
    x, w = x.double(), w.double()[:, 0]
    heads = torch.zeros(R, 3, W, dtype=torch.float64, device=DEV)
    ok = (slots >= 0) & (slots < len(windows)) & resume
    heads[ok] = windows.double().transpose(1, 2)[slots[ok]]
    parts, lo = [], 0
    for r, n in enumerate(lengths):
        parts += [heads[r], x[lo:lo + n]]
        lo += n
    line = torch.cat(parts)
    taps = sum(line[k:line.shape[0] - 3 + k] * w[:, k] for k in range(4)) + b.double()
    keep = torch.cat([torch.arange(n) + sum(lengths[:r]) + 3 * r for r, n in enumerate(lengths)]).to(DEV)
    y = torch.cat([F.silu(taps[keep]), torch.zeros(x.shape[0] - lo, W, dtype=torch.float64, device=DEV)])
    after = windows.clone()
    at = 0
    for r, n in enumerate(lengths):
        if n and 0 <= int(slots[r]) < len(windows):
            after[int(slots[r])] = line[at + n:at + n + 3].t().to(windows.dtype)
        at += n + 3
    return y, after


@pytest.mark.parametrize("T,W,dtype", [(5300, 2048, torch.bfloat16), (9001, 1000, torch.bfloat16), (70001, 128, torch.bfloat16), (9000, 996, torch.bfloat16),
                                       (4000, 5120, torch.bfloat16), (5000, 2048, torch.float32)])
def test_conv_of_large_tensors(T, W, dtype):
    """Above the sizes at which a thread takes several channels and boxes come through tensor maps (996: off their grid)."""
    import mamba_b200
    lengths = _many_lengths(T - 45, T)
    R = len(lengths)
    g = torch.Generator(device=DEV).manual_seed(T + W)
    x, w, b = (torch.randn(*s, generator=g, device=DEV) for s in ((T, W), (W, 1, 4), (W,)))
    x = x.to(dtype)
    slots = torch.randperm(R + 2, generator=torch.Generator().manual_seed(R))[:R].to(DEV)
    slots[4] = -1
    resume = torch.rand(R, generator=g, device=DEV) < 0.7
    windows = torch.randn(R + 2, W, 3, generator=g, device=DEV).to(dtype)
    want, after = _fast_plain_conv(x, w, b, lengths, windows, slots, resume)
    for _ in range(3):                                      # the same each time: nobody reads a window that is written already
        pool = windows.clone()
        with torch.no_grad():
            y = mamba_b200.causal_conv1d_silu_packed(x, w, b, cu_seqlens=cu_of(lengths), windows=pool, slots=slots, resume=resume)
        close(y, want, dtype, "y")
        assert torch.equal(pool, after) and (y[T - 45:] == 0).all()


@pytest.mark.parametrize("T,W,dtype", [(5300, 2048, torch.bfloat16), (5000, 1024, torch.float32), (9001, 996, torch.bfloat16)])
def test_conv_gradients_of_large_tensors(T, W, dtype):
    import mamba_b200
    lengths = _many_lengths(T - 45, T)
    g = torch.Generator(device=DEV).manual_seed(T + W)
    t = [torch.randn(*s, generator=g, device=DEV) for s in ((T, W), (W, 1, 4), (W,))]
    t[0] = t[0].to(dtype)
    dy = torch.randn(T, W, generator=g, device=DEV).to(dtype)
    leaves, exact = [v.clone().requires_grad_() for v in t], [v.double().requires_grad_() for v in t]
    y = mamba_b200.causal_conv1d_silu_packed(*leaves, cu_seqlens=cu_of(lengths))
    none = torch.full((len(lengths),), -1, device=DEV)
    want, _ = _fast_plain_conv(*exact, lengths, torch.zeros(1, W, 3, device=DEV), none, none > 0)
    close(y, want, dtype, "y")
    for k, a, b in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, exact, dy.double())):
        close(a, b, a.dtype, k)


def test_conv_garbage_behind_and_across():
    import mamba_b200
    lengths, W = [21, 13, 40], 64
    g = torch.Generator().manual_seed(0)
    x, w, b = torch.randn(90, W, generator=g).to(DEV), torch.randn(W, 1, 4, generator=g).to(DEV), torch.randn(W, generator=g).to(DEV)
    dy = torch.randn(90, W, generator=g).to(DEV)
    def run(x, dy):
        x = x.clone().requires_grad_()
        y = mamba_b200.causal_conv1d_silu_packed(x, w, b, cu_seqlens=cu_of(lengths))
        return y.detach(), torch.autograd.grad(y, x, dy)[0]
    y, dx = run(x, dy)
    x, dy = x.clone(), dy.clone()
    for v in (x, dy):
        v[21:34], v[74:] = float("nan"), float("inf")
    y2, dx2 = run(x, dy)
    keep = torch.tensor(list(range(21)) + list(range(34, 74)), device=DEV)
    assert torch.equal(y[keep], y2[keep]) and torch.equal(dx[keep], dx2[keep]) and (y2[74:] == 0).all() and (dx2[74:] == 0).all()
