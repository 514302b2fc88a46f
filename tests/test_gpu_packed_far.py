"""Packed sequences, slots and beams at the ends of their ranges: entries and rows more than 2^31 elements from the start, broadcast and
strided tensors, parameters of other shapes, as many sequences as there may be.  Compared with the same operators on small tensors, exactly
where the arithmetic is the same, and otherwise within 1e-5 of the largest value (two splits of the same sums in float32)."""
import pytest
import torch

from tests.test_gpu_packed import DEV, close, cu_of, inputs, plain_scan

pytestmark = pytest.mark.gpu


def one_step(got, want):
    """Two roundings of nearly the same value: at most one bfloat16 step (2^-7 of the value) apart."""
    got, want = got.double(), want.double()
    assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-5 * want.abs().max()).all()


def test_slots_behind_2_to_the_31():
    import mamba_b200
    W, N, T = 1024, 16, 40
    S = 2 ** 31 // (W * N) + 6
    t = inputs(1, T, W, dtype=torch.bfloat16)
    cu, far = cu_of([25, 15]), torch.tensor([S - 1, S - 4], device=DEV)
    near = torch.tensor([5, 2], device=DEV)
    big, small = torch.zeros(S, W, N, device=DEV), torch.zeros(6, W, N, device=DEV)
    small[near] = torch.randn(2, W, N, device=DEV)
    big[far] = small[near]
    resume = torch.tensor([True, False], device=DEV)
    with torch.no_grad():
        for piece in (0, 16):
            got = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu, states=big, slots=far, resume=resume, piece_length=piece)
            want = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu, states=small, slots=near, resume=resume, piece_length=piece)
            assert torch.equal(got, want) and torch.equal(big[far], small[near])
        rows = {k: t[k][:2] for k in ("x", "delta", "B", "C", "z")}
        y, _ = mamba_b200.ssm_step_fn(h=big, A=t["A"], D=t["D"], delta_bias=t["delta_bias"], slots=far, **rows)
        w, _ = mamba_b200.ssm_step_fn(h=small, A=t["A"], D=t["D"], delta_bias=t["delta_bias"], slots=near, **rows)
        assert torch.equal(y, w) and torch.equal(big[far], small[near])
        parents = torch.tensor([[1, 1]], device=DEV)
        new = mamba_b200.beam_reorder(far.view(1, 2), parents, [big])
        assert new.tolist() == [[S - 4, S - 1]] and torch.equal(big[S - 1], small[2]) and torch.equal(big[S - 4], small[2])
    assert not big[:S - 6].any()


def test_windows_behind_2_to_the_31():
    import mamba_b200
    W, T = 4096, 40
    S = 2 ** 31 // (W * 3) + 6
    x, weight = torch.randn(T, W, device=DEV).bfloat16(), torch.randn(W, 1, 4, device=DEV)
    cu, far, near = cu_of([25, 15]), torch.tensor([S - 1, S - 4], device=DEV), torch.tensor([5, 2], device=DEV)
    big, small = torch.zeros(S, W, 3, device=DEV, dtype=torch.bfloat16), torch.randn(6, W, 3, device=DEV).bfloat16()
    big[far] = small[near]
    resume = torch.tensor([True, False], device=DEV)
    with torch.no_grad():
        for x_ in (x, torch.randn(T, W + 1, device=DEV).bfloat16()[:, 1:]):         # with and without a tensor map
            got = mamba_b200.causal_conv1d_silu_packed(x_, weight, cu_seqlens=cu, windows=big, slots=far, resume=resume)
            want = mamba_b200.causal_conv1d_silu_packed(x_, weight, cu_seqlens=cu, windows=small, slots=near, resume=resume)
            assert torch.equal(got, want) and torch.equal(big[far], small[near])
        got, _ = mamba_b200.conv_step_fn(x[:2], big, weight, None, slots=far)
        want, _ = mamba_b200.conv_step_fn(x[:2], small, weight, None, slots=near)
        assert torch.equal(got, want) and torch.equal(big[far], small[near])
    assert not big[:S - 6].any()


@pytest.mark.parametrize("off", [0, 1])
def test_rows_behind_2_to_the_31(off):
    """The last sequences of tensors of more than 2^31 values, on the 16-byte grid and off it, against the same sequences alone."""
    import mamba_b200
    W, last = 5120, [70, 3, 200]
    T = 2 ** 31 // W + 300
    g = torch.Generator(DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    buf = torch.zeros(T, W + 8, device=DEV, dtype=torch.bfloat16)
    x = buf[:, off:W + off]
    n = sum(last)
    x[T - n:] = r(n, W).bfloat16()
    delta = x
    A, BC = -torch.rand(W, 16, generator=g, device=DEV), torch.zeros(T, 32, device=DEV, dtype=torch.bfloat16)
    BC[T - n:] = r(n, 32).bfloat16()
    bias = r(W) * 0.5 - 3
    cu = cu_of([T - n] + last)
    tail = slice(T - n, T)
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(x, delta, A, BC[:, :16], BC[:, 16:], None, None, bias, cu_seqlens=cu, piece_length=0)[tail].clone()
        want = mamba_b200.selective_scan_packed(x[tail], delta[tail], A, BC[tail, :16], BC[tail, 16:], None, None, bias, cu_seqlens=cu_of(last), piece_length=0)
        assert torch.equal(y, want)
        weight = r(W, 1, 4)
        y = mamba_b200.causal_conv1d_silu_packed(x, weight, cu_seqlens=cu)[tail].clone()
        assert torch.equal(y, mamba_b200.causal_conv1d_silu_packed(x[tail], weight, cu_seqlens=cu_of(last)))
    leaf, w = x.detach().requires_grad_(), weight.requires_grad_()
    got, = torch.autograd.grad(mamba_b200.causal_conv1d_silu_packed(leaf, w, cu_seqlens=cu), leaf, x)
    got = got[tail].clone()
    alone = x[tail].detach().requires_grad_()
    want, = torch.autograd.grad(mamba_b200.causal_conv1d_silu_packed(alone, w, cu_seqlens=cu_of(last)), alone, x[tail])
    one_step(got, want)
    del got, leaf
    leaf = x.detach().requires_grad_()
    call = lambda u, d, bc, c: mamba_b200.selective_scan_packed(u, d, A, bc[:, :16], bc[:, 16:], None, None, bias, cu_seqlens=c, piece_length=0)
    got, = torch.autograd.grad(call(leaf, delta, BC, cu), leaf, x)
    got = got[tail].clone()
    want, = torch.autograd.grad(call(alone, delta[tail], BC[tail], cu_of(last)), alone, x[tail])
    one_step(got, want)


def test_as_many_sequences_as_there_may_be():
    import mamba_b200
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 4, (65534,), generator=g).tolist()
    W = 32
    t = inputs(2, sum(lengths) + 3, W)
    cu = cu_of(lengths)
    where = torch.randperm(65534, generator=g).to(DEV)
    states = torch.zeros(65534, W, 16, device=DEV)
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu, states=states, slots=where, max_length=3)
    want, pool = plain_scan(t, lengths, torch.zeros(65534, W, 16), where.cpu())
    close(y, want, what="y")
    close(states, pool, what="states")
    with pytest.raises(RuntimeError, match="limit"):
        mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of(lengths + [0]))


@pytest.mark.parametrize("W", [32, 37])
def test_broadcast_and_strided_inputs(W):
    """Rows and columns of stride 0, transposed tensors, every second row, D and the bias as (1, ED), a gradient that is one broadcast number."""
    import mamba_b200
    lengths = [30, 2, 50]
    T = sum(lengths)
    t = inputs(7, T, W)
    cu = cu_of(lengths, torch.int64)
    odd = dict(t, x=t["x"].t().contiguous().t(), delta=t["delta"][:1].expand(T, W), B=torch.stack([t["B"], t["C"]], 1).view(2 * T, 16)[::2],
               z=t["z"][:, :1].expand(T, W))
    odd["D"], odd["delta_bias"] = t["D"].view(1, W), t["delta_bias"].view(W, 1)
    same = {k: v.contiguous() for k, v in odd.items()}
    same["D"], same["delta_bias"] = t["D"], t["delta_bias"]
    runs = []
    for q in (odd, same):
        leaves = {k: v.detach().requires_grad_() for k, v in q.items()}
        y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu)
        runs.append((y, torch.autograd.grad(y.sum(), list(leaves.values()))))
    close(runs[0][0], runs[1][0], what="y")
    for k, a, b in zip(odd, runs[0][1], runs[1][1]):
        assert a.shape == odd[k].shape
        close(a.reshape(b.shape), b, what=k)
    weight, bias = torch.randn(W, 1, 4, device=DEV, requires_grad=True), torch.randn(1, W, device=DEV, requires_grad=True)
    runs = []
    for x in (odd["x"], same["x"], t["x"][:1].expand(T, W), t["x"][:1].repeat(T, 1)):
        leaf = x.detach().requires_grad_()
        y = mamba_b200.causal_conv1d_silu_packed(leaf, weight, bias, cu_seqlens=cu)
        runs.append((y, *torch.autograd.grad(y.sum(), (leaf, weight, bias))))
    for a, b in (runs[:2], runs[2:]):
        for u, v in zip(a, b):
            close(u, v)


def test_the_last_choice_of_a_large_vocabulary():
    """Logits of more than 2^31 values: the rows at the end."""
    import mamba_b200
    G, K, V = 4100, 4, 131072
    logits = torch.zeros(G, K, V, device=DEV, dtype=torch.bfloat16)
    logits[-2:] = torch.randn(2, K, V, device=DEV).bfloat16()
    scores = torch.randn(G, K, device=DEV)
    got = mamba_b200.beam_select(logits, scores)
    want = mamba_b200.beam_select(logits[-2:].clone(), scores[-2:].clone())
    assert torch.equal(got[0][-2:], want[0]) and torch.equal(got[1][-2:], want[1]) and torch.equal(got[2][-2:], want[2])


@pytest.mark.parametrize("piece", [0, 32])
def test_backward_twice_and_mixed_types(piece):
    """One forward, two backward passes; activations and parameters of different types get gradients of their own."""
    import mamba_b200
    lengths = [100, 0, 37]
    t = inputs(11, sum(lengths), 64, dtype=torch.bfloat16)
    t["z"], t["A"], t["D"] = t["z"].float(), t["A"].bfloat16(), t["D"].bfloat16()
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu_of(lengths), piece_length=piece)
    dy = torch.randn_like(y)
    first = torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)
    second = torch.autograd.grad(y, list(leaves.values()), dy)
    wide = {k: v.detach().float().requires_grad_() for k, v in t.items()}
    want = torch.autograd.grad(mamba_b200.selective_scan_packed(**wide, cu_seqlens=cu_of(lengths), piece_length=piece), list(wide.values()), dy.float())
    for (k, v), a, b, w in zip(leaves.items(), first, second, want):
        assert a.dtype == b.dtype == v.dtype and a.shape == v.shape
        close(a, w, v.dtype, what=k)
        one_step(a, b) if v.dtype == torch.bfloat16 else close(a, b, what=k)
