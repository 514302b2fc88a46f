"""Packed scans whose 32-channel tiles are a few more than the SMs and whose 48-channel ones are not: they take a kernel of their own.  Tolerances as for
the other packed scans."""
import pytest
import torch

from tests.test_gpu_packed import DEV, close, cu_of, inputs, plain_scan

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def is_wide(items, W):
    return items * -(-W // 32) > sms() and items * -(-W // 48) <= sms()


@pytest.mark.parametrize("length", [1, 16, 61, 130])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate,bias", [(True, True), (False, False)])
def test_one_prompt(length, dtype, gate, bias):
    """One uncut prompt of a wide layer, on a slot that resumes and on one that does not, with rows behind it."""
    import mamba_b200
    W = 32 * (sms() + 12)
    assert is_wide(1, W)
    t = inputs(length, length + 5, W, 16, dtype, gate, bias)
    for resume in (True, False):
        pool = torch.randn(3, W, 16, generator=torch.Generator().manual_seed(1)).to(DEV)
        want, after = plain_scan(t, [length], pool, [2], [resume])
        with torch.no_grad():
            y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of([length]), states=pool, slots=torch.tensor([2], device=DEV),
                                                 resume=torch.tensor([resume], device=DEV), piece_length=0)
        close(y, want, dtype, "y")
        close(pool, after, what="states")
        assert (y[length:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [[33, 1, 0, 40], [17, 16, 15, 50]])
def test_documents(lengths, dtype):
    """A few uncut documents of a 1536-wide layer, with every gradient and with slots."""
    import mamba_b200
    W, R = 1536, sms() // 48 + 1
    lengths = (lengths * R)[:R]
    assert is_wide(R, W)
    T = sum(lengths) + 3
    t = inputs(T, T, W, 16, dtype)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu_of(lengths), piece_length=0)
    dy = torch.randn(T, W, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    exact = {k: v.double().cpu().requires_grad_() for k, v in t.items()}
    want, _ = plain_scan(exact, lengths)
    close(y, want, dtype, "y")
    for k, a, b in zip(leaves, got, torch.autograd.grad(want, list(exact.values()), dy.double().cpu())):
        close(a, b, a.dtype, "d" + k)
    pool, slots, resume = torch.randn(R + 1, W, 16, generator=torch.Generator().manual_seed(2)).to(DEV), torch.arange(R).flip(0), torch.arange(R) % 2 == 0
    want, after = plain_scan(t, lengths, pool, slots, resume)
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of(lengths), states=pool, slots=slots.to(DEV), resume=resume.to(DEV), piece_length=0)
    close(y, want, dtype, "y")
    close(pool, after, what="states")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("piece", [16, 96])
def test_cut(piece, dtype):
    """Few channels and many pieces, whose carries are folded as they start."""
    import mamba_b200
    W, n = 40, sms() * 2 // 3
    T = n * piece + 7
    lengths = [T // 2, 5, 0, T - T // 2 - 5 - 30]
    assert is_wide(T // piece + len(lengths), W)
    t = inputs(T, T, W, 16, dtype)
    slots, resume = torch.tensor([3, 1, 0, 2]), torch.tensor([True, False, True, True])
    pool = torch.randn(5, W, 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    want, after = plain_scan(t, lengths, pool, slots, resume)
    with torch.no_grad():
        y = mamba_b200.selective_scan_packed(**t, cu_seqlens=cu_of(lengths), states=pool, slots=slots.to(DEV), resume=resume.to(DEV), piece_length=piece)
    close(y, want, dtype, "y")
    close(pool, after, what="states")
    if piece > 16:
        return
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    dy = torch.randn(T, W, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    y = mamba_b200.selective_scan_packed(**leaves, cu_seqlens=cu_of(lengths), piece_length=piece)
    got = torch.autograd.grad(y, list(leaves.values()), dy)
    exact = {k: v.double().cpu().requires_grad_() for k, v in t.items()}
    want, _ = plain_scan(exact, lengths)
    close(y, want, dtype, "y")
    for k, a, b in zip(leaves, got, torch.autograd.grad(want, list(exact.values()), dy.double().cpu())):
        close(a, b, a.dtype, "d" + k)
