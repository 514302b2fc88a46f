"""Offsets and slots of any kind: packed scans and convolutions, forward and backward, through the C entry points, with every tensor that they are given
a view inside a larger one.  What surrounds the views, slots that no sequence has and the inputs are bit for bit as before, whatever the offsets are."""
import ctypes

import pytest
import torch

from tests.test_gpu_packed import DEV, inputs
from tests.test_packed_cpu import Packed

pytestmark = pytest.mark.gpu
GUARD, EDGE = 7.0, 8


class Frames:
    """Views inside tensors of GUARD, and whether all that surrounds them still is."""

    def __init__(self):
        self.all = []

    def rows(self, *shape, dtype=torch.float32, value=None):
        """(rows, ...) with EDGE rows more in front and behind, and EDGE columns more on both sides of a matrix."""
        wide = len(shape) == 2
        big = torch.full((shape[0] + 2 * EDGE, *(shape[1:-1] if wide else shape[1:]), *([shape[-1] + 2 * EDGE] if wide else [])), GUARD, dtype=dtype, device=DEV)
        view = big[EDGE:EDGE + shape[0]]
        if wide:
            view = view[:, EDGE:EDGE + shape[1]]
        if value is not None:
            view.copy_(value)
        self.all.append((big, view))
        return view

    def flat(self, *shape, dtype=torch.float32):
        """A dense tensor of zeros in the middle of a longer one."""
        n = 1
        for s in shape:
            n *= s
        big = torch.full((n + 64,), GUARD, dtype=dtype, device=DEV)
        view = big[32:32 + n].view(shape)
        view.zero_()
        self.all.append((big, view))
        return view

    def whole(self):
        for big, view in self.all:
            inside = view.clone()
            view.fill_(GUARD)
            ok = bool((big == GUARD).all())
            view.copy_(inside)
            if not ok:
                return False
        return True


def offsets_of(kind, T):
    if kind == "many":
        return torch.randint(-T // 3, T + T // 3, (701,), generator=torch.Generator().manual_seed(0)).tolist()
    if kind == "many, rising":
        return sorted(offsets_of("many", T))
    return {"fall": [0, 30, 10, 40], "backwards": [5, 4, 3, 2], "beyond": [0, 100, 20, T + 60], "far": [-5, 10, 2000000000, -7], "behind the end": [T, T, 0, 0],
            "nothing": [0, 0, 0, 0], "most": [3, 11, 12, 2 ** 31 - 1], "least": [-2 ** 31, -2 ** 31, 7, 9]}[kind]


KINDS = ["fall", "backwards", "beyond", "far", "behind the end", "nothing", "most", "least", "many", "many, rising"]


def sequences(kind, T, where, n_slots):
    cu = torch.tensor(offsets_of(kind, T), dtype=torch.int32, device=DEV)
    R = len(cu) - 1
    slots = torch.full((R,), -1, device=DEV)
    slots[:3] = torch.tensor(where, device=DEV)
    if R > 3:
        slots[3:] = torch.arange(R - 3, device=DEV) * 2 ** 31 + n_slots         # all of them outside
    resume = torch.arange(R, device=DEV) % 2 == 0
    return cu, slots, resume


def p(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("kind", KINDS)
# (cut for d_state 16 and tensors that tensor maps describe)
@pytest.mark.parametrize("W,N,dtype,piece,parts", [(32, 16, torch.float32, 0, 1), (32, 16, torch.float32, 16, 1), (32, 16, torch.float32, 96, 2),
                                                   (40, 16, torch.bfloat16, 0, 1), (40, 16, torch.bfloat16, 16, 1), (40, 16, torch.bfloat16, 96, 2),
                                                   (37, 16, torch.float32, 0, 1), (24, 8, torch.bfloat16, 0, 1), (20, 64, torch.float32, 0, 1)])
def test_scan(kind, W, N, dtype, piece, parts):
    from mamba_b200 import _lib
    lib, T, S, code = _lib.load(), 300, 4, _lib.dtype_code(dtype)
    f, t = Frames(), inputs(0, T, W, N, dtype)
    x, delta, z, dy = (f.rows(T, W, dtype=dtype, value=t[k]) for k in ("x", "delta", "z", "x"))
    B, C = (f.rows(T, N, dtype=dtype, value=t[k]) for k in ("B", "C"))
    A, D, bias = f.flat(W, N), f.flat(W), f.flat(W)
    A.copy_(t["A"]), D.copy_(t["D"]), bias.copy_(t["delta_bias"])
    given = [v.clone() for v in (x, delta, z, dy, B, C, A, D, bias)]
    for where in ([2, -1, 4], [0, 3, 2 ** 31]):
        cu, slots, resume = sequences(kind, T, where, S)
        R = len(cu) - 1
        pool = torch.full((S + 2, W, N), 3.0, device=DEV)
        states = pool[1:S + 1]
        y = f.rows(T, W, dtype=dtype)
        pieces = f.flat(2, lib.mb200_packed_parts(T, R, piece // parts), W, N) if piece else None
        seqs = Packed(cu.data_ptr(), R, T, slots.data_ptr(), resume.data_ptr(), S)
        strides = lambda *ts: [v.stride(0) for v in ts]
        rc = lib.mb200_sscan_packed_fwd(ctypes.byref(seqs), p(x), p(delta), p(z), p(A), p(B), p(C), p(D), p(bias), p(states), p(y), None, p(pieces), W, N,
                                        *strides(x, delta, z, B, C, y), piece, parts, code, 1, stream())
        assert rc == 0
        named = [s for s in where if 0 <= s < S]
        assert (pool[0] == 3).all() and (pool[-1] == 3).all()
        assert all((states[s] == 3).all() for s in range(S) if s not in named)
    # without slots: with saved states, and the backward
    cu = sequences(kind, T, [0, 0, 0], S)[0]
    seqs = Packed(cu.data_ptr(), R, T, None, None, 0)
    y, dx, dd, dz = (f.rows(T, W, dtype=dtype) for _ in range(4))
    saved = f.flat(lib.mb200_packed_saved_states(T, R), W, N)
    grads = f.flat(lib.mb200_packed_parts(T, R, piece // parts), W, N) if piece else None
    dB, dC, dA, dD, db = f.flat(T, N), f.flat(T, N), f.flat(W, N), f.flat(W), f.flat(W)
    flags = 1 | _lib.PAIRED_STATES
    assert lib.mb200_sscan_packed_fwd(ctypes.byref(seqs), p(x), p(delta), p(z), p(A), p(B), p(C), p(D), p(bias), None, p(y), p(saved), p(pieces), W, N,
                                      *strides(x, delta, z, B, C, y), piece, parts, code, flags, stream()) == 0
    assert lib.mb200_sscan_packed_bwd(ctypes.byref(seqs), p(x), p(delta), p(z), p(A), p(B), p(C), p(D), p(bias), p(dy), p(saved), p(pieces), p(grads),
                                      p(dx), p(dd), p(dz), p(dB), p(dC), p(dA), p(dD), p(db), W, N, *strides(x, delta, z, B, C, dy, dx, dd, dz),
                                      piece, parts, code, flags, stream()) == 0
    assert f.whole()
    assert all(torch.equal(a, b) for a, b in zip(given, (x, delta, z, dy, B, C, A, D, bias)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,W,dtype", [(300, 64, torch.float32), (300, 128, torch.bfloat16), (300, 37, torch.float32), (300, 37, torch.bfloat16),
                                       (5000, 1024, torch.float32), (8000, 1024, torch.bfloat16)])
def test_convolution(kind, T, W, dtype):
    from mamba_b200 import _lib
    lib, S, code = _lib.load(), 4, _lib.dtype_code(dtype)
    f, g = Frames(), torch.Generator(DEV).manual_seed(W)
    x, dy = (f.rows(T, W, dtype=dtype, value=torch.randn(T, W, generator=g, device=DEV)) for _ in range(2))
    w, bias = f.flat(W, 4), f.flat(W)
    w.normal_(generator=g), bias.normal_(generator=g)
    given = [v.clone() for v in (x, dy, w, bias)]
    for where in ([2, -1, 4], [0, 3, 2 ** 31]):
        cu, slots, resume = sequences(kind, T, where, S)
        R = len(cu) - 1
        pool = torch.full((S + 2, W, 3), 3.0, dtype=dtype, device=DEV)
        windows, y = pool[1:S + 1], f.rows(T, W, dtype=dtype)
        seqs = Packed(cu.data_ptr(), R, T, slots.data_ptr(), resume.data_ptr(), S)
        assert lib.mb200_conv1d_silu_packed_fwd(ctypes.byref(seqs), p(x), p(w), p(bias), p(windows), p(y), W, 4, x.stride(0), y.stride(0), code, stream()) == 0
        named = [s for s in where if 0 <= s < S]
        assert (pool[0] == 3).all() and (pool[-1] == 3).all() and all((windows[s] == 3).all() for s in range(S) if s not in named)
    seqs = Packed(cu.data_ptr(), R, T, None, None, 0)
    dx, dw, db = f.rows(T, W, dtype=dtype), f.flat(W, 4), f.flat(W)
    assert lib.mb200_conv1d_silu_packed_bwd(ctypes.byref(seqs), p(x), p(w), p(bias), p(dy), p(dx), p(dw), p(db), W, 4, x.stride(0), dy.stride(0), dx.stride(0),
                                            code, stream()) == 0
    assert f.whole()
    assert all(torch.equal(a, b) for a, b in zip(given, (x, dy, w, bias)))


@pytest.mark.parametrize("W,N,dtype", [(32, 16, torch.float32), (40, 16, torch.bfloat16), (37, 16, torch.float32), (20, 8, torch.float32)])
def test_steps(W, N, dtype):
    """Slots just outside the pool, and far outside."""
    from mamba_b200 import _lib
    lib, S, code = _lib.load(), 4, _lib.dtype_code(dtype)
    where = [2, -1, 4, 0, 2 ** 31, -2 ** 62, 2 ** 62, 2 ** 32 + 1]
    n = len(where)
    f, t = Frames(), inputs(1, n, W, N, dtype)
    x, delta, z = (f.rows(n, W, dtype=dtype, value=t[k]) for k in ("x", "delta", "z"))
    B, C, y = f.rows(n, N, dtype=dtype, value=t["B"]), f.rows(n, N, dtype=dtype, value=t["C"]), f.rows(n, W, dtype=dtype)
    xc, slots = f.flat(n, W, dtype=dtype), torch.tensor(where, device=DEV)
    pool, windows = torch.full((S + 2, W, N), 3.0, device=DEV), torch.full((S + 2, W, 3), 3.0, dtype=dtype, device=DEV)
    assert lib.mb200_ssm_step_slots(p(x), p(delta), p(z), p(t["A"]), 0, 0, p(B), p(C), p(t["D"]), 0, p(t["delta_bias"]), 0, p(pool[1:]), p(slots), S, p(y), n, W, N,
                                    x.stride(0), delta.stride(0), z.stride(0), B.stride(0), C.stride(0), y.stride(0), code, 1, stream()) == 0
    w = torch.randn(W, 4, device=DEV)
    assert lib.mb200_conv_step_slots(p(x), p(windows[1:]), p(slots), S, p(w), 0, None, 0, p(xc), n, W, 4, x.stride(0), code, stream()) == 0
    for v in (pool, windows):
        assert all((v[i] == 3).all() for i in (0, 2, 4, S + 1)) and all((v[1 + s] != 3).any() for s in (0, 2))
    outside = [i for i, s in enumerate(where) if not 0 <= s < S]
    assert (y[outside] == 0).all() and (xc[outside] == 0).all() and f.whole()
