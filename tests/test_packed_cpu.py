"""CPU-side checks of packed sequences, slots and beams: the entry points refuse bad arguments before any CUDA call, sizes of workspaces
are those of their formulas, and CPU tensors are refused."""
import ctypes

import pytest
import torch

EINVAL, EDTYPE, ENSTATE, ETOOBIG = -1, -2, -3, -6


class Packed(ctypes.Structure):
    _fields_ = [("cu_seqlens", ctypes.c_void_p), ("sequences", ctypes.c_int64), ("rows", ctypes.c_int64), ("slots", ctypes.c_void_p),
                ("resume", ctypes.c_void_p), ("n_slots", ctypes.c_int64)]


def _lib():
    from mamba_b200 import _lib
    return _lib.load()


def _seqs(sequences=2, rows=20, cu=1 << 20, slots=None, n_slots=0):
    return ctypes.byref(Packed(cu, sequences, rows, slots, None, n_slots))


P = 1 << 20          # a pointer that is only compared with NULL and looked at for its alignment


@pytest.mark.parametrize("seqs,code", [(None, EINVAL), (dict(sequences=-1), EINVAL), (dict(rows=-1), EINVAL), (dict(n_slots=-1), EINVAL), (dict(cu=None), EINVAL),
                                       (dict(rows=1 << 30), ETOOBIG), (dict(sequences=65535), ETOOBIG)])
def test_sequences(seqs, code):
    lib = _lib()
    s = None if seqs is None else _seqs(**seqs)
    assert lib.mb200_sscan_packed_fwd(s, *[P] * 12, 32, 16, *[32] * 6, 0, 1, 0, 0, None) == code
    assert lib.mb200_sscan_packed_bwd(s, *[P] * 20, 32, 16, *[32] * 9, 0, 1, 0, 0, None) == code
    assert lib.mb200_conv1d_silu_packed_fwd(s, *[P] * 5, 32, 4, 32, 32, 0, None) == code
    assert lib.mb200_conv1d_silu_packed_bwd(s, *[P] * 7, 32, 4, 32, 32, 32, 0, None) == code


def test_scan_arguments():
    lib = _lib()

    def fwd(s=None, ptrs=None, ED=32, N=16, piece=0, parts=1, dtype=0, flags=0):
        return lib.mb200_sscan_packed_fwd(s or _seqs(), *(ptrs or [P] * 12), ED, N, *[32] * 6, piece, parts, dtype, flags, None)

    def bwd(s=None, ptrs=None, ED=32, N=16, piece=0, parts=1, dtype=0, flags=0):
        return lib.mb200_sscan_packed_bwd(s or _seqs(), *(ptrs or [P] * 20), ED, N, *[32] * 9, piece, parts, dtype, flags, None)

    for f, n in ((fwd, 12), (bwd, 20)):
        assert f(ED=-1) == EINVAL and f(piece=-16) == EINVAL and f(piece=24) == EINVAL and f(piece=48, parts=2) == EINVAL and f(parts=0) == EINVAL
        assert f(piece=1 << 40) == ETOOBIG and f(parts=1 << 60) == ETOOBIG and f(piece=16, parts=1 << 60) == ETOOBIG
        assert f(dtype=2) == EDTYPE and f(N=12) == ENSTATE
        assert f(s=_seqs(rows=0)) == 0 and f(ED=0) == 0                  # nothing to do
        assert f(ptrs=[None] + [P] * (n - 1)) == EINVAL                  # x
        no_bias = [P] * n
        no_bias[7] = None
        assert f(ptrs=no_bias, flags=1) == EINVAL                    # softplus without a bias
        assert f(flags=2) == -8                                          # right to left: unsupported
        assert f(N=8, piece=16) == EINVAL                                # cut for d_state 16 alone
    assert fwd(ptrs=[P] * 8 + [None] + [P] * 3, s=_seqs(slots=P, n_slots=4)) == EINVAL      # slots of no pool
    assert fwd(ptrs=[P] * 8 + [P + 4] + [P] * 3) == -4 and fwd(ptrs=[P] * 10 + [P + 8, P]) == -4   # states, carries off the grid
    assert bwd(s=_seqs(slots=P, n_slots=4)) == EINVAL                    # no gradient through slots
    assert lib.mb200_packed_parts(100, 3, 16) == 100 // 16 + 3 + 1 and lib.mb200_packed_parts(100, 3, 0) == 0
    assert lib.mb200_packed_saved_states(100, 3) == 100 // lib.mb200_sscan_chunk() + 3


def test_conv_arguments():
    lib = _lib()
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(), *[P] * 5, 32, 3, 32, 32, 0, None) == ETOOBIG          # d_conv 4 alone
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(), *[P] * 5, -1, 4, 32, 32, 0, None) == EINVAL
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(), *[P] * 5, 32, 4, 32, 32, 5, None) == EDTYPE
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(slots=P, n_slots=2), P, P, P, None, P, 32, 4, 32, 32, 0, None) == EINVAL
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(), None, P, P, None, P, 32, 4, 32, 32, 0, None) == EINVAL
    assert lib.mb200_conv1d_silu_packed_fwd(_seqs(rows=0), *[P] * 5, 32, 4, 32, 32, 0, None) == 0
    assert lib.mb200_conv1d_silu_packed_bwd(_seqs(slots=P, n_slots=2), *[P] * 7, 32, 4, 32, 32, 32, 0, None) == EINVAL
    assert lib.mb200_conv1d_silu_packed_bwd(_seqs(), *[P] * 4, None, P, P, 32, 4, 32, 32, 32, 0, None) == EINVAL


def test_step_arguments():
    lib = _lib()

    def scan(slots=P, n_slots=4, B=2, N=16, dtype=0, states=P):
        return lib.mb200_ssm_step_slots(P, P, P, P, 0, 0, P, P, P, 0, P, 0, states, slots, n_slots, P, B, 32, N, *[32] * 6, dtype, 0, None)

    def conv(slots=P, n_slots=4, B=2, K=4, windows=P):
        return lib.mb200_conv_step_slots(P, windows, slots, n_slots, P, 0, P, 0, P, B, 32, K, 32, 0, None)

    assert scan(slots=None) == EINVAL and scan(n_slots=-1) == EINVAL and scan(B=-1) == EINVAL and scan(N=12) == ENSTATE and scan(dtype=3) == EDTYPE
    assert scan(states=None) == EINVAL and scan(B=65536) == ETOOBIG and scan(states=P + 4) == -4 and scan(slots=None, B=0) == 0
    assert conv(slots=None) == EINVAL and conv(n_slots=-1) == EINVAL and conv(B=-1) == EINVAL and conv(K=9) == ETOOBIG and conv(K=0) == EINVAL
    assert conv(windows=None) == EINVAL and conv(B=65536) == ETOOBIG and conv(slots=None, B=0) == 0


def test_beam_arguments():
    lib = _lib()

    def select(groups=2, beams=3, V=9, num=3, end=0, stride=9, dtype=0, finished=None, logits=P, scratch=P):
        return lib.mb200_beam_select(logits, P, finished, scratch, P, P, P, groups, beams, V, num, end, stride, dtype, None)

    assert select(groups=-1) == EINVAL and select(beams=0) == EINVAL and select(V=0) == EINVAL and select(num=0) == EINVAL and select(num=28) == EINVAL
    assert select(dtype=2) == EDTYPE and select(finished=P, end=9) == EINVAL and select(finished=P, end=-1) == EINVAL
    assert select(beams=65) == ETOOBIG and select(V=99, num=65) == ETOOBIG and select(V=1 << 30) == ETOOBIG and select(groups=65536) == ETOOBIG
    assert select(groups=1 << 60, beams=64) == ETOOBIG and select(V=1 << 62) == ETOOBIG
    assert select(logits=None) == EINVAL and select(scratch=None) == EINVAL and select(scratch=P + 8) == -4 and select(groups=0) == 0
    assert lib.mb200_beam_select_scratch_bytes(0, 3, 9, 3) == 0 and lib.mb200_beam_select_scratch_bytes(1, 1, 0, 1) == 0

    def reorder(slots=P, parents=P + 64, out=P + 128, groups=2, beams=3, n_slots=9, pools=(P,), sizes=(64,)):
        n = len(pools)
        return lib.mb200_beam_reorder(slots, parents, out, groups, beams, n_slots, (ctypes.c_void_p * max(n, 1))(*pools), (ctypes.c_int64 * max(n, 1))(*sizes), n, None)

    assert reorder(groups=-1) == EINVAL and reorder(beams=-1) == EINVAL and reorder(n_slots=-1) == EINVAL and reorder(slots=None) == EINVAL
    assert reorder(out=P) == EINVAL and reorder(out=P + 64) == EINVAL and reorder(pools=(None,)) == EINVAL and reorder(sizes=(-1,)) == EINVAL
    assert reorder(beams=65) == ETOOBIG and reorder(groups=1366) == ETOOBIG and reorder(sizes=(1 << 31,)) == ETOOBIG and reorder(n_slots=1 << 31) == ETOOBIG
    assert reorder(groups=0) == 0 and reorder(beams=0) == 0


def test_cpu_tensors_are_refused():
    import mamba_b200
    x, A, B, cu = torch.zeros(4, 8), -torch.ones(8, 16), torch.zeros(4, 16), torch.tensor([0, 4])
    slots = torch.zeros(4, dtype=torch.long)
    for call in (lambda: mamba_b200.selective_scan_packed(x, x, A, B, B, cu_seqlens=cu),
                 lambda: mamba_b200.causal_conv1d_silu_packed(x, torch.zeros(8, 1, 4), cu_seqlens=cu),
                 lambda: mamba_b200.ssm_step_fn(x, torch.zeros(4, 8, 16), x, A, B, B, slots=slots),
                 lambda: mamba_b200.conv_step_fn(x, torch.zeros(4, 8, 3), torch.zeros(8, 1, 4), None, slots=slots),
                 lambda: mamba_b200.beam_select(torch.zeros(1, 4, 9), torch.zeros(1, 4)),
                 lambda: mamba_b200.beam_reorder(slots.view(1, 4), slots.view(1, 4), [])):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
