"""Scratch of the column sums (csrc/ghm_gemm.hip colsum_plan / wcolsum_plan): what the *_part_elems functions
say is enough for every call of at most that many rows, and the plans' buffers hold every call of their
own backward.  The number of chunks does not grow with the rows (494 for 10,368 of them, 512 for 10,240), so
a buffer sized by the plan of all rows was too small for the text rows alone."""
import ctypes

import pytest
import torch


def _lib():
    from ghmclip import _native
    return _native.hip_lib()


def _wcolsum_floats(M, N, C):
    """What ghm_wcolsum writes to its scratch: chunks x (C N sums and the class totals, padded)."""
    n = max(1, min((M + 7) // 8, 512))
    rows = -(-M // n)
    return -(-M // rows) * (C * N + 4 * ((C + 3) // 4))


def _colsum_floats(M, N):
    col_blocks = 1 if N // 4 < 256 else (N // 4 + 255) // 256
    n = max(1, min(max(1, 256 // col_blocks), (M + 7) // 8))
    rows = -(-M // n)
    return -(-M // rows) * N


@pytest.mark.parametrize("N,C", [(256, 10), (128, 64), (512, 1)])
def test_weighted_sums_scratch_is_enough_for_fewer_rows(N, C):
    most = 0
    for M in range(1, 24000):
        most = max(most, _wcolsum_floats(M, N, C))
        assert _lib().ghm_wcolsum_part_elems(M, N, C) >= most, M


@pytest.mark.parametrize("N", [64, 1024, 81 * 256])
def test_column_sums_scratch_is_enough_for_fewer_rows(N):
    most = 0
    for M in range(1, 24000):
        most = max(most, _colsum_floats(M, N))
        assert _lib().ghm_colsum_part_elems(M, N) >= most, M


def _calls(monkeypatch, run):
    """The calls of run() with no device: (name, arguments as numbers)."""
    from ghmclip import _native
    seen = []
    value = lambda a: a.value if isinstance(a, ctypes._SimpleCData) else a  # noqa: E731
    monkeypatch.setattr(_native, "call", lambda name, *args: seen.append((name, [value(a) for a in args])))
    run()
    return seen


def _check(seen, buffers):
    """Every column sum's scratch lies in one of the buffers."""
    n = 0
    for name, a in seen:
        if name == "ghm_wcolsum":  # W, tok, C, X, rps, seq_rows, off, M, N, out, wsum, part
            part, need = a[11], _wcolsum_floats(a[7], a[8], a[2])
        elif name == "ghm_colsum":  # X, M, N, out, part
            part, need = a[4], _colsum_floats(a[1], a[2])
        else:
            continue
        n += 1
        home = [b for b in buffers if b.data_ptr() <= part < b.data_ptr() + 4 * b.numel()]
        assert home and part + 4 * need <= home[0].data_ptr() + 4 * home[0].numel(), (name, a)
    assert n


@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("B,D", [(128, 256), (4, 128), (77, 128), (126, 256)])
def test_vlm_backward_scratch(B, D, joint, monkeypatch):
    from ghmclip.models import vlm
    monkeypatch.setattr(vlm, "_stream", lambda: ctypes.c_void_p(0))
    T, P, V = (161, 81, 10) if joint else (81, 1, 10)
    model = vlm.AutoRegressiveTransformer(T, P, V, D, 1, [0, 0], 4, 4 * D, auto_regressive=True, sequential=not joint)
    plan = vlm.VlmPlan(1, T, B, n_prefix=P, num_class=V, n_embd=D, device="cpu", precision="x3", joint=joint)
    p = {n: x.detach() for n, x in model.named_parameters()}
    g = {n: torch.empty_like(x) for n, x in p.items()}
    plan._xt_fwd = plan.xt
    _check(_calls(monkeypatch, lambda: plan.backward(p, g)), [plan.colpart])
