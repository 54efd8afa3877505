"""Scratch of the column sums (csrc/ghm_gemm.hip colsum_plan / wcolsum_plan), beside it that of the split products and
of the LayerNorm gradients: what the *_part_elems functions
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


def _scratch(name, a):
    """(address, floats) of what a call writes to scratch."""
    if name == "ghm_wcolsum":  # W, tok, C, X, rps, seq_rows, off, M, N, out, wsum, part
        return [(a[11], _wcolsum_floats(a[7], a[8], a[2]))]
    if name == "ghm_colsum":  # X, M, N, out, part
        return [(a[4], _colsum_floats(a[1], a[2]))]
    if name in ("ghm_gemm_x3", "ghm_gemm_f32") and a[2] == 4:  # slabs, and the row sums of a ta = 1 product
        M, N, nsplit = a[16], a[17], a[19]
        return [(a[10], nsplit * M * N)] + ([(a[12], nsplit * M)] if a[12] else [])
    if name == "ghm_ln_rows_bwd":  # dY, X, stats, w, dres, dX, part, M, D
        return [(a[6], _lib().ghm_ln_rows_blocks(a[7]) * 2 * a[8])]
    return []


def _check(seen, plan):
    """Every call's scratch lies in one of the plan's buffers."""
    buffers = [b for b in vars(plan).values() if isinstance(b, torch.Tensor)]
    sums = 0
    for name, a in seen:
        sums += name in ("ghm_wcolsum", "ghm_colsum")
        for at, floats in _scratch(name, a):
            home = [b for b in buffers if b.data_ptr() <= at < b.data_ptr() + b.numel() * b.element_size()]
            assert home and all(at + 4 * floats <= b.data_ptr() + b.numel() * b.element_size() for b in home), (name, a)
    assert sums


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
    _check(_calls(monkeypatch, lambda: plan.backward(p, g)), plan)


def _encoder_shapes(T, D, V):
    s = {"token_embeddings.weight": (V, D), "position_embeddings.weight": (T, D), "_read_out.weight": (10, D),
         "_read_out.bias": (10,), "_out.weight": (1, T), "_out.bias": (1,), "_mlps.0.0.weight": (4 * D, D),
         "_mlps.0.0.bias": (4 * D,), "_mlps.0.2.weight": (D, 4 * D), "_mlps.0.2.bias": (D,)}
    s.update({f"_{k}.0.weight": (D, D) for k in ("queries", "keys", "values")})
    s.update({f"_lns_{i}.0.{w}": (D,) for i in (1, 2) for w in ("weight", "bias")})
    return s


@pytest.mark.parametrize("kind,N,T,D,V", [("gemm", 640, 81, 64, 10), ("gemm", 77, 27, 256, 10), ("gemm", 128, 81, 256, 10),
                                          ("encoder", 640, 81, 128, 16), ("encoder", 126, 81, 128, 16),
                                          ("cdm", 128, 162, 128, 10), ("cdm", 77, 162, 128, 10)])
def test_other_backward_scratch(kind, N, T, D, V, monkeypatch):
    from ghmclip.models import cdm, gemm_encoder, hip_encoder
    for m in (cdm, gemm_encoder, hip_encoder):
        monkeypatch.setattr(m, "_stream", lambda: ctypes.c_void_p(0))
    if kind == "gemm":
        plan = gemm_encoder.GemmEncoderPlan(1, T, N, num_class=10, vocab=V, n_embd=D, device="cpu")
        shapes = _encoder_shapes(T, D, V)
    elif kind == "encoder":
        plan = hip_encoder.EncoderPlan(1, T, N, num_class=10, vocab=V, n_embd=D, device="cpu", precision="x3")
        shapes = _encoder_shapes(T, D, V)
    else:
        plan = cdm.CdmPlan(1, T, 81, N, device="cpu", precision="x3", joint=True)
        shapes = {**_encoder_shapes(T, D, V), "t_embedding.weight": (V, D)}
    p, g = ({n: torch.empty(s) for n, s in shapes.items()} for _ in range(2))
    _check(_calls(monkeypatch, lambda: plan.backward(p, g)), plan)
