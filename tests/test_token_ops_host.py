"""CPU tests of the token operators' host side: what the C entry points and the Python
wrappers refuse (checked before anything touches a device), the row addressing of
strided logits, and the oracle of the GPU tests against autograd in 64 bits."""
import ctypes
import math

import pytest
import torch

from oracle import token_oracle as O


def _lib():
    from ghmclip import _native
    return _native.hip_lib()


P = ctypes.c_void_p(4096)  # stands for a device buffer; refused calls never read it


def _score(**kw):
    a = dict(logits=P, dtype=0, n_inner=4, so=0, si=10, rows=4, V=10, targets=P, bits=64, ignore=-100, top_k=2,
             logprob=P, entropy=P, stats=None, top_lp=P, top_id=P, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib().ghm_token_logprobs(*a.values())


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(V=0), dict(V=(1 << 30) + 1), dict(rows=-1),
                                dict(rows=1 << 31), dict(n_inner=0), dict(so=-1), dict(si=-1), dict(top_k=-1),
                                dict(top_k=65, V=100), dict(top_k=11), dict(bits=16), dict(logits=None),
                                dict(logprob=None), dict(targets=None), dict(top_lp=None), dict(top_id=None),
                                dict(ws_bytes=-1)])
def test_score_refusals(kw):
    assert _score(**kw) == -22
    assert _lib().ghm_last_error_string()


def test_score_nothing_to_do():
    assert _score(rows=0, logits=None) == 0


def _score_bwd(**kw):
    a = dict(logits=P, dtype=0, n_inner=4, so=0, si=10, rows=4, V=10, targets=P, bits=64, ignore=-100, top_k=2,
             top_id=P, stats=P, entropy=P, g_lp=P, g_ent=P, g_top=P, dz=P, stream=None)
    a.update(kw)
    return _lib().ghm_token_logprobs_bwd(*a.values())


@pytest.mark.parametrize("kw", [dict(dtype=7), dict(V=-3), dict(stats=None), dict(dz=None), dict(targets=None),
                                dict(entropy=None), dict(top_id=None), dict(top_k=0), dict(bits=1)])
def test_score_bwd_refusals(kw):
    assert _score_bwd(**kw) == -22


def _distill(**kw):
    a = dict(logits=P, dtype=0, n_inner=4, so=0, si=10, rows=4, V=10, ids=P, ibits=64, t=P, tdtype=0, k=3, y=P,
             ybits=64, ignore=-100, tau=1.0, alpha=0.5, reduction=1, loss=P, row_loss=P, stats=P, norm=P, gs=1.0,
             dz=P, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib().ghm_distill(*a.values())


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(ibits=8), dict(tdtype=5), dict(k=0), dict(k=1025), dict(tau=0.0),
                                dict(tau=-1.0), dict(tau=math.inf), dict(tau=math.nan), dict(tau=1e-7), dict(tau=1e7), dict(alpha=1.5),
                                dict(alpha=math.nan), dict(alpha=0.5, y=None), dict(reduction=3), dict(loss=None),
                                dict(norm=None), dict(row_loss=None), dict(stats=None), dict(logits=None),
                                dict(ids=None), dict(t=None), dict(ybits=3), dict(ws_bytes=-1)])
def test_distill_refusals(kw):
    assert _distill(**kw) == -22


def _distill_bwd(**kw):
    a = dict(logits=P, dtype=0, n_inner=4, so=0, si=10, rows=4, V=10, ids=P, ibits=64, t=P, tdtype=0, k=3, y=P,
             ybits=64, ignore=-100, tau=1.0, alpha=0.5, stats=P, norm=P, g=P, g_rows=0, dz=P, stream=None)
    a.update(kw)
    return _lib().ghm_distill_bwd(*a.values())


@pytest.mark.parametrize("kw", [dict(stats=None), dict(g=None), dict(dz=None), dict(tau=0.0), dict(k=0)])
def test_distill_bwd_refusals(kw):
    assert _distill_bwd(**kw) == -22


def test_distill_of_no_rows_takes_null_targets():
    """An empty batch's buffers are null, its targets among them."""
    none = dict(rows=0, logits=None, ids=None, t=None, y=None, dz=None, alpha=0.5)
    assert _distill(**none, row_loss=None, reduction=0) != -22  # (no device here to ask for a launch error)
    assert _distill_bwd(**none, g=None) == 0


def _embed(**kw):
    a = dict(tok=P, bits=64, w=P, dtype=0, ws=8, scale=1.0, out=P, N=4, V=10, D=8, stream=None)
    a.update(kw)
    return _lib().ghm_embed_rows_fwd(*a.values())


def _embed_bwd(**kw):
    a = dict(tok=P, bits=64, g=P, dtype=0, gs=8, scale=1.0, pad=-1, dw=P, N=4, V=10, D=8, ws=P, ws_bytes=1 << 40,
             stream=None)
    a.update(kw)
    return _lib().ghm_embed_rows_bwd(*a.values())


@pytest.mark.parametrize("kw", [dict(bits=9), dict(dtype=3), dict(V=0), dict(V=1 << 31), dict(D=0), dict(D=(1 << 20) + 1),
                                dict(N=-1), dict(N=1 << 31), dict(tok=None)])
def test_embed_refusals(kw):
    assert _embed(**kw) == -22
    assert _embed_bwd(**kw) == -22


@pytest.mark.parametrize("kw", [dict(pad=10), dict(pad=-2), dict(dw=None), dict(gs=-1), dict(ws_bytes=-1)])
def test_embed_bwd_refusals(kw):
    assert _embed_bwd(**kw) == -22


def test_wrappers_refuse_cpu_tensors():
    from ghmclip import models as M
    z = torch.zeros(2, 5)
    with pytest.raises(RuntimeError, match="HIP device"):
        M.token_logprobs(z, torch.zeros(2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="HIP device"):
        M.distill_loss(z, torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1))
    with pytest.raises(RuntimeError, match="HIP device"):
        M.scaled_embedding(torch.zeros(2, dtype=torch.long), z)
    with pytest.raises(ValueError, match="reduction"):
        M.TopLogitsDistillLoss(reduction="median")


def test_forward_mode_derivatives_are_refused():
    """A dual tensor needs no gradient, and a result without a tangent reads as derivative 0."""
    import torch.autograd.forward_ad as fwAD
    from ghmclip import models as M
    z, ids, t = torch.zeros(2, 5), torch.zeros(2, 1, dtype=torch.long), torch.zeros(2, 1)
    with fwAD.dual_level():
        dual = fwAD.make_dual(z, torch.ones_like(z))
        for f in (lambda: M.token_logprobs(dual), lambda: M.distill_loss(dual, ids, t),
                  lambda: M.distill_loss_and_grad(dual, ids, t), lambda: M.TopLogitsDistillLoss()(dual, ids, t),
                  lambda: M.scaled_embedding(ids, dual)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_limits_match_the_header():
    import os
    import re

    from conftest import ROOT
    from ghmclip.models import token_ops as T
    src = open(os.path.join(ROOT, "include", "ghm_hip.h")).read()
    for name in ("GHM_TOP_MAX", "GHM_DISTILL_MAX"):
        assert getattr(T, name) == int(re.search(rf"#define {name} (\d+)", src).group(1))


@pytest.mark.parametrize("make,copied", [
    (lambda x: x, False), (lambda x: x[:, 1:], False), (lambda x: x[::2], False), (lambda x: x[1:2, 2:5], False),
    (lambda x: x[..., 1:], False), (lambda x: x[:, :, :1].expand(-1, -1, 4), True),
    (lambda x: x[:1].expand(3, -1, -1), False), (lambda x: x.transpose(1, 2), True), (lambda x: x[0, 0], False),
    (lambda x: x.view(2, 2, 6, 7)[:, :, 1:], False), (lambda x: x.view(2, 2, 6, 7)[:, :1, 1:], False),
    (lambda x: x.view(4, 2, 3, 7)[:, :1, 1:], False), (lambda x: x.view(2, 2, 2, 3, 7)[:, 1:, :, 1:], True),
    (lambda x: x[:, :, :1], False), (lambda x: x[:0], False)])
def test_row_addressing(make, copied):
    """Element (r / n_inner) * s_outer + (r % n_inner) * s_inner is where row r starts."""
    from ghmclip.models.token_ops import _rows
    t = make(torch.arange(4 * 6 * 7, dtype=torch.float32).view(4, 6, 7))
    V = t.shape[-1]
    u, n_inner, so, si = _rows(t)
    assert (u is not t) == copied
    flat = torch.as_strided(u, (u.storage_offset() * 0 + u.untyped_storage().nbytes() // 4,), (1,), 0)
    want = t.reshape(-1, V)
    for r in range(want.shape[0]):
        at = u.storage_offset() + (r // n_inner) * so + (r % n_inner) * si
        assert torch.equal(flat[at:at + V], want[r])


# ---- the oracle itself ----------------------------------------------------


def test_oracle_score_gradient_is_autograds():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(5, 9, generator=g, dtype=torch.float64, requires_grad=True)
    y = torch.tensor([0, 8, 3, -100, 2])
    r = O.score(z.detach(), y, 3)
    logp = torch.log_softmax(z, -1)
    live = y != -100
    lp = torch.where(live, logp.gather(-1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    ent = torch.where(live, -(logp.exp() * logp).sum(-1), 0.0)
    top = torch.where(live[:, None], logp.gather(-1, r["top_id"].clamp(min=0)), 0.0)
    assert torch.allclose(r["logprob"], lp.detach(), atol=1e-14) and torch.allclose(r["entropy"], ent.detach(), atol=1e-14)
    g1, g2, g3 = torch.randn(5, generator=g).double(), torch.randn(5, generator=g).double(), torch.randn(5, 3, generator=g).double()
    want, = torch.autograd.grad((lp * g1).sum() + (ent * g2).sum() + (top * g3).sum(), z)
    got, _ = O.score_grad(z.detach(), y, r, g1, g2, g3)
    assert torch.allclose(got, want, atol=1e-13)


def test_oracle_alternatives_break_ties_by_id():
    z = torch.tensor([[1.0, 3.0, 3.0, -0.0, 0.0, 3.0], [float("nan"), 1.0, 1.0, float("inf"), 0.0, -1.0]])
    r = O.score(z.double(), None, 5)
    assert r["top_id"].tolist() == [[1, 2, 5, 0, 3], [0, 3, 1, 2, 4]]


@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.3), (0.5, 0.0)])
def test_oracle_distill_gradient_is_autograds(tau, alpha):
    g = torch.Generator().manual_seed(1)
    z = torch.randn(4, 7, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 3, 3], [6, -1, 2], [-1, -1, -1], [1, 2, 4]])
    t = torch.randn(4, 3, generator=g, dtype=torch.float64)
    t[3, 1] = -math.inf
    y = torch.tensor([2, 5, 1, -100])
    r = O.distill(z.detach(), ids, t, y if alpha < 1 else None, tau, alpha)
    has = (ids >= 0) & ~torch.isneginf(t)
    q = torch.where(has, torch.exp(t / tau), 0.0)
    q = q / q.sum(-1, keepdim=True).clamp(min=1e-30)
    kl = (torch.special.xlogy(q, q) - q * torch.log_softmax(z / tau, -1).gather(-1, ids.clamp(min=0))).sum(-1)
    row = alpha * tau * tau * kl
    if alpha < 1:
        row = row + (1 - alpha) * torch.nn.functional.cross_entropy(z, y, reduction="none", ignore_index=-100)
        row = torch.where(y != -100, row, 0.0)
    assert torch.allclose(r["row_loss"], row.detach(), atol=1e-13)
    want, = torch.autograd.grad(row.sum(), z)
    assert torch.allclose(r["dz"], want, atol=1e-13)
    assert int(r["counted"].sum()) == 3
