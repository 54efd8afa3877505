"""Token operators over a vocabulary of any size (csrc/ghm_score.hip, ghm_distill.hip, ghm_embed.hip): scores of
given tokens, distillation from a teacher's top logits, scaled embedding.

They stand beside the fixed-vocabulary kernels of the VLM (``ghm_ce_kl``,
``ghm_tok_embed_fwd``, ``ghm_wcolsum``: 8-bit tokens, f32, at most 64 values) and
have no counterpart in the reference.  Logits, tables and gradients are float32,
bfloat16 or float16 on a HIP device; sums, statistics and losses are float32.  Work
is issued on the current stream of the tensors' device; nothing synchronises, so
token ids are not checked on the host: an id outside the vocabulary gives NaN in
what depends on it in its own row (and adds nothing to an embedding gradient).  Gradients are of first order and
reverse mode; a second one and forward-mode tangents raise.
"""
from collections import namedtuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from .. import _native
from .hip_encoder import require_hip

__all__ = ["TokenScores", "token_logprobs", "distill_loss", "distill_loss_and_grad", "TopLogitsDistillLoss",
           "scaled_embedding", "ScaledEmbedding"]

GHM_TOP_MAX = 64  # include/ghm_hip.h
GHM_DISTILL_MAX = 1024  # include/ghm_hip.h

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ID_BITS = {torch.uint8: 8, torch.int32: 32, torch.int64: 64}
_REDUCTION = {"none": 0, "mean": 1, "sum": 2}

TokenScores = namedtuple("TokenScores", "logprob entropy top_logprob top_id")


def _dtype(t, what):
    try:
        return _DTYPE[t.dtype]
    except KeyError:
        raise TypeError(f"{what}: float32, bfloat16 or float16, got {t.dtype}") from None


def _ids(t, shape, device, what, bits=(8, 32, 64)):
    """Checked token ids, contiguous: (tensor, bits)."""
    if not isinstance(t, torch.Tensor) or _ID_BITS.get(t.dtype) not in bits:
        raise TypeError(f"{what}: an integer tensor of {' / '.join(map(str, bits))} bits "
                        f"(uint8, int32, int64), got {getattr(t, 'dtype', type(t))}")
    if t.shape != shape:
        raise ValueError(f"{what}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what}: on {t.device}, expected {device}")
    return t.contiguous(), _ID_BITS[t.dtype]


def _rows(t):
    """(tensor, n_inner, s_outer, s_inner) of the rows of ``t`` [..., V]; copied only
    if its values are not consecutive or its leading dimensions need more than two strides."""
    V = t.shape[-1]
    if t.is_contiguous():
        return t, max(1, t.numel() // V), 0, V
    if V == 1 or t.stride(-1) == 1:
        dims = []  # (size, stride), neighbours that form one stride merged
        for n, st in zip(t.shape[:-1], t.stride()[:-1]):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * st:
                dims[-1] = (dims[-1][0] * n, st)
            else:
                dims.append((n, st))
        if not dims:
            return t, 1, 0, V
        if len(dims) == 1:
            return t, dims[0][0], 0, dims[0][1]
        if len(dims) == 2:
            return t, dims[1][0], dims[0][1], dims[1][1]
    t = t.contiguous()
    return t, max(1, t.numel() // V), 0, V


def _ptr(t):
    return None if t is None else t.data_ptr()


# the handle of a device's current stream without a torch.cuda.Stream object around it
# (2 us of a 15 us call, 9 us on autograd's thread)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, name, *args):
    """Call an entry point on the device's current stream."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _native.call(name, *args, _raw_stream(device.index))
    return _native.call(name, *args, _raw_stream(device.index))


def _check_tangent(t, what):
    """Forward-mode tangents are refused: a dual tensor without requires_grad takes the calls past
    autograd, whose results would carry none (derivative 0).  Asked only while a level of
    forward-mode differentiation is open (0.1 us a call in place of 0.9)."""
    if getattr(forward_ad, "_current_level", 0) < 0:
        return
    if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what}: forward-mode derivatives are not offered")


def _check_logits(logits):
    _check_tangent(logits, "logits")
    require_hip(logits)
    code = _dtype(logits, "logits")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits: expected [..., V] with V >= 1, got {tuple(logits.shape)}")
    return code


def _first_order(backward):
    """A backward that is not itself differentiable: torch's wrapper refuses a second
    gradient; it is only entered where a graph of the backward is built (4 us a call)."""
    refusing = torch.autograd.function.once_differentiable(backward)

    def either(ctx, *grads):
        return (refusing if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(either)


# ---- scores ---------------------------------------------------------------


def _score(logits, y, bits, top_k, ignore_index, want_stats):
    code, dev, lead, V = _DTYPE[logits.dtype], logits.device, logits.shape[:-1], logits.shape[-1]
    z, n_inner, so, si = _rows(logits)
    rows = logits.numel() // V
    logprob = None if y is None else torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=dev) if want_stats else None
    top_lp = torch.empty((*lead, top_k), dtype=torch.float32, device=dev) if top_k else None
    top_id = torch.empty((*lead, top_k), dtype=torch.int64, device=dev) if top_k else None
    nws = _native.hip_lib().ghm_token_logprobs_ws(rows, V, top_k, code)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
    _call(dev, "ghm_token_logprobs", z.data_ptr(), code, n_inner, so, si, rows, V, _ptr(y), bits, ignore_index, top_k,
          _ptr(logprob), entropy.data_ptr(), _ptr(stats), _ptr(top_lp), _ptr(top_id), _ptr(ws), nws)
    return logprob, entropy, top_lp, top_id, stats


class _ScoreFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, y, bits, top_k, ignore_index):
        logprob, entropy, top_lp, top_id, stats = _score(logits, y, bits, top_k, ignore_index, True)
        ctx.set_materialize_grads(False)
        ctx.args = bits, top_k, ignore_index
        ctx.save_for_backward(logits, y, entropy, top_id, stats)
        if top_id is not None:
            ctx.mark_non_differentiable(top_id)
        return logprob, entropy, top_lp, top_id

    @_first_order
    def backward(ctx, g_lp, g_ent, g_top, _g_id):
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None, None, None
        logits, y, entropy, top_id, stats = ctx.saved_tensors
        bits, top_k, ignore_index = ctx.args
        dev, V = logits.device, logits.shape[-1]
        z, n_inner, so, si = _rows(logits)
        g_lp, g_ent, g_top = (None if g is None else g.contiguous() for g in (g_lp, g_ent, g_top))
        dz = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        _call(dev, "ghm_token_logprobs_bwd", z.data_ptr(), _DTYPE[logits.dtype], n_inner, so, si, logits.numel() // V,
              V, _ptr(y), bits, ignore_index, top_k, _ptr(top_id), stats.data_ptr(), entropy.data_ptr(), _ptr(g_lp),
              _ptr(g_ent), _ptr(g_top), dz.data_ptr())
        return dz, None, None, None, None


def token_logprobs(logits, targets=None, top_k=0, ignore_index=-100):
    """Log probabilities of given tokens under softmax(logits), with the entropy of each
    row and its ``top_k`` most likely values, from one pass over the logits.

    logits [..., V]; targets [...] (uint8 / int32 / int64) or None.  Returns
    TokenScores(logprob [...], entropy [...], top_logprob [..., top_k], top_id
    [..., top_k] int64): float32; logprob is None without targets, the last two with
    top_k = 0.  Alternatives descend; equal values rank by ascending id, NaN first.
    logprob, entropy and top_logprob are differentiable in the logits.

    A row whose target is ``ignore_index`` is padding: not read, 0 (top_id -1), gradient
    0.  A logit of -inf has probability 0; a row without a finite maximum is NaN.  A target
    outside 0 .. V - 1 makes its row's logprob NaN, and a gradient through it; entropy and
    alternatives do not depend on it.  top_k <= min(64, V)."""
    _check_logits(logits)
    if not isinstance(top_k, int) or not 0 <= top_k <= min(GHM_TOP_MAX, logits.shape[-1]):
        raise ValueError(f"top_k: 0 .. min({GHM_TOP_MAX}, V = {logits.shape[-1]}), got {top_k!r}")
    y, bits = (None, 64) if targets is None else _ids(targets, logits.shape[:-1], logits.device, "targets")
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenScores(*_ScoreFn.apply(logits, y, bits, top_k, ignore_index))
    return TokenScores(*_score(logits, y, bits, top_k, ignore_index, False)[:4])


# ---- distillation ---------------------------------------------------------


def _distill_check(logits, top_ids, top_logits, targets, temperature, alpha):
    """Checked arguments: (logits, ids, t, y) and (id bits, target bits, temperature, alpha)."""
    _check_logits(logits)
    dev, lead = logits.device, logits.shape[:-1]
    k = top_ids.shape[-1] if isinstance(top_ids, torch.Tensor) and top_ids.dim() else 0
    if not 1 <= k <= GHM_DISTILL_MAX:
        raise ValueError(f"top_ids: expected [..., k] with k in 1 .. {GHM_DISTILL_MAX}")
    ids, ibits = _ids(top_ids, (*lead, k), dev, "top_ids", bits=(32, 64))
    if not isinstance(top_logits, torch.Tensor) or top_logits.shape != ids.shape or top_logits.device != dev:
        raise ValueError(f"top_logits: expected shape {tuple(ids.shape)} on {dev}")
    _dtype(top_logits, "top_logits")
    y, ybits = (None, 64) if targets is None else _ids(targets, lead, dev, "targets")
    temperature, alpha = float(temperature), float(alpha)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature: 1e-6 .. 1e6, got {temperature}")
    if not 0 <= alpha <= 1 or (alpha < 1 and targets is None):
        raise ValueError(f"alpha: 0 .. 1, below 1 only with targets, got {alpha}")
    return (logits, ids, top_logits.detach().contiguous(), y), (ibits, ybits, temperature, alpha)


def _distill_args(tensors, opts, ignore_index):
    """The arguments of ghm_distill / ghm_distill_bwd up to alpha, and the logits they point to."""
    logits, ids, t, y = tensors
    ibits, ybits, temperature, alpha = opts
    V = logits.shape[-1]
    z, n_inner, so, si = _rows(logits)
    return (z.data_ptr(), _DTYPE[logits.dtype], n_inner, so, si, logits.numel() // V, V, ids.data_ptr(), ibits,
            t.data_ptr(), _DTYPE[t.dtype], ids.shape[-1], _ptr(y), ybits, ignore_index, temperature, alpha), z


def _distill(logits, args, reduction, grad_scale=None):
    """(loss, stats, norm, dlogits or None) of ghm_distill: the statistics, the norm, the
    row losses of a reduced loss and the workspace share one buffer."""
    dev, code, rows, V = logits.device, args[1], args[5], args[6]
    dz = None if grad_scale is None else torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    loss = torch.empty(logits.shape[:-1] if reduction == "none" else (), dtype=torch.float32, device=dev)
    nws = _native.hip_lib().ghm_distill_ws(rows, V, code)
    r4 = rows + (-rows) % 4
    buf = torch.empty(4 * rows + 4 + r4 + nws // 4 + 4, dtype=torch.float32, device=dev)
    at = buf.data_ptr()  # stats, norm, row losses, workspace; each at a multiple of 16 bytes
    row_loss = loss.data_ptr() if reduction == "none" else at + 16 * (rows + 1)
    _call(dev, "ghm_distill", *args, _REDUCTION[reduction], loss.data_ptr(), row_loss, at, at + 16 * rows,
          1.0 if grad_scale is None else grad_scale, _ptr(dz), at + 16 * (rows + 1) + 4 * r4, nws)
    return loss, buf, at + 16 * rows, dz


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, t, y, opts, ignore_index, reduction):
        args, _z = _distill_args((logits, ids, t, y), opts, ignore_index)
        loss, buf, _, _ = _distill(logits, args, reduction)
        ctx.args = opts, ignore_index, reduction
        ctx.save_for_backward(logits, ids, t, y, buf)
        return loss

    @_first_order
    def backward(ctx, g):
        logits, ids, t, y, buf = ctx.saved_tensors
        opts, ignore_index, reduction = ctx.args
        args, _z = _distill_args((logits, ids, t, y), opts, ignore_index)
        g = g.contiguous()
        dz = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        at = buf.data_ptr()
        _call(logits.device, "ghm_distill_bwd", *args, at, at + 16 * args[5] if reduction == "mean" else None,
              g.data_ptr(), int(reduction == "none"), dz.data_ptr())
        return dz, None, None, None, None, None, None


def _check_reduction(reduction):
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction: {', '.join(_REDUCTION)}, got {reduction!r}")


def distill_loss(logits, top_ids, top_logits, targets=None, *, temperature=1.0, alpha=1.0, ignore_index=-100,
                 reduction="mean"):
    """Distillation from a teacher's top logits, differentiable in the student's logits:

        (1 - alpha) CE(logits, targets) + alpha temperature^2 KL(q || softmax(logits / temperature))

    with q = softmax(top_logits / temperature) over the entries a row holds.  logits
    [..., V]; top_ids [..., k] (int32 / int64) and top_logits [..., k]: the teacher's
    alternatives, k <= 1024 (log probabilities, as token_logprobs returns them, serve as
    well); a negative id or a logit of -inf marks an absent entry, repeated ids add up.
    targets [...]: hard labels, needed for alpha < 1; alpha = 0 leaves the teacher's logits out.

    reduction "mean": over the counted rows (0 if there is none) -- those whose target is
    not ``ignore_index``, or without targets those with an entry --; "sum"; "none": one
    float32 loss per row.  Rows that do not count have loss and gradient 0.  An id at or
    above V, or a target outside 0 .. V - 1, makes its row NaN.  The teacher's logits get no
    gradient."""
    _check_reduction(reduction)
    tensors, opts = _distill_check(logits, top_ids, top_logits, targets, temperature, alpha)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillFn.apply(*tensors, opts, ignore_index, reduction)
    args, _z = _distill_args(tensors, opts, ignore_index)
    return _distill(logits, args, reduction)[0]


def distill_loss_and_grad(logits, top_ids, top_logits, targets=None, *, temperature=1.0, alpha=1.0,
                          ignore_index=-100, reduction="mean", grad_scale=1.0):
    """``distill_loss`` and ``grad_scale`` times its gradient in the logits (reduction
    "none": the gradient of the sum) from one call, outside autograd, as the fused
    trainers take their losses: (loss, dlogits)."""
    _check_reduction(reduction)
    tensors, opts = _distill_check(logits, top_ids, top_logits, targets, temperature, alpha)
    args, _z = _distill_args(tensors, opts, ignore_index)
    loss, _, _, dz = _distill(logits, args, reduction, float(grad_scale))
    return loss, dz


class TopLogitsDistillLoss(nn.Module):
    """``distill_loss`` as a module (beside KLdiv and ConditionalGuidedCELoss):
    forward(logits, top_ids, top_logits, targets=None)."""

    def __init__(self, temperature=1.0, alpha=1.0, ignore_index=-100, reduction="mean"):
        super().__init__()
        _check_reduction(reduction)
        self.temperature, self.alpha = temperature, alpha
        self.ignore_index, self.reduction = ignore_index, reduction

    def forward(self, logits, top_ids, top_logits, targets=None):
        return distill_loss(logits, top_ids, top_logits, targets, temperature=self.temperature, alpha=self.alpha,
                            ignore_index=self.ignore_index, reduction=self.reduction)


# ---- embedding ------------------------------------------------------------


def _embed(tok, bits, weight, scale):
    V, D = weight.shape
    w = weight if D == 1 or weight.stride(1) == 1 else weight.contiguous()
    out = torch.empty((*tok.shape, D), dtype=weight.dtype, device=weight.device)
    _call(weight.device, "ghm_embed_rows_fwd", tok.data_ptr(), bits, w.data_ptr(), _DTYPE[weight.dtype], w.stride(0),
          scale, out.data_ptr(), tok.numel(), V, D)
    return out


class _EmbedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, tok, bits, scale, padding_idx):
        ctx.save_for_backward(tok)
        ctx.args = bits, scale, padding_idx, weight.shape
        return _embed(tok, bits, weight, scale)

    @_first_order
    def backward(ctx, g):
        tok, = ctx.saved_tensors
        bits, scale, padding_idx, (V, D) = ctx.args
        N, dev = tok.numel(), g.device
        if g.is_contiguous():
            stride = D
        else:
            g, n_inner, _, stride = _rows(g)
            if n_inner != max(1, N):  # rows of two strides
                g, stride = g.contiguous(), D
        dw = torch.empty((V, D), dtype=g.dtype, device=dev)
        nws = _native.hip_lib().ghm_embed_rows_bwd_ws(N, V, D)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        _call(dev, "ghm_embed_rows_bwd", tok.data_ptr(), bits, g.data_ptr(), _DTYPE[g.dtype], stride, scale, padding_idx,
              dw.data_ptr(), N, V, D, ws.data_ptr(), nws)
        return dw, None, None, None, None


def scaled_embedding(tokens, weight, scale=1.0, padding_idx=None):
    """scale * weight[tokens]: tokens [...] (uint8 / int32 / int64), weight [V, D] ->
    [..., D] in weight's dtype.  Differentiable in weight: the gradient sums the rows of
    each token in float32, in the order they appear (sorted tokens, no atomics: the same
    bits every run), and rounds once; row ``padding_idx`` gets none.  A token outside
    0 .. V - 1 gives a NaN row and adds nothing to the gradient."""
    _check_tangent(weight, "weight")
    require_hip(weight)
    _dtype(weight, "weight")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight: expected [V, D], got {tuple(weight.shape)}")
    tok, bits = _ids(tokens, getattr(tokens, "shape", None), weight.device, "tokens")
    V = weight.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif not -V <= padding_idx < V:
        raise ValueError(f"padding_idx: -{V} .. {V - 1}, got {padding_idx}")
    elif padding_idx < 0:
        padding_idx += V
    if torch.is_grad_enabled() and weight.requires_grad:
        return _EmbedFn.apply(weight, tok, bits, float(scale), padding_idx)
    return _embed(tok, bits, weight, float(scale))


class ScaledEmbedding(nn.Embedding):
    """nn.Embedding whose rows are multiplied by ``scale`` (default 1), on
    ``scaled_embedding``: same parameter, initialisation and padding_idx.  max_norm,
    scale_grad_by_freq and sparse are not offered."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)

    def forward(self, tokens):
        return scaled_embedding(tokens, self.weight, self.scale, self.padding_idx)
