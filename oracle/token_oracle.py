"""Token operators in 64 bits, from their definitions, with bounds on what
a 32-bit evaluation may be off (half a step of f32 is 2^-24 relative).

Bounds, u = 2^-24: with d = z - m a term e^d carries |d| 3u (difference, product with
log2 e and that constant's own rounding) + 2u (2^x to one step); a sum of positive terms
adds u for each term of the longest chain of additions that one lane makes, and a few for
the joins.  Each function returns the values and their absolute bounds side by side.
"""
import math

import torch

U = 2.0 ** -24
# the f32 exponential returns 0 below 2^-126: a probability is off by up to that much, and
# so is what is multiplied by it, times the factor (a row descending over 87 units: a factor
# of |log p + H| = 80 on a value of 1.2e-38)
FLUSH = 2.0 ** -126
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 0.0}
# half the smallest step near zero (subnormals; the f32 exponential flushes them)
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.float64: 0.0}


def round_bound(value, dtype):
    """One rounding of `value` to dtype."""
    return value.abs() * HALF[dtype] + TINY[dtype]


def _chain(V):
    """Longest chain of additions: a lane takes at least every 64th value of a long row,
    short rows are summed by one lane; plus the joins over lanes, waves and parts."""
    return min(V, 64 + V // 64) + 20


def _stats(z, c=1.0):
    """m, log sum exp((z - m) c), its bound, p, and E_p |d| c."""
    m = z.max(-1, keepdim=True).values
    d = (z - m) * c
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    p = e / s
    ed = torch.where(p > 0, p * d.abs(), 0.0).sum(-1, keepdim=True)
    ls = s.log()
    rel = U * (_chain(z.shape[-1]) + 2 + 6 * ed)  # of s; c != 1 adds its own two roundings to d
    return m, d, ls, rel + 2 * U * ls.abs(), p, ed


def top_ids(z, k):
    """ids by (value descending, id ascending), NaN first, -0 equal to +0."""
    key = torch.where(torch.isnan(z), math.inf, z + 0.0)
    nan = torch.isnan(z)
    # NaN above +inf: order by (is NaN, value) with a stable descending sort of each
    order = key.sort(dim=-1, descending=True, stable=True).indices
    again = nan.gather(-1, order).to(torch.int8).sort(dim=-1, descending=True, stable=True).indices
    return order.gather(-1, again)[..., :k]


def score(z, targets, top_k, ignore_index=-100):
    """z [n, V] float64, targets [n] or None."""
    n, V = z.shape
    m, d, ls, bls, p, ed = _stats(z)
    logp = d - ls
    blogp = bls + 2 * U * d.abs() + 2 * U * (d.abs() + ls.abs())
    finite_p = torch.where(p > 0, p * logp, torch.where(torch.isnan(p), p, 0.0))
    ent = -finite_p.sum(-1, keepdim=True)
    bent = bls + ed * (2 * bls + 8 * U * (1 + _chain(V))) + 4 * U * (ls.abs() + ed)
    live = torch.ones(n, 1, dtype=torch.bool, device=z.device) if targets is None else (targets != ignore_index)[:, None]
    out = {"logp": logp, "blogp": blogp, "p": p, "live": live}
    out["entropy"], out["bentropy"] = (torch.where(live, x, 0.0)[:, 0] for x in (ent, bent))
    if targets is not None:
        ok = (targets >= 0) & (targets < V)
        at = torch.where(ok, targets, 0)[:, None]
        lp = torch.where(ok[:, None], logp.gather(-1, at), math.nan)
        out["logprob"], out["blogprob"] = (torch.where(live, x, 0.0)[:, 0] for x in (lp, blogp.gather(-1, at)))
    ids = top_ids(z, top_k)
    out["top_logprob"], out["btop_logprob"] = (torch.where(live, x.gather(-1, ids), 0.0) for x in (logp, blogp))
    out["top_id"] = torch.where(live, ids, -1)
    return out


def score_grad(z, targets, r, g_lp=None, g_ent=None, g_top=None):
    """dz and its bound before the rounding to the logits' type."""
    n, V = z.shape
    zero = torch.zeros(n, dtype=z.dtype, device=z.device)
    g1 = zero if g_lp is None else g_lp
    g2 = (zero if g_ent is None else g_ent)[:, None]
    gs = g1[:, None] + (0 if g_top is None else g_top.sum(-1, keepdim=True))
    ag = g1.abs()[:, None] + (0 if g_top is None else g_top.abs().sum(-1, keepdim=True))
    p, logp, H = r["p"], r["logp"], r["entropy"][:, None]
    lp0 = torch.where(p > 0, logp, 0.0)
    inner = gs + g2 * (lp0 + H)
    dz = torch.where(torch.isnan(p), p, -p * inner)
    b0 = torch.where(p > 0, r["blogp"], 0.0)
    relp = b0 + 3 * U * lp0.abs() + 4 * U
    bound = p * (relp * inner.abs() + g2.abs() * (b0 + r["bentropy"][:, None] + 4 * U * (lp0.abs() + H.abs()))
                 + 70 * U * ag) + 2 * FLUSH * inner.abs()
    if g_lp is not None:
        ok = (targets >= 0) & (targets < V)
        at = torch.where(ok, targets, 0)[:, None]
        dz.scatter_add_(-1, at, g1[:, None])
        bound.scatter_add_(-1, at, 4 * U * g1.abs()[:, None])
        dz[(~ok) & r["live"][:, 0]] = math.nan
    if g_top is not None:
        dz.scatter_add_(-1, r["top_id"].clamp(min=0), g_top)
        bound.scatter_add_(-1, r["top_id"].clamp(min=0), 4 * U * g_top.abs())
    return torch.where(r["live"], dz, 0.0), torch.where(r["live"], bound, 0.0)


def distill(z, ids, t, targets, tau, alpha, ignore_index=-100):
    """Row losses, the gradient of their sum, counted rows, with bounds."""
    n, V = z.shape
    has = (ids >= 0) & ~torch.isneginf(t)
    some = has.any(-1, keepdim=True)
    tt = torch.where(has, t, -math.inf)
    mt = torch.where(some, tt.max(-1, keepdim=True).values, 0.0)
    dt = torch.where(has, (t - mt) / tau, -math.inf)
    et = torch.exp(dt)
    st = et.sum(-1, keepdim=True)
    q = torch.where(some, et / torch.where(some, st, 1.0), 0.0)
    k = ids.shape[-1]
    lq = torch.where(q > 0, torch.where(q > 0, q, 1.0).log(), 0.0)
    adt = torch.where(has & (q > 0), dt.abs(), 0.0)
    bst = U * (min(k, 64) + 22 + 6 * (q * adt).sum(-1, keepdim=True)) + 2 * U * torch.where(some, st, 1.0).log().abs()
    blq = bst + 6 * U * adt + 2 * U * lq.abs()
    bad = (has & (ids >= V)).any(-1, keepdim=True)
    at = ids.clamp(0, V - 1)
    m, d, l2, bl2, p, ed = _stats(z, 1.0 / tau)
    logp = d - l2
    blogp = bl2 + 6 * U * d.abs() + 2 * U * l2.abs()
    lpj, bj = logp.gather(-1, at), blogp.gather(-1, at)
    term = torch.where(q > 0, q * (lq - lpj), 0.0)
    bterm = torch.where(q > 0, q * (blq + bj + (blq + 6 * U + 3 * U * lq.abs()) * (lq - lpj).abs()
                                    + 2 * U * (lq.abs() + lpj.abs())), 0.0)
    kl, bkl = term.sum(-1), bterm.sum(-1) + U * (min(k, 64) + 22) * term.abs().sum(-1)
    a2 = alpha * tau * tau
    loss, bloss = a2 * kl, a2 * (bkl + 6 * U * kl.abs())
    relp = torch.where(p > 0, blogp + 3 * U * logp.abs() + 4 * U, 0.0)
    dz = torch.where(some, p, 0.0)
    bdz = torch.where(some, p * (relp + 6 * U) + 2 * FLUSH, 0.0)
    dz = dz.scatter_add(-1, at, -q)
    bdz = bdz.scatter_add(-1, at, q * (blq + 3 * U * lq.abs() + (10 + k) * U))
    dz, bdz = alpha * tau * dz, alpha * tau * (bdz + 8 * U * dz.abs())
    counted = some[:, 0]
    if targets is not None:
        counted = targets != ignore_index
        ok = (targets >= 0) & (targets < V)
        bad = bad | (~ok & counted)[:, None]
        y = torch.where(ok, targets, 0)[:, None]
        m, d, l1, bl1, p1, _ = _stats(z)
        logp1 = d - l1
        b1 = bl1 + 4 * U * (d.abs() + l1.abs())
        loss = loss - (1 - alpha) * logp1.gather(-1, y)[:, 0]
        bloss = bloss + (1 - alpha) * (b1.gather(-1, y)[:, 0] + 6 * U * logp1.gather(-1, y)[:, 0].abs())
        rel1 = torch.where(p1 > 0, b1 + 3 * U * logp1.abs() + 4 * U, 0.0)
        g1 = p1.scatter_add(-1, y, torch.full_like(y, -1, dtype=z.dtype))
        dz = dz + (1 - alpha) * g1
        bdz = bdz + (1 - alpha) * (p1 * (rel1 + 6 * U) + 6 * U * g1.abs() + 2 * FLUSH)
    bloss = bloss + 4 * U * loss.abs()
    dz = torch.where(bad, math.nan, dz)
    loss = torch.where(bad[:, 0], math.nan, loss)
    c = counted[:, None]
    return {"row_loss": torch.where(counted, loss, 0.0), "brow_loss": torch.where(counted, bloss, 0.0),
            "dz": torch.where(c, dz, 0.0), "bdz": torch.where(c, bdz + 6 * U * dz.abs(), 0.0), "counted": counted}


def embed(tokens, w, scale):
    """scale * w[tokens] (NaN rows for tokens outside the table) and its bound before the last rounding."""
    ok = (tokens >= 0) & (tokens < w.shape[0])
    out = torch.where(ok[:, None], w[torch.where(ok, tokens, 0)] * scale, math.nan)
    return out, U * out.abs()


def embed_grad(tokens, dout, scale, V, padding_idx=None):
    """sum over each token's rows: n terms make n - 1 roundings of at most the sum of magnitudes."""
    ok = (tokens >= 0) & (tokens < V)
    t = tokens[ok].long()
    dw = torch.zeros(V, dout.shape[1], dtype=dout.dtype).index_add_(0, t, dout[ok])
    mag = torch.zeros_like(dw).index_add_(0, t, dout[ok].abs())
    cnt = torch.bincount(t, minlength=V)[:, None]
    if padding_idx is not None:
        dw[padding_idx], mag[padding_idx] = 0, 0
    return dw * scale, mag * abs(scale) * U * (cnt + 1)
