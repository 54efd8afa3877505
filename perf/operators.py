"""Cases that time the token operators: scoring (token_logprobs), distillation from a
teacher's top logits (distill_loss, distill_loss_and_grad) and the scaled embedding
with its gradient by sorted tokens (scaled_embedding).

``own`` False computes each operator in elementary torch operations in 32 bits,
True through ghmclip's public entry points.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
ROWS_V = 4096 * 131072  # the largest rows x vocabulary of a case


def listed():
    return [
        # the repository's sequential VLM batch (128 sequences, 1 prefix + 80 text tokens, 10 token
        # values): training-time scores of every position, logits read past the prefix row
        {"name": "score_vlm", "op": "score", "rows": 128 * 80, "T": 80, "prefix": 1, "V": 10, "dtype": "f32",
         "top": 3, "grad": False, "masked": False},
        # one decoding step of four sequences over a large vocabulary: latency counts
        {"name": "score_decode", "op": "score", "rows": 4, "T": 1, "prefix": 0, "V": 131072, "dtype": "bf16",
         "top": 20, "grad": False, "masked": True},
        # scoring long prompts: every position, the teacher's alternatives kept for distillation
        {"name": "score_prompt", "op": "score", "rows": 4096, "T": 2048, "prefix": 0, "V": 131072, "dtype": "bf16",
         "top": 32, "grad": False, "masked": False},
        # a policy-gradient step: log probabilities and entropy with their gradient, odd vocabulary
        {"name": "score_policy", "op": "score", "rows": 2000, "T": 500, "prefix": 0, "V": 50001, "dtype": "f32",
         "top": 0, "grad": True, "masked": False},
        # the VLM batch distilled from a teacher's 4 best of 10 values, with hard labels
        {"name": "distill_vlm", "op": "distill", "call": "step", "rows": 128 * 80, "T": 80, "prefix": 1, "V": 10,
         "dtype": "f32", "k": 4, "tau": 2.0, "alpha": 0.5, "hard": True},
        # a large student step from stored alternatives: loss and gradient in one call
        {"name": "distill_large", "op": "distill", "call": "step", "rows": 4096, "T": 2048, "prefix": 0, "V": 131072,
         "dtype": "bf16", "k": 64, "tau": 1.0, "alpha": 1.0, "hard": False},
        # through autograd, temperature and hard labels mixed, odd vocabulary, ragged alternatives
        {"name": "distill_mixed", "op": "distill", "call": "autograd", "rows": 1023, "T": 341, "prefix": 0,
         "V": 32001, "dtype": "f32", "k": 32, "tau": 2.0, "alpha": 0.7, "hard": True},
        # a small validation batch: the loss alone
        {"name": "distill_eval", "op": "distill", "call": "eval", "rows": 24, "T": 24, "prefix": 0, "V": 65536,
         "dtype": "f16", "k": 16, "tau": 1.5, "alpha": 1.0, "hard": False},
        # the input rows of one decoding step of eight sequences
        {"name": "embed_decode", "op": "embed", "N": 8, "V": 131072, "D": 4096, "dtype": "bf16", "grad": False,
         "padding": False},
        # the VLM batch's 81-token rows through a 256-wide table of 10 values, forward and backward
        {"name": "embed_vlm", "op": "embed", "N": 128 * 81, "V": 10, "D": 256, "dtype": "f32", "grad": True,
         "padding": False},
        # a pre-training step's table: frequent and rare tokens, padding among them
        {"name": "embed_step", "op": "embed", "N": 16384, "V": 65536, "D": 2048, "dtype": "bf16", "grad": True,
         "padding": True},
        # a long batch over a small odd table and an odd width
        {"name": "embed_long", "op": "embed", "N": 131071, "V": 5003, "D": 1001, "dtype": "f32", "grad": True,
         "padding": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["score", "distill", "embed"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "embed":
        V, D = _log_int(rng, 10, 131072), _log_int(rng, 32, 4096)
        # gradient tables of at most the largest listed case's size
        if V * D * SIZE[dtype] > 1 << 29:
            V = (1 << 29) // (D * SIZE[dtype])
        N = _log_int(rng, 1, min(131072, (1 << 29) // (D * SIZE[dtype])))
        return {"op": "embed", "N": N, "V": V, "D": D, "dtype": dtype, "grad": rng.random() < 0.7,
                "padding": rng.random() < 0.3}
    V = _log_int(rng, 10, 131072)
    T = _log_int(rng, 1, 512)
    rows = T * _log_int(rng, 1, max(1, min(16384 // T, ROWS_V * 2 // (V * T * SIZE[dtype]))))
    c = {"op": op, "rows": rows, "T": T, "prefix": rng.choice([0, 0, 1]), "V": V, "dtype": dtype}
    if op == "score":
        grad = rng.random() < 0.5
        return {**c, "top": 0 if grad else min(V, _log_int(rng, 1, 64)), "grad": grad, "masked": rng.random() < 0.3}
    hard = rng.random() < 0.5
    return {**c, "call": rng.choice(["step", "step", "autograd", "eval"]), "k": min(V, _log_int(rng, 1, 64)),
            "tau": rng.choice([1.0, 1.5, 2.0, 4.0]), "alpha": rng.choice([0.3, 0.5, 0.9]) if hard else 1.0,
            "hard": hard}


# ---- inputs ---------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(case, g):
    """Model outputs [sequences, T, V], a view past `prefix` leading positions; a few
    likely values stand out of each row."""
    n, T, P, V = case["rows"] // case["T"], case["T"], case["prefix"], case["V"]
    z = torch.empty(n, T + P, V, dtype=DTYPES[case["dtype"]], device="cuda").normal_(0, 2, generator=g)
    likely = torch.randint(0, V, (n, T + P, 1), device="cuda", generator=g)
    z.scatter_(2, likely, z.gather(2, likely) + 8)
    return z[:, P:, :], likely[:, P:, 0]


def _zipf(n, V, g):
    """Token ids whose frequency falls with their rank, ranks spread over the table."""
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
    rank = (torch.exp(u * math.log(V + 1)) - 1).long().clamp_(0, V - 1)
    step = next(s for s in (7919, 104729, 1) if math.gcd(s, V) == 1)
    return rank * step % V


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "embed":
        s["tokens"] = _zipf(case["N"], case["V"], g)
        s["pad"] = 0 if case["padding"] else None
        if case["padding"]:
            s["tokens"][case["N"] - case["N"] // 16:] = 0
        s["weight"] = torch.empty(case["V"], case["D"], dtype=DTYPES[case["dtype"]], device="cuda").normal_(
            0, 0.02, generator=g).requires_grad_(case["grad"])
        s["scale"] = math.sqrt(case["D"])
        s["dout"] = None
        if case["grad"]:
            s["dout"] = torch.empty(case["N"], case["D"], dtype=DTYPES[case["dtype"]], device="cuda").normal_(
                0, 0.01, generator=g)
        return s
    z, likely = _logits(case, g)
    n, T, V = z.shape
    y = torch.where(torch.rand(n, T, device="cuda", generator=g) < 0.6, likely,
                    torch.randint(0, V, (n, T), device="cuda", generator=g))
    y[torch.rand(n, T, device="cuda", generator=g) < 0.02] = IGNORE  # padded positions
    if case["op"] == "score":
        if case["masked"]:  # values a grammar or a sampler has ruled out
            z.masked_fill_(torch.rand(V, device="cuda", generator=g) < 0.3, -math.inf)
            z.scatter_(2, likely[..., None], 9.0)
            y = torch.where(y == IGNORE, y, likely)
        s["targets"], s["top"] = y, case["top"]
        if case["grad"]:
            s["g_lp"] = torch.randn(n, T, device="cuda", generator=g)
            s["g_ent"] = torch.full((n, T), 0.01, device="cuda")
    else:
        k = case["k"]
        j = torch.arange(k, device="cuda")
        step = torch.randint(1, max(2, V // k + 1), (n, T, 1), device="cuda", generator=g).clamp_(max=max(1, V // k))
        ids = (likely[..., None] + j * step) % V  # distinct: k steps stay within the vocabulary
        t = torch.randn(n, T, k, device="cuda", generator=g) * 1.5
        t[..., 0] += 4
        keep = torch.randint(0, k + 1, (n, T, 1), device="cuda", generator=g)  # alternatives a row holds
        whole = torch.rand(n, T, 1, device="cuda", generator=g) < 0.8
        s["ids"] = torch.where(whole | (j < keep), ids, -1)
        s["t"] = t
        s["targets"] = y if case["hard"] else None
    s["logits"] = z.requires_grad_(bool(case.get("grad") or case.get("call") == "autograd"))
    return s


# ---- the framework's calls ------------------------------------------------

_fw = None


def _framework():
    global _fw
    if _fw is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "multimodal-ghm_amd"))
        from ghmclip import models
        _fw = models
    return _fw


def _run_own(s):
    fw = _framework()
    if s["op"] == "embed":
        out = fw.scaled_embedding(s["tokens"], s["weight"], s["scale"], padding_idx=s["pad"])
        if s["dout"] is None:
            return [out]
        return [out.detach(), torch.autograd.grad(out, s["weight"], s["dout"])[0]]
    if s["op"] == "score":
        r = fw.token_logprobs(s["logits"], s["targets"], top_k=s["top"], ignore_index=IGNORE)
        if s["grad"]:
            dz, = torch.autograd.grad((r.logprob, r.entropy), s["logits"], (s["g_lp"], s["g_ent"]))
            return [r.logprob.detach(), r.entropy.detach(), dz]
        return [r.logprob, r.entropy, r.top_logprob, r.top_id]
    args = (s["logits"], s["ids"], s["t"], s["targets"])
    opts = {"temperature": s["tau"], "alpha": s["alpha"], "ignore_index": IGNORE}
    if s["call"] == "step":
        loss, dz = fw.distill_loss_and_grad(*args, **opts)
        return [loss, dz]
    loss = fw.distill_loss(*args, **opts)
    if s["call"] == "eval":
        return [loss]
    return [loss.detach(), torch.autograd.grad(loss, s["logits"])[0]]


# ---- the plain forms ------------------------------------------------------


def _log_softmax(z):
    d = z - z.amax(-1, keepdim=True)
    return d - d.exp().sum(-1, keepdim=True).log()


def _plain_score(s):
    z = s["logits"].detach().float()
    y, counted = s["targets"].clamp(min=0), s["targets"] != IGNORE
    logp = _log_softmax(z)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    lp = torch.where(counted, logp.gather(-1, y[..., None])[..., 0], 0.0)
    ent = torch.where(counted, -plogp.sum(-1), 0.0)
    if s["grad"]:
        g1, g2 = s["g_lp"][..., None], s["g_ent"][..., None]
        dz = -(p * g1) - g2 * (plogp + p * ent[..., None])
        dz.scatter_add_(-1, y[..., None], g1)
        dz = torch.where(counted[..., None], dz, 0.0)
        return [lp, ent, dz.to(s["logits"].dtype)]
    del p, plogp
    # unique 64-bit keys: the value's order above, the lower id first among equals
    bits = (z + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    V = z.shape[-1]
    key = (order << 32) | (V - 1 - torch.arange(V, device=z.device))
    ids = V - 1 - (key.topk(s["top"], dim=-1).values & 0xffffffff)
    top = logp.gather(-1, ids)
    return [lp, ent, torch.where(counted[..., None], top, 0.0), torch.where(counted[..., None], ids, -1)]


def _plain_distill(s):
    z, tau, a = s["logits"].detach().float(), s["tau"], s["alpha"]
    present = s["ids"] >= 0
    teacher = present.any(-1)
    ids = s["ids"].clamp(min=0)
    counted = teacher if s["targets"] is None else s["targets"] != IGNORE
    t = torch.where(present, s["t"] / tau, -math.inf)
    t = torch.where(teacher[..., None], t, 0.0)
    logq = torch.where(present, _log_softmax(t), 0.0)
    q = torch.where(present, logq.exp(), 0.0)
    logp = _log_softmax(z / tau)
    row = a * tau * tau * (q * (logq - logp.gather(-1, ids))).sum(-1)
    count = counted.sum().clamp(min=1)
    if s["call"] != "eval":
        dz = logp.exp_() * teacher[..., None]
        dz.scatter_add_(-1, ids, -q)
        dz *= a * tau
    if s["targets"] is not None:
        y = s["targets"].clamp(min=0)[..., None]
        logp = _log_softmax(z)
        row = row - (1 - a) * logp.gather(-1, y)[..., 0]
        if s["call"] != "eval":
            logp = logp.exp_()
            logp.scatter_add_(-1, y, torch.full_like(logp[..., :1], -1.0))
            dz += (1 - a) * logp
    loss = torch.where(counted, row, 0.0).sum() / count
    if s["call"] == "eval":
        return [loss]
    dz = torch.where(counted[..., None], dz / count, 0.0)
    return [loss, dz.to(s["logits"].dtype)]


def _plain_embed(s):
    w = s["weight"].detach()
    out = (w[s["tokens"]].float() * s["scale"]).to(w.dtype)
    if s["dout"] is None:
        return [out]
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, s["tokens"], s["dout"].float())
    dw *= s["scale"]
    if s["pad"] is not None:
        dw[s["pad"]] = 0
    return [out, dw.to(w.dtype)]


def run(state):
    if own:
        return _run_own(state)
    return {"score": _plain_score, "distill": _plain_distill, "embed": _plain_embed}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "embed":
        N, V, D = case["N"], case["V"], case["D"]
        # ids and the rows they name are read (a row once, however often it is named), every output row written
        byt = N * 8 + min(N, V) * D * e + N * D * e
        if case["grad"]:
            byt += N * D * e + V * D * e
        return {"bytes": byt, "flops": N * D * (2 if case["grad"] else 1)}
    n, V = case["rows"], case["V"]
    if case["op"] == "score":
        byt = n * V * e + n * 8 + n * 8 + n * case["top"] * 12
        return {"bytes": byt + (n * V * e + n * 8 if case["grad"] else 0), "flops": n * V * (10 if case["grad"] else 5)}
    byt = n * V * e + n * case["k"] * 12 + (n * 8 if case["hard"] else 0)
    return {"bytes": byt + (n * V * e if case["call"] != "eval" else 0), "flops": n * V * (8 if case["hard"] else 5)}


# ---- the definitions in 64 bits -------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        w = s["weight"].detach()
        out = torch.nn.functional.embedding(s["tokens"], w).double().mul_(s["scale"])
        if not case["grad"]:
            return [out]
        # one row of ones and zeros per id would be the definition; ids in order give the same sums
        order = s["tokens"].argsort(stable=True)
        ids, count = s["tokens"][order].unique_consecutive(return_counts=True)
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        step = max(1, (1 << 27) // case["N"])
        for a in range(0, case["D"], step):  # column blocks keep the running sums small
            run_ = torch.cat([torch.zeros(1, min(step, case["D"] - a), dtype=torch.float64, device=w.device),
                              s["dout"][order, a:a + step].double().cumsum(0)])
            end = count.cumsum(0)
            dw[ids, a:a + step] = run_[end] - run_[end - count]
        dw *= s["scale"]
        if s["pad"] is not None:
            dw[s["pad"]] = 0
        return [out, dw]
    z = s["logits"].detach()
    n, T, V = z.shape
    z = z.reshape(n * T, V)
    if case["op"] == "score":
        y = s["targets"].reshape(-1)
        parts = []
        for a in range(0, n * T, max(1, (1 << 27) // V)):
            b = min(n * T, a + max(1, (1 << 27) // V))
            lse = torch.logsumexp(z[a:b].double(), -1)
            lp = z[a:b].double().sub_(lse[:, None])
            yy = y[a:b]
            live = (yy != IGNORE)
            ent = -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1)
            res = [torch.where(live, lp[torch.arange(b - a, device=z.device), yy.clamp(min=0)], 0.0),
                   torch.where(live, ent, 0.0)]
            if case["grad"]:
                g1, g2 = (s[k].reshape(-1)[a:b, None].double() for k in ("g_lp", "g_ent"))
                hot = torch.nn.functional.one_hot(yy.clamp(min=0), V).double() if V <= 64 else None
                p = lp.exp()
                dz = g2 * (torch.special.xlogy(p, p).neg_() - p * ent[:, None]) - g1 * p
                if hot is not None:
                    dz += g1 * hot
                else:
                    dz[torch.arange(b - a, device=z.device), yy.clamp(min=0)] += g1[:, 0]
                res.append(dz * live[:, None])
            else:
                top = lp.topk(case["top"], dim=-1).values
                res.append(torch.where(live[:, None], top, 0.0))
            parts.append(res)
        cat = [torch.cat(x) for x in zip(*parts)]
        cat[0], cat[1] = cat[0].view(n, T), cat[1].view(n, T)
        cat[2] = cat[2].view(n, T, -1)
        return cat if case["grad"] else cat + [None]
    k, tau, a = case["k"], case["tau"], case["alpha"]
    ids, t = s["ids"].reshape(n * T, k), s["t"].reshape(n * T, k).double()
    has = (ids >= 0).sum(-1) > 0
    live = has if s["targets"] is None else s["targets"].reshape(-1) != IGNORE
    t = torch.where(ids >= 0, t, -math.inf)
    q = torch.where(has[:, None], torch.softmax(torch.where(has[:, None], t / tau, 0.0), -1), 0.0)
    count = max(1, int(live.sum()))
    loss, grads = 0.0, []
    for b in range(0, n * T, max(1, (1 << 27) // V)):
        e = min(n * T, b + max(1, (1 << 27) // V))
        zz = z[b:e].double()
        P = torch.softmax(zz / tau, -1)
        qq, ii = q[b:e], ids[b:e].clamp(min=0)
        lse = torch.logsumexp(zz / tau, -1, keepdim=True)
        row = a * tau ** 2 * (torch.special.xlogy(qq, qq) - qq * (zz.gather(-1, ii) / tau - lse)).sum(-1)
        hard = s["targets"] is not None
        r = torch.arange(e - b, device=z.device)
        yy = s["targets"].reshape(-1)[b:e].clamp(min=0) if hard else None
        if hard:
            row = row + (1 - a) * (torch.logsumexp(zz, -1) - zz[r, yy])
        loss = loss + float((row * live[b:e]).sum())
        if case["call"] != "eval":
            dz = P.mul_(has[b:e, None]).scatter_add_(-1, ii, -qq).mul_(a * tau)
            if hard:
                one = torch.softmax(zz, -1)
                one[r, yy] -= 1
                dz += (1 - a) * one
            grads.append(dz.mul_(live[b:e, None]).div_(count))
    loss = torch.tensor(loss / count, dtype=torch.float64)
    return [loss] if case["call"] == "eval" else [loss, torch.cat(grads).view(n, T, V)]
