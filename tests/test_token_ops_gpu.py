"""The token operators (csrc/ghm_score.hip, ghm_distill.hip, ghm_embed.hip) against their definitions in 64 bits
(oracle/token_oracle.py, which also gives the bound that a 32-bit evaluation with one
final rounding may be off; the values below are never measured ones)."""
import gc
import math

import pytest
import torch

from oracle import token_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    from ghmclip import _native
    assert _native.hip_lib().ghm_device_ok() == 1
    torch.cuda.synchronize()  # what ran before this file has ended
    gc.collect()
    torch.cuda.empty_cache()
    yield
    torch.cuda.synchronize()
    gc.collect()
    torch.cuda.empty_cache()  # up to 40 GB


def _M():
    from ghmclip import models
    return models


def _near(got, want, bound, what):
    got = got.detach().double().to(want.device)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    err, b = (got - want)[fin].abs(), bound[fin]
    assert not torch.isnan(b).any(), what
    bad = err > b
    assert not bad.any(), f"{what}: off by {err[bad].max().item():.3e}, {(err[bad] / b[bad]).max().item():.2f} x the bound"


def _grad_near(got, want, bound, dtype, what):
    _near(got, want, bound * (1 + O.HALF[dtype]) + O.round_bound(want, dtype), what)


def _logits(rows, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, V, generator=g) * spread
    z[torch.arange(rows), torch.randint(0, V, (rows,), generator=g)] += 7
    return z.to(dtype)


def _targets(rows, V, seed, ignored=True):
    g = torch.Generator().manual_seed(seed + 1)
    y = torch.randint(0, V, (rows,), generator=g)
    if ignored and rows > 2:
        y[rows // 2] = -100
    return y


def _check_score(z, y, k, got, what, ignore=-100):
    """z on the CPU in its own type."""
    r = O.score(z.double(), y, k, ignore)
    if y is not None:
        _near(got.logprob, r["logprob"], r["blogprob"], what + " logprob")
    _near(got.entropy, r["entropy"], r["bentropy"], what + " entropy")
    if k:
        assert torch.equal(got.top_id.cpu(), r["top_id"]), what + " top_id"
        _near(got.top_logprob, r["top_logprob"], r["btop_logprob"], what + " top_logprob")
    return r


SHAPES = [(1, 1), (3, 2), (5, 10), (513, 10), (7, 31), (7, 32), (7, 33), (4, 64), (3, 65), (66, 127), (2, 257), (9, 500),
          (5, 1000), (2, 1024), (2, 2048), (2, 2049), (6, 3999), (3, 4097), (2, 8193), (1, 32771), (3, 70001), (300, 513),
          (1, 200003), (5, 140001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
def test_score(rows, V, dtype):
    M = _M()
    z, y = _logits(rows, V, dtype, rows + V), _targets(rows, V, rows + V)
    for k in sorted({0, 1, min(V, 5), min(V, 64)}):
        got = M.token_logprobs(z.to(DEV), y.to(DEV), top_k=k)
        assert got.logprob.dtype == got.entropy.dtype == torch.float32
        _check_score(z, y, k, got, f"k {k}")
        assert (got.top_id is None) == (k == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
def test_score_gradient(rows, V, dtype):
    M = _M()
    z, y = _logits(rows, V, dtype, rows + 3 * V), _targets(rows, V, V)
    k = min(V, 7)
    g = torch.Generator().manual_seed(5)
    g1, g2, g3 = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, k, generator=g)
    leaf = z.to(DEV).requires_grad_()
    got = M.token_logprobs(leaf, y.to(DEV), top_k=k)
    r = _check_score(z, y, k, got, "forward")
    assert not got.top_id.requires_grad
    both = (got.logprob * g1.to(DEV)).sum() + (got.entropy * g2.to(DEV)).sum() + (got.top_logprob * g3.to(DEV)).sum()
    dz, = torch.autograd.grad(both, leaf, retain_graph=True)
    want, bound = O.score_grad(z.double(), y, r, g1.double(), g2.double(), g3.double())
    assert dz.dtype == dtype
    _grad_near(dz, want, bound, dtype, "all three")
    dz, = torch.autograd.grad(got.logprob, leaf, g1.to(DEV), retain_graph=True)
    want, bound = O.score_grad(z.double(), y, r, g1.double())
    _grad_near(dz, want, bound, dtype, "logprob alone")
    dz, = torch.autograd.grad(got.top_logprob, leaf, g3.to(DEV))
    want, bound = O.score_grad(z.double(), y, r, None, None, g3.double())
    _grad_near(dz, want, bound, dtype, "alternatives alone")


def test_score_gradient_against_differences():
    M = _M()
    z, y = _logits(3, 7, torch.float32, 2, 1.0), torch.tensor([1, 6, 3])
    w = torch.randn(3, 2, generator=torch.Generator().manual_seed(3))

    def f(x):
        r = M.token_logprobs(x.to(DEV), y.to(DEV))
        return torch.stack([r.logprob, r.entropy], -1).double().cpu()
    leaf = z.to(DEV).requires_grad_()
    r = M.token_logprobs(leaf, y.to(DEV))
    dz, = torch.autograd.grad((r.logprob, r.entropy), leaf, (w[:, 0].to(DEV), w[:, 1].to(DEV)))
    h = 2.0 ** -6
    for v in range(7):
        e = torch.zeros_like(z)
        e[:, v] = h
        num = ((f(z + e) - f(z - e)) / (2 * h) * w.double()).sum(-1)
        # h^2 / 6 times a third derivative of at most 6 ln V, plus the rounding of two values over 2 h
        tol = (h * h * math.log(7) + 2 * 32 * O.U / (2 * h) * 4) * w.double().abs().sum(-1)
        assert ((dz[:, v].double().cpu() - num).abs() <= tol).all()


@pytest.mark.parametrize("V", [10, 300, 5000, 40000])
@pytest.mark.parametrize("bits", [torch.uint8, torch.int32, torch.int64])
def test_score_targets(V, bits):
    """Padding rows are not read (NaN in them changes nothing), ids outside the
    vocabulary poison their own row only."""
    M = _M()
    z, y = _logits(6, V, torch.float32, V), torch.tensor([3, 9, 200, 1, 0, 7])
    ignore = 9
    z[1] = math.nan
    leaf = z.to(DEV).requires_grad_()
    got = M.token_logprobs(leaf, y.to(bits).to(DEV), top_k=3, ignore_index=ignore)
    _check_score(z, y, 3, got, "ids", ignore)
    assert got.logprob[1] == 0 and got.entropy[1] == 0 and (got.top_id[1] == -1).all()
    assert torch.isnan(got.logprob[2]).item() == (V == 10)
    dz, = torch.autograd.grad(got.logprob.sum(), leaf)
    assert (dz[1] == 0).all() and torch.isnan(dz[2]).all().item() == (V == 10)
    assert torch.isfinite(dz[[0, 3, 4, 5]]).all()
    if bits != torch.uint8:
        got = M.token_logprobs(z.to(DEV), torch.tensor([-1, 9, V, 1, 0, 7], dtype=bits).to(DEV), ignore_index=ignore)
        assert torch.isnan(got.logprob[[0, 2]]).all() and torch.isfinite(got.logprob[3:]).all()
        assert torch.isfinite(got.entropy[[0, 2, 3]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 40, 200, 3000, 9000, 70001])
def test_score_masks_and_special_values(V, dtype):
    M = _M()
    z, y = _logits(10, V, dtype, V), torch.zeros(10, dtype=torch.long)
    low = torch.finfo(dtype).min
    z[0, 1:] = -math.inf                 # one value left
    z[1, : V // 2] = -math.inf           # fewer values than alternatives in a part of the row
    z[2, ::2] = low                      # the type's lowest value as a mask
    z[3] = low                           # ... everywhere: uniform
    z[4] = -math.inf                     # nothing left: no distribution
    z[5, V - 1] = math.nan
    z[6, 3] = math.inf
    z[7] = 0.5                           # all equal
    z[8] = torch.arange(V).to(dtype) / 16  # ascending: every step brings new alternatives
    z[9] = torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0)
    k = min(V, 20)
    leaf = z.to(DEV).requires_grad_()
    got = M.token_logprobs(leaf, y.to(DEV), top_k=k)
    r = _check_score(z, y, k, got, "special")
    dz, = torch.autograd.grad((got.logprob.sum() + got.entropy.sum()), leaf)
    one = torch.ones(10, dtype=torch.float64)
    want, bound = O.score_grad(z.double(), y, r, one, one)
    rows = [0, 1, 2, 3, 7, 8, 9]
    _grad_near(dz[rows], want[rows], bound[rows], dtype, "gradient")
    assert torch.isnan(dz[[4, 5, 6]]).any(-1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 33, 200, 300, 3000, 9000, 70001])
def test_score_first_value_nan(V, dtype):
    """NaN ranks first at every id, the first one too."""
    M = _M()
    z = _logits(6, V, dtype, V)
    z[:, 0] = math.nan
    z[1, V // 2] = z[2, V - 1] = math.nan
    z[3, 1] = math.inf
    z[4, 1:] = -math.inf
    z[5] = math.nan
    for k in (1, 3, min(V, 64)):
        _check_score(z, None, k, M.token_logprobs(z.to(DEV), top_k=k), f"k {k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 700, 20000])
def test_score_ties(V, dtype):
    """Few distinct values: the alternatives are the lowest ids of the largest values."""
    M = _M()
    g = torch.Generator().manual_seed(V)
    z = torch.randint(-3, 4, (9, V), generator=g).to(dtype)
    z[3] = -z[3].abs()
    z[4, V // 3:] = 3
    z[5] = torch.arange(V, 0, -1).to(dtype)
    for k in (1, 5, 33, 50):
        got = M.token_logprobs(z.to(DEV), top_k=k)
        assert got.logprob is None
        _check_score(z, None, k, got, f"ties k {k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", [(1030, 3000), (1100, 9001), (520, 20001), (513, 40001), (512, 70003), (600, 131072)])
def test_many_rows(rows, V, dtype):
    """The kernels of many long rows (one wave or several per row, rows kept in registers or
    read twice), checked on the device in 64 bits; vocabulary-sized offsets in odd rows."""
    M = _M()
    z, y = _logits(rows, V, dtype, V).to(DEV), _targets(rows, V, V).to(DEV)
    k = 24
    leaf = z.clone().requires_grad_()
    got = M.token_logprobs(leaf, y, top_k=k)
    r = O.score(z.double(), y, k)
    for name in ("logprob", "entropy", "top_logprob"):
        _near(getattr(got, name), r[name], r["b" + name], name)
    assert torch.equal(got.top_id, r["top_id"])
    none = M.token_logprobs(z, y)
    assert none.top_id is None and none.top_logprob is None
    _near(none.logprob, r["logprob"], r["blogprob"], "without alternatives")
    g = torch.linspace(-1, 1, rows, device=DEV)
    dz, = torch.autograd.grad((got.logprob, got.entropy), leaf, (g, 2 * g))
    want, bound = O.score_grad(z.double(), y, r, g.double(), 2 * g.double())
    _grad_near(dz, want, bound, dtype, "score gradient")
    del r, want, bound, dz
    ids, t = (x.to(DEV) for x in _teacher(rows, V, k, V))
    for tau, alpha in ((1.0, 1.0), (2.0, 0.5)):
        o = O.distill(z.double(), ids, t.double(), y if alpha < 1 else None, tau, alpha)
        n = int(o["counted"].sum())
        loss, dz = M.distill_loss_and_grad(z, ids, t, y if alpha < 1 else None, temperature=tau, alpha=alpha)
        total = o["row_loss"].sum()
        _near(loss, total / n, (o["brow_loss"].sum() + (rows + 28) * O.U * o["row_loss"].abs().sum()) / n, "mean")
        _grad_near(dz, o["dz"] / n, (o["bdz"] + 4 * O.U * o["dz"].abs()) / n, dtype, "step")
        loss = M.distill_loss(leaf, ids, t, y if alpha < 1 else None, temperature=tau, alpha=alpha, reduction="sum")
        got, = torch.autograd.grad(loss, leaf)
        _grad_near(got, o["dz"], o["bdz"] + 4 * O.U * o["dz"].abs(), dtype, "autograd")


@pytest.mark.parametrize("V", [2, 10, 32, 33, 64, 100, 256])
def test_likely_values_keep_their_digits(V):
    """One value holds nearly everything: log p = -log1p(rest), relative to itself.  The rest
    is a sum of V terms of |d| <= 24 units (3 u |d| + 2 u each), so off by (V + 90) u."""
    M = _M()
    g = torch.Generator().manual_seed(V)
    z = torch.randn(40, V, generator=g)
    y = torch.randint(0, V, (40,), generator=g)
    z[torch.arange(40), y] += 8 + 10 * torch.rand(40, generator=g)
    got = M.token_logprobs(z.to(DEV), y.to(DEV), top_k=1)
    d = z.double() - z.double().gather(-1, y[:, None])
    rest = torch.where(torch.arange(V) == y[:, None], 0.0, d.exp()).sum(-1)
    want = -torch.log1p(rest)
    _near(got.logprob, want, (V + 90) * O.U * want.abs(), "logprob")
    _near(got.top_logprob[:, 0], want, (V + 90) * O.U * want.abs(), "alternative")
    loss = M.distill_loss(z.to(DEV), y[:, None].to(DEV), torch.zeros(40, 1, device=DEV), reduction="none")
    _near(loss, -want, (V + 94) * O.U * want.abs(), "distillation of one entry")


def test_score_views():
    """Rows read in place past a prefix, every second row, values of a wider row, shifted
    storage, transposed and expanded logits; leading dimensions kept."""
    M = _M()
    g = torch.Generator().manual_seed(9)
    for dtype in DTYPES:
        base = (torch.randn(4, 6, 37, generator=g) * 2).to(dtype)
        for make in (lambda x: x[:, 1:], lambda x: x[::2], lambda x: x[..., 3:20], lambda x: x[0, 0],
                     lambda x: x.transpose(1, 2), lambda x: x[:1].expand(3, -1, -1), lambda x: x[1:, 2:4, 5:],
                     lambda x: x[:, :1, :1], lambda x: x[:0]):
            z = make(base)
            lead, V = z.shape[:-1], z.shape[-1]
            y = torch.randint(0, V, lead, generator=g)
            k = min(V, 4)
            on = make(base.to(DEV)).detach().requires_grad_()
            got = M.token_logprobs(on, y.to(DEV), top_k=k)
            assert got.logprob.shape == got.entropy.shape == lead and got.top_id.shape == (*lead, k)
            flat = M.TokenScores(got.logprob.reshape(-1), got.entropy.reshape(-1), got.top_logprob.reshape(-1, k),
                                 got.top_id.reshape(-1, k))
            if z.numel() == 0:
                continue
            r = _check_score(z.reshape(-1, V), y.reshape(-1), k, flat, "view")
            dz, = torch.autograd.grad(got.logprob.sum(), on)
            want, bound = O.score_grad(z.reshape(-1, V).double(), y.reshape(-1), r, torch.ones(max(1, y.numel())).double())
            assert dz.shape == z.shape
            _grad_near(dz.reshape(-1, V), want, bound, dtype, "view gradient")


def test_offsets_beyond_32_bits():
    """Rows 2^31 elements apart, in and out of every operator."""
    M = _M()
    V, step = 1000, 1 << 31
    buf = torch.empty(2 * step + V + 8, dtype=torch.bfloat16, device=DEV)
    z = torch.as_strided(buf, (3, V), (step, 1), 3)
    zc, y = _logits(3, V, torch.bfloat16, 1), torch.tensor([5, 999, 0])
    z.copy_(zc)
    _check_score(zc, y, 4, M.token_logprobs(z, y.to(DEV), top_k=4), "far rows")
    ids, t = torch.tensor([[1, 2], [3, 4], [999, 0]]), torch.randn(3, 2)
    loss, dz = M.distill_loss_and_grad(z, ids.to(DEV), t.to(DEV), reduction="sum")
    r = O.distill(zc.double(), ids, t.double(), None, 1.0, 1.0)
    _near(loss, r["row_loss"].sum(), r["brow_loss"].sum() + 8 * O.U * r["row_loss"].abs().sum(), "far loss")
    _grad_near(dz, r["dz"], r["bdz"], torch.bfloat16, "far gradient")
    del buf, z
    D = 4096  # a table of more than 2^32 elements
    V = (1 << 20) + 3
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    tok = torch.tensor([V - 1, 5, V - 1, 1 << 20, 524288])
    rows = torch.randn(5, D).to(torch.bfloat16)
    w[tok] = rows[[2, 1, 2, 3, 4]].to(DEV)
    w.requires_grad_()
    out = M.scaled_embedding(tok.to(DEV), w, 2.0)
    assert torch.equal(out.detach().cpu(), rows[[2, 1, 2, 3, 4]] * 2)
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    assert dw[V - 1].eq(4).all() and dw[5].eq(2).all() and dw[1 << 20].eq(2).all() and dw[524288].eq(2).all()
    assert int(dw.ne(0).any(-1).sum()) == 4


# ---- distillation ---------------------------------------------------------


def _teacher(rows, V, k, seed, ragged=True):
    g = torch.Generator().manual_seed(seed + 7)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)])
    t = torch.randn(rows, k, generator=g) * 2
    if ragged and rows > 3:
        ids[1] = -1                      # no entry at all
        ids[2, k // 2:] = -1
        t[3, 0] = -math.inf
    return ids, t


def _check_distill(z, ids, t, y, tau, alpha, dtype, what):
    M = _M()
    r = O.distill(z.double(), ids, t.double(), y, tau, alpha)
    on = [z.to(DEV), ids.to(DEV), t.to(DEV), None if y is None else y.to(DEV)]
    opts = dict(temperature=tau, alpha=alpha)
    rows = M.distill_loss(*on, reduction="none", **opts)
    assert rows.dtype == torch.float32
    _near(rows, r["row_loss"], r["brow_loss"], what + " rows")
    n = max(1, int(r["counted"].sum()))
    total, btotal = r["row_loss"].sum(), r["brow_loss"].sum() + (len(z) + 24) * O.U * r["row_loss"].abs().sum()
    loss, dz = M.distill_loss_and_grad(*on, **opts)
    _near(loss, total / n, btotal / n + 4 * O.U * total.abs() / n, what + " mean")
    _grad_near(dz, r["dz"] / n, (r["bdz"] + 4 * O.U * r["dz"].abs()) / n, dtype, what + " step gradient")
    leaf = on[0].clone().requires_grad_()
    loss = M.distill_loss(leaf, *on[1:], reduction="sum", **opts)
    _near(loss, total, btotal, what + " sum")
    got, = torch.autograd.grad(loss * 3, leaf)
    _grad_near(got, 3 * r["dz"], 3 * (r["bdz"] + 4 * O.U * r["dz"].abs()), dtype, what + " autograd")
    up = torch.linspace(-1, 2, len(z), dtype=torch.float64)
    got, = torch.autograd.grad(M.distill_loss(leaf, *on[1:], reduction="none", **opts), leaf, up.float().to(DEV))
    u32 = up.float().double()[:, None]
    _grad_near(got, u32 * r["dz"], (r["bdz"] + 4 * O.U * r["dz"].abs()) * u32.abs(), dtype, what + " rows' autograd")
    return loss


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V", SHAPES)
def test_distill(rows, V, dtype):
    z, y = _logits(rows, V, dtype, rows + V), _targets(rows, V, V + 2)
    for k, tau, alpha in ((min(V, 4), 1.0, 1.0), (min(V, 17), 2.0, 1.0), (min(V, 64), 1.0, 0.5), (min(V, 5), 3.0, 0.25),
                          (1, 0.5, 0.0)):
        ids, t = _teacher(rows, V, k, rows + V)
        _check_distill(z, ids, t, y if alpha < 1 or k == 1 else None, tau, alpha, dtype, f"k {k} tau {tau} alpha {alpha}")


@pytest.mark.parametrize("V", [10, 40, 3000, 20000, 70001])
@pytest.mark.parametrize("k", [1, 3, 1000, 1024])
def test_distill_entries(V, k):
    """More entries than values, repeated ids, teacher logits of 16 bits, 32-bit ids."""
    g = torch.Generator().manual_seed(V + k)
    z = _logits(6, V, torch.float32, V)
    ids = torch.randint(0, V, (6, k), generator=g).int()
    t = torch.randn(6, k, generator=g).to(torch.bfloat16)
    if k > 1:
        ids[1] = ids[1, 0]
        ids[2, 1] = -5
    y = _targets(6, V, 1)
    _check_distill(z, ids.long(), t.float(), None, 2.0, 1.0, torch.float32, "entries")
    M = _M()
    a = M.distill_loss_and_grad(z.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV).int(), temperature=2.0, alpha=0.5)
    b = M.distill_loss_and_grad(z.to(DEV), ids.long().to(DEV), t.float().to(DEV), y.to(DEV), temperature=2.0, alpha=0.5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("V", [10, 300, 3000, 20000, 70001])
def test_distill_special_values(V):
    M = _M()
    z = _logits(8, V, torch.float32, V)
    ids, t = _teacher(8, V, 4, V, ragged=False)
    y = torch.full((8,), 2)
    y[7] = -100
    z[0, :] = -math.inf
    z[0, ids[0]] = 1.0                   # only the teacher's values are left
    z[0, 2] = 0.0
    z[1, ids[1, 1]] = -math.inf          # the student rules out a value the teacher holds: infinite loss
    z[7] = math.nan                      # padding: not read
    t[7] = math.nan
    r = O.distill(z[:2].double(), ids[:2], t[:2].double(), None, 1.0, 1.0)
    rows = M.distill_loss(z[:2].to(DEV), ids[:2].to(DEV), t[:2].to(DEV), reduction="none")
    _near(rows, r["row_loss"], r["brow_loss"].nan_to_num(0, 0), "ruled out")
    assert rows[1] == math.inf
    ids[2, 0] = V                        # an id outside the vocabulary
    y[3] = V + 5
    t[4, 1] = math.nan
    t[5, 1] = math.inf
    for tau, alpha in ((1.0, 0.5), (2.0, 0.5)):
        loss, dz = M.distill_loss_and_grad(z.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV), temperature=tau, alpha=alpha,
                                           reduction="none")
        assert torch.isnan(loss[2:6]).all() and torch.isfinite(loss[[0, 6, 7]]).all()
        assert torch.isnan(dz[2:6]).any(-1).all() and torch.isfinite(dz[[0, 1, 6, 7]]).all() and (dz[7] == 0).all()


def _spread_rows(V, dtype, seed):
    """Rows whose values lie far apart, (logits, ids, teacher's logits, targets): finite masks that end or
    begin inside a lane's, a wave's or a part's values, and values of tens of thousands.  The teacher's
    entries and the targets are values that no mask holds."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(7, V, generator=g) * 3
    z[4] = (torch.randn(V, generator=g) * 2e4).clamp(-6e4, 6e4)
    z[5] = torch.linspace(-6e4, 6e4, V)          # the maximum rises with every step
    low = torch.finfo(dtype).min
    masks = torch.zeros(7, V, dtype=torch.bool)
    masks[0, :V // 2] = True
    masks[1, V // 2:] = True
    masks[2, ::2] = True
    masks[3, :V - 1] = True                      # one value left, the last
    z = z.to(dtype)
    z[masks] = low
    z[2, 1::4] = -1e4 * (2 if dtype == torch.float16 else 1e3)
    k = min(V // 2, 5)
    ids = torch.stack([(~m).nonzero()[:, 0][torch.randint(0, int((~m).sum()), (k,), generator=g)] for m in masks])
    ids[2] = ids[2] // 4 * 4 + 3 if V >= 8 else ids[2]
    ids[2].clamp_(max=(V - 4) // 4 * 4 + 3)
    return z, ids, torch.randn(7, k, generator=g) * 2, ids[:, 0].clone()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tau", [1e-6, 1e-3, 20.0, 1e3, 1e4, 1e6])
@pytest.mark.parametrize("V", [10, 100, 700, 3000, 9001, 40000, 70001, 140001, 300001])
def test_distill_temperatures_with_values_far_apart(V, tau, dtype):
    """Both ends of the accepted temperatures: what is e^-10000 at a temperature of 1 is 0.99 at one
    of 10^6, in rows of one lane, one wave, several waves and parts; the loss alone, the loss with its gradient
    and the gradient from saved statistics, each against the definition."""
    M = _M()
    z, ids, t, y = _spread_rows(V, dtype, V)
    # a gradient is alpha temperature (p - q): times a power of two that keeps it within f16
    up = 2.0 ** -20 if tau == 1e6 else 1.0
    for alpha in (1.0, 0.5):
        yy = y if alpha < 1 else None
        r = O.distill(z.double(), ids, t.double(), yy, tau, alpha)
        on = [z.to(DEV), ids.to(DEV), t.to(DEV), None if yy is None else yy.to(DEV)]
        opts = dict(temperature=tau, alpha=alpha, reduction="none")
        want, bound = up * r["dz"], up * (r["bdz"] + 4 * O.U * r["dz"].abs())
        loss, dz = M.distill_loss_and_grad(*on, grad_scale=up, **opts)
        _near(loss, r["row_loss"], r["brow_loss"], f"alpha {alpha}, step")
        _grad_near(dz, want, bound, dtype, f"alpha {alpha}, step's gradient")
        _near(M.distill_loss(*on, **opts), r["row_loss"], r["brow_loss"], f"alpha {alpha}, loss alone")
        leaf = on[0].requires_grad_()
        loss = M.distill_loss(leaf, *on[1:], **opts)
        _near(loss, r["row_loss"], r["brow_loss"], f"alpha {alpha}, loss")
        dz, = torch.autograd.grad(loss, leaf, torch.full_like(loss, up))
        _grad_near(dz, want, bound, dtype, f"alpha {alpha}, autograd")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 33, 100, 300, 3000, 9000, 40000, 140001])
def test_distill_bad_targets_without_entries(V, dtype):
    """alpha = 1 and no teacher's entry: a target outside the vocabulary makes its row NaN, the gradient's
    too, in rows of every length; one that holds only that it counts is 0."""
    z, y = _logits(6, V, dtype, V), torch.tensor([1, V, -1, V - 1, -100, 1 << 40])
    ids, t = _teacher(6, V, 4, V, ragged=False)
    ids[[1, 3, 4]] = -1
    t[2] = -math.inf
    for tau in (1.0, 2.0):
        _check_distill(z, ids, t, y, tau, 1.0, dtype, f"tau {tau}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 33, 100, 300, 3000, 9000, 40000, 140001])
def test_distill_rows_without_a_distribution(V, dtype):
    """A row without a finite maximum is NaN, loss and gradient, whether or not the teacher has an
    entry there and whatever the gradient is scaled with."""
    M = _M()
    z, y = _logits(8, V, dtype, V), torch.zeros(8, dtype=torch.long)
    ids, t = _teacher(8, V, 4, V, ragged=False)
    z[:3] = -math.inf
    z[3, V - 1] = math.nan
    z[4, V // 2] = math.inf
    ids[[0, 3, 4, 5]] = -1
    y[2] = -100
    for tau, alpha in ((1.0, 1.0), (2.0, 1.0), (1.0, 0.5), (2.0, 0.5), (2.0, 0.0)):
        _check_distill(z, ids, t, y, tau, alpha, dtype, f"tau {tau} alpha {alpha}")
        loss, dz = M.distill_loss_and_grad(z.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV), temperature=tau, alpha=alpha,
                                           reduction="none", grad_scale=0.0)
        bad = torch.tensor([True, True, False, True, True, False, False, False])
        assert torch.equal(loss.isnan().cpu(), bad) and torch.equal(dz.isnan().all(-1).cpu(), bad)
        assert (dz[~bad] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 33, 300, 3000, 40000, 140001])
def test_distill_without_the_teacher(V, dtype):
    """alpha = 0 is the hard labels' loss alone, gradient and all, whatever the teacher's logits hold and
    though the student may have ruled its values out."""
    M = _M()
    z, y = _logits(5, V, dtype, V), torch.tensor([0, 1, 2, -100, 3])
    ids, t = _teacher(5, V, 4, V, ragged=False)
    t[0, 1], t[1, 2], t[4] = math.nan, math.inf, math.nan
    z[2, ids[2, 0]] = -math.inf if ids[2, 0] != 2 else z[2, ids[2, 0]]
    clean = t.nan_to_num(0, 0)
    for tau in (1.0, 2.0):
        r = O.distill(z.double(), ids[:, :1], torch.full((5, 1), -math.inf).double(), y, tau, 0.0)
        on = [z.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV)]
        opts = dict(temperature=tau, alpha=0.0, reduction="none")
        loss, dz = M.distill_loss_and_grad(*on, **opts)
        _near(loss, r["row_loss"], r["brow_loss"], "loss")
        _grad_near(dz, r["dz"], r["bdz"] + 4 * O.U * r["dz"].abs(), dtype, "step")
        leaf = on[0].requires_grad_()
        got, = torch.autograd.grad(M.distill_loss(leaf, *on[1:], **opts).sum(), leaf)
        _grad_near(got, r["dz"], r["bdz"] + 4 * O.U * r["dz"].abs(), dtype, "autograd")
        again = M.distill_loss_and_grad(on[0].detach(), on[1], clean.to(DEV), on[3], **opts)
        assert torch.equal(again[0], loss) and torch.equal(again[1], dz)


def test_distill_nothing_counts():
    M = _M()
    z = _logits(5, 77, torch.float32, 0).to(DEV).requires_grad_()
    ids, t = torch.full((5, 3), -1, device=DEV), torch.zeros(5, 3, device=DEV)
    loss = M.distill_loss(z, ids, t)
    dz, = torch.autograd.grad(loss, z)
    assert loss == 0 and (dz == 0).all()
    y = torch.full((5,), -100, device=DEV)
    loss, dz = M.distill_loss_and_grad(z.detach(), ids, t, y, alpha=0.5)
    assert loss == 0 and (dz == 0).all()
    loss, dz = M.distill_loss_and_grad(z.detach()[:0], ids[:0], t[:0])
    assert loss == 0 and dz.shape == (0, 77)
    assert M.distill_loss(z.detach()[:0], ids[:0], t[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("V", [10, 77, 3000])
def test_distill_empty_batch_with_hard_labels(V):
    """No row at all, with targets and alpha below 1: the loss of nothing and an empty gradient."""
    M = _M()
    z = torch.zeros(0, V, device=DEV, requires_grad=True)
    ids, t = torch.zeros(0, 3, dtype=torch.long, device=DEV), torch.zeros(0, 3, device=DEV)
    y = torch.zeros(0, dtype=torch.long, device=DEV)
    for reduction in ("mean", "sum", "none"):
        loss = M.distill_loss(z, ids, t, y, alpha=0.5, temperature=2.0, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and (loss == 0).all()
        dz, = torch.autograd.grad(loss, z, torch.ones_like(loss))
        assert dz.shape == z.shape
        loss, dz = M.distill_loss_and_grad(z.detach(), ids, t, y, alpha=0.5, reduction=reduction)
        assert (loss == 0).all() and dz.shape == z.shape


def test_distill_views_and_module():
    M = _M()
    base = _logits(24, 37, torch.bfloat16, 3).view(4, 6, 37)
    ids, t = _teacher(20, 37, 5, 1)
    z = base.to(DEV)[:, 1:]
    r = O.distill(base[:, 1:].reshape(20, 37).double(), ids, t.double(), None, 2.0, 1.0)
    leaf = z.detach().requires_grad_()
    loss = M.TopLogitsDistillLoss(temperature=2.0, reduction="sum")(leaf, ids.view(4, 5, 5).to(DEV), t.view(4, 5, 5).to(DEV))
    loss.backward()
    _near(loss, r["row_loss"].sum(), r["brow_loss"].sum() + 44 * O.U * r["row_loss"].abs().sum(), "view loss")
    _grad_near(leaf.grad.reshape(20, 37), r["dz"], r["bdz"] + 4 * O.U * r["dz"].abs(), torch.bfloat16, "view gradient")


def test_distill_gradient_against_differences():
    M = _M()
    z, y = _logits(3, 7, torch.float32, 2, 1.0), torch.tensor([1, 6, 3])
    ids, t = torch.tensor([[0, 3], [6, 2], [5, -1]]), torch.tensor([[1.0, 0.5], [2.0, -1.0], [0.3, 9.0]])
    opts = dict(temperature=2.0, alpha=0.5)

    def f(x):
        return M.distill_loss(x.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV), reduction="none", **opts).double().cpu()
    _, dz = M.distill_loss_and_grad(z.to(DEV), ids.to(DEV), t.to(DEV), y.to(DEV), reduction="sum", **opts)
    h = 2.0 ** -6
    for v in range(7):
        e = torch.zeros_like(z)
        e[:, v] = h
        num = (f(z + e) - f(z - e)) / (2 * h)
        # third derivatives of the two log-sum-exps: at most 1 and 1 / tau
        assert ((dz[:, v].double().cpu() - num).abs() <= h * h + 2 * 64 * O.U * 8 / (2 * h)).all()


# ---- embedding ------------------------------------------------------------

EMBED_SHAPES = [(1, 1, 1), (1, 10, 256), (7, 3, 5), (64, 10, 64), (1000, 10, 33), (513, 257, 128), (4096, 50, 8),
                (3000, 70001, 16), (9000, 300, 96), (20000, 7, 130), (40000, 1000, 40), (33, 5, 4096), (70000, 2, 8),
                (4097, 70001, 16), (16384, 600, 8), (16385, 3001, 24), (300, 1100000, 4), (270001, 5000, 12),
                (9000, 511, 7), (9000, 512, 3), (100, 40, 4100), (12000, 300000, 8),
                (40000, 7, 450), (500, 32, 1025), (100, 33, 70)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,D", EMBED_SHAPES)
def test_embedding(N, V, D, dtype):
    M = _M()
    g = torch.Generator().manual_seed(N + V + D)
    tok = (torch.rand(N, generator=g) ** 3 * V).long().clamp(max=V - 1)
    w = torch.randn(V, D, generator=g).to(dtype)
    dout = torch.randn(N, D, generator=g).to(dtype)
    scale = float(torch.tensor(math.sqrt(D)))
    for pad in (None, V - 1):
        leaf = w.to(DEV).requires_grad_()
        out = M.scaled_embedding(tok.to(DEV), leaf, scale, padding_idx=pad)
        want, bound = O.embed(tok, w.double(), scale)
        assert out.dtype == dtype
        _grad_near(out, want, bound, dtype, "rows")
        dw, = torch.autograd.grad(out, leaf, dout.to(DEV))
        want, bound = O.embed_grad(tok, dout.double(), scale, V, pad)
        _grad_near(dw, want, bound, dtype, "gradient")
        again, = torch.autograd.grad(M.scaled_embedding(tok.to(DEV), leaf, scale, padding_idx=pad), leaf, dout.to(DEV))
        assert torch.equal(dw, again)


@pytest.mark.parametrize("N,V,D", EMBED_SHAPES + [(262144, 40, 8), (262145, 600, 5), (600000, 70001, 3), (32768, 32, 512)])
@pytest.mark.parametrize("hot", [False, True])
def test_embedding_gradient_sums_every_row_once(N, V, D, hot):
    """Whole numbers: their sums are exact in f32 in any order (at most 8 N < 2^23), so a row that is left
    out, taken twice or given to another token changes the result.  hot: nearly all rows are of
    one token, whose sum goes over every chunk and block."""
    M = _M()
    g = torch.Generator().manual_seed(N + V + D)
    tok = (torch.rand(N, generator=g) ** 3 * V).long().clamp(max=V - 1)
    if hot:
        tok = torch.where(torch.rand(N, generator=g) < 0.98, V // 2, tok)
    dout = torch.randint(-8, 9, (N, D), generator=g)
    want = torch.zeros(V, D, dtype=torch.float64).index_add_(0, tok, dout.double())
    for pad in (None, tok[-1].item()):
        if pad is not None:
            want[pad] = 0
        for dtype in DTYPES:
            leaf = torch.zeros(V, D, dtype=dtype, device=DEV, requires_grad=True)
            out = M.scaled_embedding(tok.to(DEV), leaf, 0.5, padding_idx=pad)
            dw, = torch.autograd.grad(out, leaf, dout.to(dtype).to(DEV))
            assert torch.equal(dw.cpu(), (want * 0.5).float().to(dtype)), (dtype, pad)


@pytest.mark.parametrize("bits", [torch.uint8, torch.int32, torch.int64])
@pytest.mark.parametrize("N", [5, 3000, 30000])
def test_embedding_tokens(N, bits):
    """Tokens of every width and outside the table, one token repeated, none of a range,
    shapes of any rank, strided tables and gradients."""
    M = _M()
    g = torch.Generator().manual_seed(N)
    V, D = 200, 24
    tok = torch.randint(0, 256 if bits == torch.uint8 else 230, (N,), generator=g)
    if bits != torch.uint8:
        tok[0], tok[-1] = -1, V
    w, dout = torch.randn(V, 2 * D, generator=g), torch.randn(N, D + 7, generator=g)
    leaf = w.to(DEV)[:, :D].detach().requires_grad_()
    out = M.scaled_embedding(tok.to(bits).to(DEV), leaf, 0.5)
    want, bound = O.embed(tok, w[:, :D].double(), 0.5)
    _grad_near(out, want, bound, torch.float32, "rows")
    dw, = torch.autograd.grad(out, leaf, dout.to(DEV)[:, :D])
    want, bound = O.embed_grad(tok, dout[:, :D].double(), 0.5, V)
    _grad_near(dw, want, bound, torch.float32, "gradient")
    one = torch.full((N,), 3, dtype=bits, device=DEV).view(-1, 5 if N % 5 == 0 else 1)
    out = M.scaled_embedding(one, leaf, 1.0)
    assert out.shape == (*one.shape, D)
    dw, = torch.autograd.grad(out.sum(), leaf)  # an expanded gradient
    assert (dw[3] == N).all() and int(dw.ne(0).any(-1).sum()) == 1
    dw, = torch.autograd.grad(M.scaled_embedding(one[:0], leaf), leaf, torch.zeros(0, one.shape[1], D, device=DEV))
    assert (dw == 0).all()


def test_embedding_module():
    M = _M()
    torch.manual_seed(0)
    ref = torch.nn.Embedding(50, 12, padding_idx=-1)
    torch.manual_seed(0)
    emb = M.ScaledEmbedding(50, 12, padding_idx=-1, scale=3.0).to(DEV)
    assert torch.equal(ref.weight, emb.weight.cpu())
    tok = torch.tensor([[1, 49, 3], [1, 1, 0]])
    emb(tok.to(DEV)).sum().backward()
    assert emb.weight.grad[1].eq(9).all() and emb.weight.grad[49].eq(0).all() and emb.weight.grad[2].eq(0).all()


# ---- how they are called --------------------------------------------------


def test_refusals():
    M = _M()
    z = torch.zeros(4, 10, device=DEV)
    y = torch.zeros(4, dtype=torch.long, device=DEV)
    with pytest.raises(TypeError, match="float32"):
        M.token_logprobs(z.double(), y)
    with pytest.raises(TypeError, match="targets"):
        M.token_logprobs(z, y.float())
    with pytest.raises(ValueError, match="targets"):
        M.token_logprobs(z, y[:3])
    with pytest.raises(ValueError, match="targets"):
        M.token_logprobs(z, y.cpu())
    for k in (-1, 11, 65, 2.0):
        with pytest.raises(ValueError, match="top_k"):
            M.token_logprobs(z, y, top_k=k)
    with pytest.raises(ValueError, match="V >= 1"):
        M.token_logprobs(z[:, :0])
    ids, t = torch.zeros(4, 2, dtype=torch.long, device=DEV), torch.zeros(4, 2, device=DEV)
    for bad in (dict(temperature=0.0), dict(temperature=math.inf), dict(temperature=math.nan),
                dict(temperature=1e-7), dict(temperature=1e7), dict(alpha=0.5),
                dict(alpha=-0.1), dict(alpha=1.1), dict(reduction="median")):
        with pytest.raises(ValueError):
            M.distill_loss(z, ids, t, **bad)
    with pytest.raises(TypeError, match="top_ids"):
        M.distill_loss(z, ids.to(torch.uint8), t)
    with pytest.raises(ValueError, match="top_ids"):
        M.distill_loss(z, ids[:3], t)
    with pytest.raises(ValueError, match="top_ids"):
        M.distill_loss(z, ids[:, :0], t[:, :0])
    with pytest.raises(ValueError, match="top_logits"):
        M.distill_loss(z, ids, t[:, :1])
    with pytest.raises(TypeError, match="top_logits"):
        M.distill_loss(z, ids, t.double())
    w = torch.zeros(10, 4, device=DEV)
    with pytest.raises(TypeError, match="weight"):
        M.scaled_embedding(y, w.double())
    with pytest.raises(TypeError, match="tokens"):
        M.scaled_embedding(y.float(), w)
    with pytest.raises(ValueError, match="weight"):
        M.scaled_embedding(y, w[0])
    for pad in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            M.scaled_embedding(y, w, padding_idx=pad)


def test_calls_without_leading_dimensions_or_targets():
    M = _M()
    z = _logits(1, 50, torch.float32, 1)
    one, y = z[0].to(DEV).requires_grad_(), torch.tensor(7, device=DEV)
    r = O.score(z.double(), torch.tensor([7]), 3)
    got = M.token_logprobs(one, y, top_k=3)
    assert got.logprob.shape == () and got.top_id.shape == (3,)
    _near(got.logprob.view(1), r["logprob"], r["blogprob"], "one row")
    loss = M.distill_loss(one, got.top_id, got.top_logprob, y, alpha=0.5, reduction="none")
    assert loss.shape == () and torch.autograd.grad(loss, one)[0].shape == (50,)
    # entropy alone, no targets
    for rows, V in ((4, 10), (4, 100), (4, 3000), (4, 140001)):
        z = _logits(rows, V, torch.float32, V)
        leaf = z.to(DEV).requires_grad_()
        got = M.token_logprobs(leaf)
        assert got.logprob is None and got.top_id is None
        r = O.score(z.double(), None, 0)
        dz, = torch.autograd.grad(got.entropy.sum(), leaf)
        want, bound = O.score_grad(z.double(), None, r, None, torch.ones(rows).double())
        _grad_near(dz, want, bound, torch.float32, "entropy alone")
    w = torch.randn(9, 6, device=DEV, requires_grad=True)
    out = M.scaled_embedding(torch.tensor(4, device=DEV), w, 3.0)
    assert torch.equal(out, w[4] * 3) and out.shape == (6,)


@pytest.mark.parametrize("V", [10, 90, 900, 9000, 70001])
def test_distill_targets_that_only_count(V):
    """alpha = 1 with targets: they say which rows count, and no more."""
    z, y = _logits(7, V, torch.float32, V), _targets(7, V, V)
    ids, t = _teacher(7, V, min(V, 6), V)
    _check_distill(z, ids, t, y, 1.5, 1.0, torch.float32, "alpha 1 with targets")


@pytest.mark.parametrize("N,V", [(60, 20), (60, 50), (6000, 300), (6000, 2000), (40000, 2000), (300000, 40)])
def test_embedding_of_padding_alone(N, V):
    """No token of the table: every row of the gradient is 0, whatever the buffer held."""
    M = _M()
    w = torch.randn(V, 8, device=DEV, requires_grad=True)
    tok = torch.full((N,), 3, device=DEV)
    tok[::2] = V + 5
    tok[1::4] = -9
    out = M.scaled_embedding(tok, w, 1.0, padding_idx=3)
    junk = torch.full((V, 8), math.nan, device=DEV)
    del junk  # the gradient is likely to take this block of the allocator
    dw, = torch.autograd.grad(out, w, torch.full_like(out, math.nan))
    assert (dw == 0).all()


@pytest.mark.parametrize("dtype,N,D", [(torch.float32, 67201, 1001), (torch.bfloat16, 131071, 1030),
                                       (torch.float16, 140001, 961), (torch.bfloat16, 9600001, 15),
                                       (torch.float32, 13500001, 5)])
def test_embedding_of_large_outputs(dtype, N, D):
    """Outputs of more than 256 MB with rows that are not whole lines, from an aligned address
    and from others: one rounded product per value, and nothing beside the output is written."""
    M = _M()
    from ghmclip.models import token_ops as T
    V = 301
    g = torch.Generator().manual_seed(D)
    w = torch.randn(V, D, generator=g).to(dtype).to(DEV)
    tok = torch.randint(0, V, (N,), generator=g)
    bad = torch.tensor([0, 7, 8, N // 2, N - 1])
    tok[bad] = torch.tensor([V, -1, V + 5, -7, 1 << 40])
    tok = tok.to(DEV)
    ok = (tok >= 0) & (tok < V)
    rows = (w.float() * 1.5).to(dtype)

    def check(out):
        for a in range(0, N, 1 << 20):
            o, t, k = out[a:a + (1 << 20)], tok[a:a + (1 << 20)], ok[a:a + (1 << 20)]
            assert torch.equal(o[k], rows[t[k]])
            assert o[~k].isnan().all()
    check(M.scaled_embedding(tok, w, 1.5))
    for off in (1, 3):
        buf = torch.full((N * D + 64,), 7., dtype=dtype, device=DEV)
        T._call(buf.device, "ghm_embed_rows_fwd", tok.data_ptr(), 64, w.data_ptr(), T._DTYPE[dtype], D, 1.5,
                buf.data_ptr() + off * buf.element_size(), N, V, D)
        check(buf[off:off + N * D].view(N, D))
        assert (buf[:off] == 7).all() and (buf[off + N * D:] == 7).all()


def test_embedding_gradient_of_two_strides():
    M = _M()
    g = torch.Generator().manual_seed(2)
    tok = torch.randint(0, 40, (5, 7), generator=g)
    w, big = torch.randn(40, 12, generator=g), torch.randn(5, 9, 12, generator=g)
    leaf = w.to(DEV).requires_grad_()
    dw, = torch.autograd.grad(M.scaled_embedding(tok.to(DEV), leaf, 1.5), leaf, big.to(DEV)[:, 1:8])
    want, bound = O.embed_grad(tok.reshape(-1), big[:, 1:8].reshape(35, 12).double(), 1.5, 40)
    _grad_near(dw, want, bound, torch.float32, "two strides")


def test_outputs_of_more_than_2_31_values():
    """Gradients past 32-bit offsets: the last rows of a 2.2e9-value batch."""
    M = _M()
    rows, V = 17000, 131072
    z = torch.empty(rows, V, dtype=torch.bfloat16, device=DEV).normal_(0, 2)
    y = torch.randint(0, V, (rows,), device=DEV)
    ids, t = torch.randint(0, V, (rows, 2), device=DEV), torch.randn(rows, 2, device=DEV)
    _, dz = M.distill_loss_and_grad(z, ids, t, reduction="sum")
    tail = slice(rows - 4, rows)
    o = O.distill(z[tail].double(), ids[tail], t[tail].double(), None, 1.0, 1.0)
    _grad_near(dz[tail], o["dz"], o["bdz"], torch.bfloat16, "distillation")
    del dz
    leaf = z.requires_grad_()
    got = M.token_logprobs(leaf, y, top_k=2)
    dz, = torch.autograd.grad(got.logprob.sum(), leaf)
    r = O.score(z.detach()[tail].double(), y[tail], 2)
    assert torch.equal(got.top_id[tail], r["top_id"])
    want, bound = O.score_grad(z.detach()[tail].double(), y[tail], r, torch.ones(4, device=DEV).double())
    _grad_near(dz[tail], want, bound, torch.bfloat16, "scores")


def _repeats(got, want):
    """got [n, *want.shape]: every got[i] is want, bit for bit (in slices: got may be large)."""
    step = max(1, (1 << 30) // max(1, want.numel()))
    return all(torch.equal(got[a:a + step], want.expand_as(got[a:a + step])) for a in range(0, len(got), step))


@pytest.mark.parametrize("V", [33, 300])
def test_more_rows_than_a_grid_has_threads(V):
    """More than 2^26 rows of one wave each, 2^32 threads: a batch of rows repeated (expanded
    logits, no copy) has the bits of that batch alone, in all of its repetitions."""
    M = _M()
    n, rows = 16400, 4099
    z, y = _logits(rows, V, torch.bfloat16, V).to(DEV), _targets(rows, V, V).to(DEV)
    ids, t = torch.randint(0, V, (rows, 1), device=DEV).int(), torch.randn(rows, 1, device=DEV).bfloat16()
    zz, yy, ii, tt = z.expand(n, -1, -1), y.int().expand(n, -1), ids.expand(n, -1, -1), t.expand(n, -1, -1)
    one, many = M.token_logprobs(z, y.int(), top_k=2), M.token_logprobs(zz, yy, top_k=2)
    assert all(_repeats(a, b) for a, b in zip(many, one))
    del one, many
    opts = dict(alpha=0.5, temperature=2.0, reduction="none")
    assert _repeats(M.distill_loss(zz, ii, tt, yy, **opts), M.distill_loss(z, ids, t, y.int(), **opts))
    for a, b in zip(M.distill_loss_and_grad(zz, ii, tt, yy, **opts), M.distill_loss_and_grad(z, ids, t, y.int(), **opts)):
        assert _repeats(a, b)
    del a, b
    grads = []
    for x in (z, zz):
        leaf = x.detach().requires_grad_()
        lead = x.shape[:-1]
        lp = M.token_logprobs(leaf, (y.int().expand(lead))).logprob
        g = torch.linspace(-1, 1, rows, device=DEV).expand(lead)
        first = torch.autograd.grad(lp, leaf, g)[0]
        del lp
        if V == 33:
            loss = M.distill_loss(leaf, ids.expand(*lead, -1), t.expand(*lead, -1), y.int().expand(lead), **opts)
            grads.append((first, torch.autograd.grad(loss, leaf, g)[0]))
            del loss
        else:
            grads.append((first,))
        del first
    assert all(_repeats(b, a) for a, b in zip(*grads))


def test_more_table_rows_than_a_grid_has_threads():
    """A lookup of more than 2^24 rows that take a block each."""
    M = _M()
    N, V, D = (1 << 24) + 5, 9, 4128
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 2 * N * D + (4 << 30):
        pytest.skip("an output of 139 GB")
    w = torch.randn(V, D, device=DEV).bfloat16()
    tok = torch.randint(0, V, (N,), device=DEV)
    out = M.scaled_embedding(tok.int(), w, 2.0)
    at = torch.cat([torch.arange(2000, device=DEV), torch.randint(0, N, (50000,), device=DEV),
                    torch.arange(N - 2000, N, device=DEV)])
    assert torch.equal(out[at], (w * 2)[tok[at]])


def test_one_row_of_2_30_values():
    """The longest row there may be.  A lane adds 2^30 / (64 parts of 8 waves of 64 lanes) = 2^15 terms, so
    the sum is off by 2^15 + 100 units relative to itself at most, 2^-8.99."""
    M = _M()
    V, rel = 1 << 30, (2 ** 15 + 100) * O.U
    torch.cuda.empty_cache()
    z = torch.empty(1, V, dtype=torch.bfloat16, device=DEV).normal_(0, 2, generator=torch.Generator(DEV).manual_seed(1))
    top = [V // 2 + 3, V - 1, 7]
    z[0, top] = torch.tensor([20.0, 20.0, 19.0], dtype=torch.bfloat16, device=DEV)
    got = M.token_logprobs(z, torch.tensor([V - 1], device=DEV), top_k=3)
    s = t = 0.0
    for a in range(0, V, 1 << 26):
        d = z[0, a:a + (1 << 26)].double() - 20
        s += float(d.exp().sum())
        t += float((d.exp() * -d).sum())
    assert got.top_id.tolist() == [top]
    assert abs(got.logprob.item() + math.log(s)) <= rel + 8 * O.U
    assert abs(got.entropy.item() - math.log(s) - t / s) <= rel + 2 * rel * t / s + 64 * O.U
    leaf = z.requires_grad_()
    dz, = torch.autograd.grad(M.token_logprobs(leaf, torch.tensor([V - 1], device=DEV)).logprob.sum(), leaf)
    at = torch.tensor([0, 7, 12345, V // 2 + 3, V - 2, V - 1], device=DEV)
    p = (z.detach()[0, at].double() - 20).exp() / s
    want = torch.where(at == V - 1, 1.0, 0.0) - p
    assert ((dz[0, at].double() - want).abs() <= 2 * rel * p + O.round_bound(want, torch.bfloat16) * 2).all()
    del dz, leaf
    ids, tl = torch.tensor([[V - 1, 0, V // 2]], device=DEV), torch.tensor([[2.0, 1.0, 0.0]], device=DEV)
    loss, dz = M.distill_loss_and_grad(z.detach(), ids, tl)
    q = torch.softmax(tl.double(), -1)
    zi = z.detach()[0, ids[0]].double()
    kl = (q * (q.log() - (zi - 20 - math.log(s)))).sum().item()
    assert abs(loss.item() - kl) <= rel + 64 * O.U * 40
    assert M.distill_loss(z.detach(), ids, tl).item() == pytest.approx(kl, abs=rel + 64 * O.U * 40)
    want = (zi - 20).exp() / s - q[0]
    assert ((dz[0, ids[0]].double() - want).abs() <= 2 * rel * (zi - 20).exp() / s + O.round_bound(want, torch.bfloat16) * 2).all()


def test_2_31_rows():
    """As many rows and tokens as there may be."""
    M = _M()
    R = (1 << 31) - 1
    torch.cuda.empty_cache()
    z, y = torch.zeros(R, 1, dtype=torch.bfloat16, device=DEV), torch.zeros(R, dtype=torch.uint8, device=DEV)
    y[-1] = 1
    got = M.token_logprobs(z, y)
    assert got.logprob[-1].isnan() and (got.logprob[:-1] == 0).all() and (got.entropy == 0).all()
    del got, y
    torch.cuda.empty_cache()
    ids = torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(R, 1)
    loss, dz = M.distill_loss_and_grad(z, ids, torch.zeros(1, 1, dtype=torch.bfloat16, device=DEV).expand(R, 1))
    assert loss == 0 and (dz == 0).all()
    del loss, dz, z
    torch.cuda.empty_cache()
    tok = torch.randint(0, 40, (R,), device=DEV, dtype=torch.uint8)
    w = torch.randn(40, 1, device=DEV).bfloat16().requires_grad_()
    out = M.scaled_embedding(tok, w, 2.0)
    for a in range(0, R, 1 << 28):
        assert torch.equal(out[a:a + (1 << 28)].detach(), (w.detach() * 2)[tok[a:a + (1 << 28)].long()])
    dw, = torch.autograd.grad(out, w, torch.ones_like(out))
    n = sum(torch.bincount(tok[a:a + (1 << 28)], minlength=40) for a in range(0, R, 1 << 28))
    # a chunk's 256 ones are exact, and each of four waves joins 2^31 / 40 / 256 / 4 of them
    rel = (2 ** 31 / 40 / 1024 + 4) * O.U
    assert ((dw[:, 0].double() - 2 * n).abs() <= 2 * n * rel + O.round_bound(2 * n.double(), torch.bfloat16)).all()
    torch.cuda.empty_cache()


def test_second_gradient_is_refused():
    M = _M()
    z = torch.randn(3, 9, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(M.token_logprobs(z, torch.zeros(3, dtype=torch.long, device=DEV)).logprob.sum(), z,
                             create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def _calls(z, y, ids, t, w, tok):
    """One run of each operator with its gradient; all outputs."""
    M = _M()
    r = M.token_logprobs(z, y, top_k=5)
    a, = torch.autograd.grad((r.logprob, r.entropy), z, (torch.ones_like(r.logprob), torch.ones_like(r.entropy)))
    loss = M.distill_loss(z, ids, t, y, temperature=2.0, alpha=0.5)
    b, = torch.autograd.grad(loss, z)
    c = M.distill_loss_and_grad(z.detach(), ids, t)
    out = M.scaled_embedding(tok, w, 2.0)
    d, = torch.autograd.grad(out, w, torch.ones_like(out))
    return [r.logprob, r.entropy, r.top_logprob, r.top_id, a, loss, b, *c, out, d]


def _inputs(rows, V, seed, dtype=torch.float32):
    z = _logits(rows, V, dtype, seed).to(DEV).requires_grad_()
    ids, t = _teacher(rows, V, 4, seed)
    g = torch.Generator().manual_seed(seed)
    return [z, _targets(rows, V, seed).to(DEV), ids.to(DEV), t.to(DEV),
            torch.randn(V, 16, generator=g).to(DEV).requires_grad_(), torch.randint(0, V, (3 * rows,), generator=g).to(DEV)]


@pytest.mark.parametrize("rows,V", [(40, 10), (3, 40000), (700, 3000)])
def test_captured_and_replayed(rows, V):
    """Two graphs and eager calls in turn: every replay has the eager bits."""
    sets = [_inputs(rows, V, s) for s in (1, 2)]
    other = _inputs(rows, V, 3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for x in sets:
            _calls(*x)
        for x in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append([o.detach() for o in _calls(*x)])
            graphs.append(g)
    torch.cuda.current_stream().wait_stream(s)
    want = [o.detach().clone() for o in _calls(*other)]
    for turn in range(3):
        with torch.no_grad():
            for x, k in zip(sets, (0, 1)):
                x[0].copy_(_logits(rows, V, torch.float32, 10 * turn + k))
        graphs[0].replay()
        graphs[1].replay()
        mine = [o.detach() for o in _calls(*other)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine, want))
        for x, got in zip(sets, outs):
            assert all(torch.equal(a, b.detach()) for a, b in zip(got, _calls(*x)))


def test_other_streams():
    """Calls on two streams at once, each on its own inputs, have the bits of calls alone."""
    sets = [_inputs(300, 9000, s, torch.bfloat16) for s in (1, 2)]
    for x in sets:
        x[4] = x[4].detach().requires_grad_()
    want = [[o.detach().clone() for o in _calls(*x)] for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append([o.detach() for o in _calls(*x)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_distilling_the_vlm():
    """A run of the operators as they are used: the teacher's next-token logits scored,
    their alternatives kept, a student's model trained on them; its parameters' gradients
    equal those of the same loss written in torch operations."""
    M = _M()
    torch.manual_seed(0)
    B, T1, V = 4, 12, 10
    kw = dict(n_token=T1 + 1, n_i_token=1, num_class=V, n_embd=128, n_guided_layers=[1, 1], n_mlp_hidden=512,
              auto_regressive=True, sequential=True, layernorm=True)
    teacher, student = (M.AutoRegressiveTransformer(n_layer=n, **kw).to(DEV) for n in (4, 3))
    xt, zi = torch.randint(0, V, (B, T1), device=DEV), torch.randn(B, 1, V, device=DEV)
    y = torch.randint(0, V, (B, T1), device=DEV)
    y[0, :3] = -100
    with torch.no_grad():
        s = M.token_logprobs(teacher(xt, zi)[0], y, top_k=4)
    live = y != -100
    assert (s.top_id[~live] == -1).all() and (s.top_id[live] >= 0).all()
    loss_fn = M.TopLogitsDistillLoss(temperature=2.0, alpha=0.7)
    logits = student(xt, zi)[0]
    loss = loss_fn(logits, s.top_id, s.top_logprob, y)
    loss.backward()
    got = {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None}
    student.zero_grad()
    logits = student(xt, zi)[0]
    z = logits.double()
    q = torch.softmax(s.top_logprob.double() / 2, -1)
    kl = (q * (q.log() - torch.log_softmax(z / 2, -1).gather(-1, s.top_id.clamp(min=0)))).sum(-1)
    ce = -torch.log_softmax(z, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0]
    want = ((0.3 * ce + 0.7 * 4 * kl) * live).sum() / live.sum()
    want.backward()
    assert abs(loss.item() - want.item()) <= 64 * O.U * abs(want.item())
    assert got
    for n, p in student.named_parameters():
        if n in got:
            # the same backward kernels on logits gradients that differ by f32 rounding; the
            # largest entry carries the scale through the layers
            assert (got[n] - p.grad).abs().max() <= 1e-4 * p.grad.abs().max() + 1e-9, n


def test_both_ends_of_a_vocabulary():
    """Scaled embedding, tied readout, distillation and scoring together on a vocabulary
    of 3,001 values: the table's gradient from both ends against 64 bits."""
    M = _M()
    V, D, B, T = 3001, 32, 3, 11
    g = torch.Generator().manual_seed(4)
    emb = M.ScaledEmbedding(V, D, scale=math.sqrt(D)).to(DEV)
    tok = torch.randint(0, V, (B, T), generator=g)
    tlog = torch.randn(B, T, V, generator=g) * 3
    s = M.token_logprobs(tlog.to(DEV), top_k=8)
    h = emb(tok.to(DEV))
    logits = h @ emb.weight.t()
    loss = M.distill_loss(logits, s.top_id, s.top_logprob, temperature=2.0)
    loss = loss - 0.01 * M.token_logprobs(logits).entropy.mean()
    loss.backward()
    w = emb.weight.detach().double().cpu().requires_grad_()
    z = (w[tok] * emb.scale) @ w.t()
    q = torch.softmax(s.top_logprob.double().cpu() / 2, -1)
    kl = 4 * (q * (q.log() - torch.log_softmax(z / 2, -1).gather(-1, s.top_id.cpu()))).sum(-1).mean()
    p = torch.softmax(z, -1)
    want = kl + 0.01 * (p * torch.log_softmax(z, -1)).sum(-1).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    # f32 products over D and V terms on both sides of the operators
    assert (emb.weight.grad.double().cpu() - w.grad).abs().max() <= 1e-5 * w.grad.abs().max()
