"""Linear layer with its epilogue, and its gradients, against float64.

Tolerances, from the arithmetic and before any run, with u half a unit of the
type (2^-9 bf16, 2^-12 fp16 of a value; doubled below for values at a power of
two): a sum of K products accumulated in fp32 is off by at most 2^-20 of the
sum of their sizes, the activations (slope at most 1.13) by 2^-20 of theirs, y
by u of itself on top.  In the backward z is rounded (its slope moves by at
most 1.2 u |z|, 0 for relu) and dz is rounded (u of it); dx and dweight sum
that over the other operand's sizes."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

import mhc_b200
from mhc_b200 import AutoPatcher, FusedLinear, MHCRewire, linear_act

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}
ACT = {"none": lambda z: z, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}
EPS = 2.0 ** -20


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _make(M, N, K, dtype, seed, bias=True, residual=True):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    x, w = r(M, K).to(dtype), (r(N, K) / K ** 0.5).to(dtype)
    return (x, w, (0.3 * r(N)).to(dtype) if bias else None, r(M, N).to(dtype) if residual else None,
            r(M, N).to(dtype))


def _within(got, want, tol, what):
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} values, worst "
                           f"{float(((got.double() - want).abs() / tol).max()):.2f}")


def _check(x, w, b, res, dy, act, y, grads):
    """y and (dx, dw, db) against float64."""
    u, tiny = U[x.dtype], TINY[x.dtype]
    X, W, D = x.double(), w.double(), dy.double()
    z = X @ W.t() + (0 if b is None else b.double())
    size = X.abs() @ W.abs().t() + (0 if b is None else b.double().abs())
    zz = z.clone().requires_grad_(True)
    a = ACT[act](zz)
    a.sum().backward()
    want = a.detach() + (0 if res is None else res.double())
    _within(y, want, u * want.abs() + 1.2 * EPS * size + EPS * a.detach().abs() + tiny + 1e-30, "y")
    if grads is None:
        return
    dz = D * zz.grad
    slope = 1.2 * u * z.abs() * D.abs() if act in ("silu", "gelu") else torch.zeros_like(D)
    noise = slope + EPS * D.abs() * (1 + size)
    if act == "relu":  # a z that is 0 to within its error may fall on either side
        noise = torch.where(z.abs() <= 2 * EPS * size + tiny, D.abs(), noise)
    rounded = noise + (u * dz.abs() + tiny if act != "none" else 0)
    dx, dw, db = grads
    for name, got, want, tol in (
            ("dx", dx, dz @ W, rounded @ W.abs() + EPS * (dz.abs() @ W.abs())),
            ("dw", dw, dz.t() @ X, rounded.t() @ X.abs() + EPS * (dz.abs().t() @ X.abs())),
            ("db", db, dz.sum(0), noise.sum(0) + EPS * dz.abs().sum(0))):
        if got is not None:
            assert got.dtype == x.dtype
            _within(got, want, tol + u * want.abs() + tiny + 1e-30, name)


# tokens: each side of the few-rows kernel (8, 16), of a tile (128); widths: one
# tile column of 64, ragged, odd (padded rows), several waves of the widest tile
# (in all three products)
SIZES = [(1, 64, 64), (1, 1500, 1001), (5, 17, 8), (8, 333, 4096), (9, 128, 40), (16, 100, 96),
         (17, 64, 64), (100, 1, 1), (130, 257, 100), (129, 72, 8), (300, 1000, 333), (77, 1500, 1001),
         (1500, 2600, 700), (2048, 4096, 264), (2300, 2040, 2000), (2300, 2042, 1999)]


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("M,N,K", SIZES)
def test_forward_and_gradients(dtype, M, N, K):
    act = ["none", "relu", "silu", "gelu"][(M + N) % 4]
    x, w, b, res, dy = _make(M, N, K, dtype, M + N + K)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, res)]
    y = linear_act(*leaves[:3], residual=leaves[3], activation=act)
    assert y.shape == (M, N) and y.dtype == dtype
    grads = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(grads[3], dy)
    _check(x, w, b, res, dy, act, y.detach(), grads[:3])
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, residual=res, activation=act), y)


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("M", [3, 12, 200])
def test_every_epilogue(act, bias, residual, M):
    x, w, b, res, dy = _make(M, 96, 120, torch.bfloat16, M, bias, residual)
    leaves = [None if t is None else t.clone().requires_grad_(True) for t in (x, w, b)]
    y = linear_act(*leaves, residual=res, activation=act)
    want = [t for t in leaves if t is not None]
    g = iter(torch.autograd.grad(y, want, dy))
    grads = [None if t is None else next(g) for t in leaves]
    _check(x, w, b, res, dy, act, y.detach(), grads)


@pytest.mark.parametrize("which", range(3))
def test_one_gradient_alone(which):
    """Each gradient without the others: a frozen weight, a frozen input, the bias only."""
    x, w, b, res, dy = _make(70, 90, 50, torch.float16, 1)
    leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, w, b))]
    y = linear_act(*leaves, residual=res, activation="silu")
    (g,) = torch.autograd.grad(y, [leaves[which]], dy)
    grads = [None] * 3
    grads[which] = g
    _check(x, w, b, res, dy, "silu", y.detach(), grads)


def test_gradient_against_differences():
    """The loss sum(y dy) along random directions of x, w and b.  y carries the type's
    rounding, u |y| a value at random signs; 0.25 of step keeps it below the slope."""
    x, w, b, res, dy = _make(64, 80, 48, torch.float16, 3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(linear_act(*leaves, residual=res, activation="gelu"), leaves, dy)
    f = lambda *t: float((linear_act(*t, residual=res, activation="gelu").double() * dy.double()).sum())  # noqa: E731
    h = 2.0 ** -5
    for i, (t, g) in enumerate(zip((x, w, b), grads)):
        for s in range(3):
            d = torch.randn(t.shape, device=DEV, generator=_gen(s)).to(t.dtype)
            up, dn = ((t + k * h * d) for k in (1, -1))
            args = [[x, w, b], [x, w, b]]
            args[0][i], args[1][i] = up, dn
            moved = (up.double() - dn.double())  # as rounded
            slope = float((g.double() * moved).sum())
            size = float(g.double().norm() * moved.norm())
            assert abs(f(*args[0]) - f(*args[1]) - slope) <= 0.05 * size


def test_strides_and_offsets():
    """Rows of a wider matrix, odd offsets, transposed and expanded operands: as copies."""
    big = torch.randn(40, 3, 200, device=DEV, generator=_gen(1)).to(torch.bfloat16)
    wide = torch.randn(150, 210, device=DEV, generator=_gen(2)).to(torch.bfloat16)
    for x, w in [(big[:, 1, 3:100], wide[:, 5:102]), (big[:, :, :64], wide[3:, 8:72]),
                 (big[:, 0, ::2], wide[:, :100]), (big[0, 0].expand(30, 200), wide[:, :200]),
                 (big[:, 0, :150], wide.t()[:90, :150]), (big[0, 0, 1:57], wide[:, 1:57])]:
        N = w.shape[0]
        res = torch.randn(*x.shape[:-1], N + 1, device=DEV, generator=_gen(3)).to(x.dtype)[..., 1:]
        out = []
        for contiguous in (False, True):
            c = (lambda t: t.contiguous()) if contiguous else (lambda t: t)
            a, b = c(x.detach()).requires_grad_(True), c(w.detach()).requires_grad_(True)
            y = linear_act(a, b, residual=c(res), activation="silu")
            dy = torch.ones(1, device=DEV, dtype=x.dtype).expand(y.shape)
            out.append((y.detach(), *torch.autograd.grad(y, [a, b], c(dy))))
        assert out[0][0].shape == (*x.shape[:-1], N)
        for p, q in zip(*out):
            assert torch.equal(p, q)


def test_no_rows():
    w = torch.randn(30, 20, device=DEV).to(torch.bfloat16).requires_grad_(True)
    b = torch.zeros(30, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    x = torch.empty(0, 5, 20, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = linear_act(x, w, b, activation="relu")
    assert y.shape == (0, 5, 30)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], y.detach())
    assert dx.shape == x.shape and not dw.any() and not db.any()


def test_nan_and_infinity_reach_their_row_only():
    for M in (4, 140):
        x, w, b, _, _ = _make(M, 70, 65, torch.bfloat16, 4, residual=False)
        x[2, 3], x[3, 64] = float("nan"), float("inf")
        for act in ("none", "relu", "silu", "gelu"):
            y = linear_act(x, w, b, activation=act)
            assert torch.isnan(y[2]).all()
            rest = [i for i in range(M) if i not in (2, 3)]
            assert torch.isfinite(y[rest]).all()
            assert not torch.isfinite(linear_act(x, w, b)[3]).any()


def test_repeatable_streams_and_graph():
    x, w, b, res, dy = _make(300, 520, 264, torch.bfloat16, 6)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def run():
        y = linear_act(*leaves, residual=res, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    for rows in (4, 300):
        xs = x[:rows].clone()
        with torch.no_grad():
            linear_act(xs, w, b)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = linear_act(xs, w, b)
            xs.mul_(2)
            g.replay()
            assert torch.equal(y, linear_act(xs, w, b))


def test_module_in_a_rewired_model():
    """FusedLinear is an nn.Linear to AutoPatcher and MHCRewire."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(FusedLinear(64, 64, activation="silu", device=DEV),
                                FusedLinear(64, 32, device=DEV))
    assert AutoPatcher.patch(model, n_streams=4, verbose=False, output_dtype="input",
                             identity_init=False) == 1
    assert isinstance(model[0], MHCRewire) and isinstance(model[0].inner, FusedLinear)
    x = torch.randn(20, 64, device=DEV).to(torch.bfloat16).requires_grad_(True)
    model(x).float().square().sum().backward()
    assert x.grad is not None and all(torch.isfinite(p.grad).all() for p in model.parameters()
                                      if p.grad is not None)
    lin = FusedLinear(48, 40, activation="gelu", device=DEV, dtype=torch.float16)
    h = torch.randn(3, 5, 48, device=DEV).half()
    r = torch.randn(3, 5, 40, device=DEV).half()
    want = F.gelu(F.linear(h.double(), lin.weight.double(), lin.bias.double())) + r.double()
    assert (lin(h, residual=r).double() - want).abs().max() < 2.0 ** -8


def test_mhc_b200_exports():
    assert mhc_b200.FusedLinear is FusedLinear


def test_differentiated_once_only():
    x, w, _, _, dy = _make(20, 48, 64, torch.bfloat16, 1)
    x.requires_grad_(), w.requires_grad_()
    plain = torch.autograd.grad(linear_act(x, w, activation="silu"), [x, w], dy)
    kept = torch.autograd.grad(linear_act(x, w, activation="silu"), [x, w], dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, kept))
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(kept[0].sum(), w)


def test_only_what_is_asked_for():
    """Each operand's gradient by itself is the one that it has among the others."""
    *ts, dy = _make(40, 56, 72, torch.float16, 2)
    f = lambda t: linear_act(t[0], t[1], t[2], residual=t[3], activation="relu")  # noqa: E731
    every = [t.clone().requires_grad_() for t in ts]
    want = torch.autograd.grad(f(every), every, dy)
    for i in range(4):
        one = [t.clone().requires_grad_(i == k) for k, t in enumerate(ts)]
        assert torch.equal(torch.autograd.grad(f(one), one[i], dy)[0], want[i])
        assert torch.equal(torch.autograd.grad(f(every), every[i], dy)[0], want[i])
    x = ts[0].clone().requires_grad_()
    y = linear_act(x, ts[1])
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
