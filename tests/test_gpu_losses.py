"""Losses on logits against a float64 restatement (torch autograd for the
gradients), at the sizes, strides and masks where the kernels change path.

Tolerances, from the arithmetic and before any run: a log probability is
(x - m) - ln S with S a sum of V positive fp32 terms, each off by at most two
units of 2^-23 (the exponential) and summed in a tree of short chains, so
|error| <= 2^-22 (8 + |x - m|).  A gradient value is c (1[target] - p): p is
off by the same relative amount, c by what its log probabilities give, and the
result is rounded once to the logits' type (2^-9 bf16, 2^-12 fp16 of it)."""

from __future__ import annotations

import pytest
import torch

import mhc_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"
IGN = -100
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(shape, dtype, seed, boost=6.0):
    g = _gen(seed)
    x = 2.0 * torch.randn(*shape, device=DEV, generator=g)
    y = torch.randint(0, shape[-1], shape[:-1], device=DEV, generator=g)
    x.scatter_add_(-1, y[..., None], torch.full_like(x[..., :1], boost))
    return x.to(dtype), y


def _ref_logp(x64, y):
    keep = y != IGN
    lp = torch.log_softmax(x64, dim=-1).gather(-1, torch.where(keep, y, 0)[..., None])[..., 0]
    return torch.where(keep, lp, torch.zeros_like(lp))


def _logp_tol(x, y):
    """Per row: 2^-22 (8 + |x_t - m|)."""
    xt = x.double().gather(-1, y.clamp(min=0)[..., None])[..., 0]
    return 2.0 ** -22 * (8 + (xt - x.double().amax(-1)).abs())


def _check_grad(got, want, coef_err, dtype):
    """coef_err: relative error allowed on a row's factor c."""
    got, want = got.double(), want.double()
    row = want.abs().amax(dim=-1, keepdim=True)
    tol = HALF_ULP[dtype] * want.abs() + (coef_err + 2.0 ** -20) * row + 2.0 ** -25
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} values, worst {((got - want).abs() / tol).max():.2f}"


# 257: a tail; 4099: one vector a thread and ends; 32000: NV=16 (bf16); 33000: two
# blocks a row; 140001: past what registers hold in fp32
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (5, 257), (1, 131072), (600, 512), (33, 4099),
                                 (9, 32000), (7, 33000), (4, 140001)])
def test_token_logprobs(dtype, T, V):
    x, y = _logits((T, V), dtype, 100 * T + V)
    if T > 2:
        y[1] = IGN
    d = torch.randn(T, device=DEV, generator=_gen(5))
    xg = x.clone().requires_grad_(True)
    lp = mhc_b200.token_logprobs(xg, y)
    lp.backward(d)
    x64 = x.double().requires_grad_(True)
    ref = _ref_logp(x64, y)
    ref.backward(d.double())
    assert lp.dtype == torch.float32 and xg.grad.dtype == dtype
    assert ((lp.double() - ref).abs() <= _logp_tol(x, y)).all()
    _check_grad(xg.grad, x64.grad, 0.0, dtype)
    if T > 2:
        assert lp[1] == 0 and not xg.grad[1].any()


def _policy_inputs(x, y, seed):
    g = _gen(seed)
    lp = _ref_logp(x.double(), y).float()
    old = lp + 0.3 * torch.randn(lp.shape, device=DEV, generator=g)
    ref = lp + 0.3 * torch.randn(lp.shape, device=DEV, generator=g)
    adv = torch.randn(lp.shape, device=DEV, generator=g)
    # clear of the clip's edges, where the slope jumps
    r = lp - old
    for e in (0.8, 1.28):
        old = torch.where((r - torch.tensor(e, device=DEV).log()).abs() < 0.01, old - 0.05, old)
        r = lp - old
    return old, ref, adv


def _policy_ref(x64, y, old, adv, ref, kl_coef, d=None):
    lp, keep = _ref_logp(x64, y), (y != IGN).double()
    r = (lp - old.double()).exp()
    u = torch.minimum(r * adv.double(), r.clamp(1 - 0.2, 1 + 0.28) * adv.double())
    k = torch.zeros_like(lp)
    if ref is not None:
        k = torch.expm1(ref.double() - lp) - (ref.double() - lp)
    n = keep.sum() if d is None else d
    return (keep * (kl_coef * k - u)).sum() / n, lp, (keep * k).sum() / n


def _policy_tol(x, y, adv, old, ref):
    """Relative error of c and absolute error of a token's loss: the log
    probability's error, twice over for the exponential's own."""
    return 4 * float(_logp_tol(x, y).max()) + 2.0 ** -20


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,kl", [(1, 7, 0.1), (3, 512, 0.0), (300, 1000, 0.05), (5, 131072, 0.05),
                                    (17, 32000, 0.0), (11, 50001, 0.05), (4, 140001, 0.05),
                                    (2, 270011, 0.05), (700, 129, 0.05)])
def test_policy_loss(dtype, T, V, kl):
    x, y = _logits((T, V), dtype, 7 * T + V)
    old, ref, adv = _policy_inputs(x, y, 3)
    if T > 2:
        y[2::3] = IGN
    kw = dict(clip_low=0.2, clip_high=0.28, kl_coef=kl, ref_logprobs=ref if kl else None)
    x64 = x.double().requires_grad_(True)
    want, lp, wkl = _policy_ref(x64, y, old, adv, ref if kl else None, kl)
    want.backward()
    tol = _policy_tol(x, y, adv, old, ref)
    scale = float(adv.abs().max()) * 4 + 1

    r = mhc_b200.policy_loss_grad(x, y, old, adv, **kw)
    assert abs(float(r.loss) - float(want)) <= tol * scale
    assert abs(float(r.kl) - float(wkl)) <= tol * 4
    assert ((r.logprobs.double() - lp).abs() <= _logp_tol(x, y)).all()
    _check_grad(r.dlogits, x64.grad, tol * 4, dtype)

    xg = x.clone().requires_grad_(True)
    a = mhc_b200.policy_loss(xg, y, old, adv, **kw)
    a.loss.backward()
    assert torch.equal(a.loss.detach(), r.loss) and torch.equal(xg.grad, r.dlogits)
    assert not a.logprobs.requires_grad and not a.kl.requires_grad
    # a scaled loss is differentiated from the logits, not by scaling what was rounded
    xs = x.clone().requires_grad_(True)
    (mhc_b200.policy_loss(xs, y, old, adv, **kw).loss * 64.0).backward()
    scaled = mhc_b200.policy_loss_grad(x, y, old, adv, grad_scale=64.0, **kw)
    _check_grad(xs.grad, 64.0 * x64.grad, tol * 4, dtype)
    _check_grad(scaled.dlogits, 64.0 * x64.grad, tol * 4, dtype)
    with torch.no_grad():
        assert torch.equal(mhc_b200.policy_loss(x, y, old, adv, **kw).loss, r.loss)


def test_policy_loss_kept_graph_and_denominator():
    x, y = _logits((40, 700), torch.float32, 1)
    old, ref, adv = _policy_inputs(x, y, 2)
    xg = x.clone().requires_grad_(True)
    loss = mhc_b200.policy_loss(xg, y, old, adv, clip_high=0.28, denominator=160).loss
    (g1,) = torch.autograd.grad(loss, xg, retain_graph=True)
    keep = g1.clone()
    g1.mul_(3.0)  # the caller's own: the next backward does not see it
    (g2,) = torch.autograd.grad(loss, xg)
    x64 = x.double().requires_grad_(True)
    want, _, _ = _policy_ref(x64, y, old, adv, None, 0.0, d=160)
    want.backward()
    _check_grad(keep, x64.grad, 1e-5, torch.float32)
    _check_grad(g2, x64.grad, 1e-5, torch.float32)


def test_policy_gradient_against_differences():
    """Central differences of the kernel's own loss along random directions: the
    loss carries 2^-24 of rounding, the step 2e-2 an O(h^2) term."""
    x, y = _logits((24, 300), torch.float32, 11)
    old, ref, adv = _policy_inputs(x, y, 12)
    kw = dict(clip_low=0.2, clip_high=0.28, kl_coef=0.1, ref_logprobs=ref)
    r = mhc_b200.policy_loss_grad(x, y, old, adv, **kw)
    for s in range(4):
        d = torch.randn(x.shape, device=DEV, generator=_gen(s))
        h = 2e-3
        up = mhc_b200.policy_loss_grad(x + h * d, y, old, adv, **kw).loss
        dn = mhc_b200.policy_loss_grad(x - h * d, y, old, adv, **kw).loss
        slope = float(r.dlogits.double().mul(d).sum())
        size = float(r.dlogits.double().norm())
        assert abs((float(up) - float(dn)) / (2 * h) - slope) <= 0.02 * size + 1e-4


def _pref_ref(x64, y, ref, cu, beta, e, d):
    lp = _ref_logp(x64, y)
    delta = torch.where(y != IGN, lp - ref.double(), torch.zeros_like(lp))
    R = torch.stack([delta[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
    z = beta * (R[0::2] - R[1::2])
    sp = torch.nn.functional.softplus
    return ((1 - e) * sp(-z) + e * sp(z)).sum() / d, lp, z


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,V", [((1, 1), 3), ((0, 4), 512), ((5, 0, 0, 0), 257),
                                    ((17, 30, 1, 64, 3, 3), 1001), ((9, 8), 32000), ((3, 2), 140001),
                                    ((300, 277), 512)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_preference_loss(dtype, lens, V, index):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1] + 2  # two rows of no sequence
    x, y = _logits((T, V), dtype, V + T)
    y[1::5] = IGN
    ref = _ref_logp(x.double(), y).float() + 0.1 * torch.randn(T, device=DEV, generator=_gen(1))
    cut = torch.tensor(cu, dtype=index, device=DEV)
    pairs, beta, e = len(lens) // 2, 0.2, 0.1
    x64 = x.double().requires_grad_(True)
    want, lp, z = _pref_ref(x64, y, ref, cu, beta, e, pairs)
    want.backward()
    # a margin sums its tokens' errors; the loss and c are at most as steep
    dz = beta * max(1, max(lens)) * 2 * float(_logp_tol(x, y).max()) + 2.0 ** -22
    kw = dict(beta=beta, label_smoothing=e)
    r = mhc_b200.preference_loss_grad(x, y, ref, cut, **kw)
    assert ((r.margins.double() - z).abs() <= dz * (1 + z.abs())).all()
    assert abs(float(r.loss) - float(want)) <= 2 * dz + 2.0 ** -22
    assert ((r.logprobs.double() - lp).abs() <= _logp_tol(x, y)).all()
    _check_grad(r.dlogits, x64.grad, 4 * dz + 1e-6, dtype)
    assert not r.dlogits[cu[-1]:].any()
    xg = x.clone().requires_grad_(True)
    a = mhc_b200.preference_loss(xg, y, ref, cut, **kw)
    a.loss.backward()
    assert torch.equal(a.loss.detach(), r.loss) and torch.equal(xg.grad, r.dlogits)
    s = mhc_b200.preference_loss_grad(x, y, ref, cut, grad_scale=32.0, denominator=3 * pairs, **kw)
    _check_grad(s.dlogits, x64.grad * (32.0 / 3), 4 * dz + 1e-6, dtype)


def test_preference_gradient_against_differences():
    x, y = _logits((40, 200), torch.float32, 21)
    cu = torch.tensor([0, 11, 20, 33, 40], device=DEV)
    ref = _ref_logp(x.double(), y).float() + 0.2
    f = lambda v: mhc_b200.preference_loss_grad(v, y, ref, cu, beta=0.3, label_smoothing=0.05)  # noqa: E731
    r = f(x)
    for s in range(4):
        d = torch.randn(x.shape, device=DEV, generator=_gen(s))
        h = 2e-3
        slope = float(r.dlogits.double().mul(d).sum())
        size = float(r.dlogits.double().norm())
        assert abs((float(f(x + h * d).loss) - float(f(x - h * d).loss)) / (2 * h) - slope) <= \
            0.02 * size + 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_logits(dtype):
    """Views read in place: shifted sequences, rows of a wider matrix at an odd
    offset, a last axis that is not contiguous (copied)."""
    full, y = _logits((4, 9, 333), dtype, 2)
    flat = full[:, :-1].reshape(-1, 333).contiguous()
    ref = 0.1 * torch.randn(4, 8, device=DEV, generator=_gen(3)) - 2.0
    t = y[:, 1:]
    cu = torch.arange(0, 33, 8, device=DEV)
    a = mhc_b200.preference_loss_grad(full[:, :-1], t, ref)
    b = mhc_b200.preference_loss_grad(flat, t.reshape(-1), ref.reshape(-1), cu)
    # the sums are grouped by each row's 16-byte boundaries, which differ here
    assert a.dlogits.shape == (4, 8, 333) and abs(float(a.loss) - float(b.loss)) <= 2.0 ** -20
    _check_grad(a.dlogits.reshape(-1, 333), b.dlogits.double(), 2.0 ** -22, dtype)
    wide, yw = _logits((21, 1011), dtype, 4)
    for view in (wide[:, 3:700], wide[1:, 5:6], wide[:, 7:]):
        yy = yw[-view.shape[0]:] % view.shape[1]
        old = torch.full(yy.shape, -1.0, device=DEV)
        adv = torch.randn(yy.shape, device=DEV, generator=_gen(6))
        p = mhc_b200.policy_loss_grad(view, yy, old, adv)
        q = mhc_b200.policy_loss_grad(view.contiguous(), yy, old, adv)
        assert abs(float(p.loss) - float(q.loss)) <= 1e-5 * (1 + abs(float(q.loss)))
        _check_grad(p.dlogits, q.dlogits.double(), 1e-5, dtype)
    cols = full[0].t()  # [333, 9], stride 1 on the first axis
    lp = mhc_b200.token_logprobs(cols, torch.zeros(333, dtype=torch.int64, device=DEV))
    want = torch.log_softmax(cols.double(), -1)[:, 0]
    assert (lp.double() - want).abs().max() <= 2.0 ** -22 * 40


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [37, 40000])
def test_masked_logits(dtype, V):
    """-inf and the type's lowest value on masked classes; a row of lowest
    values is uniform; a row of -inf, a NaN, a +inf and a bad target are NaN."""
    low = torch.finfo(dtype).min
    x, y = _logits((9, V), dtype, 5)
    y[:] = 1
    x[0, 2:] = -float("inf")
    x[1, 2:] = low
    x[2, :] = low
    x[3, :] = -float("inf")
    x[4, V - 1] = float("nan")
    x[5, 0] = float("inf")
    y[6], y[7] = V, -1
    x[8, 1] = -float("inf")
    lp = mhc_b200.token_logprobs(x, y)
    want = torch.log_softmax(x[:3].double(), -1)[:, 1]
    assert (lp[:3].double() - want).abs().max() <= 1e-5
    assert abs(float(lp[2]) + torch.tensor(float(V)).log().item()) <= 1e-5
    assert torch.isnan(lp[3:8]).all() and lp[8] == -float("inf")
    old, adv = torch.full((9,), -1.0, device=DEV), torch.ones(9, device=DEV)
    y[3:8] = IGN  # what is ignored is not read: no NaN reaches the loss
    r = mhc_b200.policy_loss_grad(x, y, old, adv, clip_high=10.0)
    assert torch.isfinite(r.loss) and torch.isfinite(r.dlogits).all()
    assert not r.dlogits[3:8].any() and not r.dlogits[0, 2:].any()
    y[3] = 1
    r = mhc_b200.policy_loss_grad(x, y, old, adv)
    assert torch.isnan(r.loss) and torch.isnan(r.dlogits[3]).all()
    assert torch.isfinite(r.dlogits[[0, 1, 2]]).all()


def test_nothing_counts():
    x, y = _logits((6, 100), torch.bfloat16, 1)
    y[:] = IGN
    z = torch.zeros(6, device=DEV)
    r = mhc_b200.policy_loss_grad(x, y, z, z, ref_logprobs=z, kl_coef=0.1)
    assert float(r.loss) == 0 and float(r.kl) == 0 and not r.dlogits.any()
    p = mhc_b200.preference_loss_grad(x, y, z, torch.tensor([0, 3, 6], device=DEV))
    assert abs(float(p.loss) - 0.6931472) < 1e-6 and not p.dlogits.any()
    e = x[:0]
    assert float(mhc_b200.policy_loss_grad(e, y[:0], z[:0], z[:0]).loss) == 0
    assert mhc_b200.token_logprobs(e, y[:0]).shape == (0,)
    p = mhc_b200.preference_loss_grad(e, y[:0], z[:0], torch.tensor([0, 0, 0], device=DEV))
    assert abs(float(p.loss) - 0.6931472) < 1e-6 and p.dlogits.shape == (0, 100)


def test_offsets_out_of_range_are_held():
    """Sequence offsets outside [0, T] are cut to it: nothing out of bounds is touched."""
    x, y = _logits((6, 100), torch.float32, 1)
    ref = torch.full((6,), -1.0, device=DEV)
    a = mhc_b200.preference_loss_grad(x, y, ref, torch.tensor([-5, 3, 99], device=DEV))
    b = mhc_b200.preference_loss_grad(x, y, ref, torch.tensor([0, 3, 6], device=DEV))
    assert torch.equal(a.loss, b.loss) and torch.equal(a.dlogits, b.dlogits)


def test_repeatable_and_on_another_stream():
    x, y = _logits((500, 3001), torch.bfloat16, 9)
    old, ref, adv = _policy_inputs(x, y, 4)
    cu = torch.tensor([0, 100, 250, 400, 500], device=DEV)
    first = (mhc_b200.policy_loss_grad(x, y, old, adv, ref_logprobs=ref, kl_coef=0.1),
             mhc_b200.preference_loss_grad(x, y, ref, cu))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = (mhc_b200.policy_loss_grad(x, y, old, adv, ref_logprobs=ref, kl_coef=0.1),
                 mhc_b200.preference_loss_grad(x, y, ref, cu))
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(first, again):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captured_in_a_graph():
    x, y = _logits((64, 2000), torch.bfloat16, 9)
    old, _, adv = _policy_inputs(x, y, 4)
    cu = torch.tensor([0, 30, 64], device=DEV)
    run = lambda: (mhc_b200.policy_loss_grad(x, y, old, adv),  # noqa: E731
                   mhc_b200.preference_loss_grad(x, y, old, cu))
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    x2, _ = _logits((64, 2000), torch.bfloat16, 10)
    x.copy_(x2)
    g.replay()
    want = run()
    for a, b in zip(out, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_logits_past_32_bits():
    """70000 rows of 32000: values past 2^31 are read and written where they are."""
    T, V = 70000, 32000
    x = torch.zeros(T, V, dtype=torch.bfloat16, device=DEV)
    y = torch.full((T,), IGN, dtype=torch.int64, device=DEV)
    for t in (0, 1, T - 1):
        y[t] = t % V
        x[t, t % V] = 4.0
    old, adv = torch.full((T,), -1.0, device=DEV), torch.ones(T, device=DEV)
    r = mhc_b200.policy_loss_grad(x, y, old, adv, clip_high=1e9)
    want = 4.0 - torch.log(torch.tensor(V - 1 + torch.e ** 4)).item()
    lp = r.logprobs[[0, 1, T - 1]]
    assert (lp - want).abs().max() <= 1e-5 and not r.logprobs[2:T - 1].any()
    p = torch.softmax(x[T - 1].double(), 0)
    c = -float((r.logprobs[T - 1].double() + 1).exp()) / 3
    row = r.dlogits[T - 1].double()
    want_row = -c * p
    want_row[(T - 1) % V] += c
    assert (row - want_row).abs().max() <= 2.0 ** -8 * abs(c)
    assert torch.equal(r.dlogits[T - 1, 1:5], r.dlogits[0, 1:5]) and not r.dlogits[2:T - 1:997].any()
    del x, r
    torch.cuda.empty_cache()
