"""What a step of AdamW does beside its arithmetic, and the arithmetic at the ends of the
types' ranges.  Tolerances as in test_gpu_adamw.py."""

from __future__ import annotations

import copy
import math
import pickle

import pytest
import torch
from test_gpu_adamw import HYPER, _check_p, _gen, _hash, _params, _quantise, _ref_step, _set_grads

import mhc_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("transposed", [False, True])
def test_a_step_is_an_in_place_change(bits, dtype, transposed):
    """A graph that saved a parameter cannot be differentiated once a step has changed it."""
    w = torch.randn(24, 16, device=DEV).to(dtype)
    p = torch.nn.Parameter(w.t() if transposed else w)
    opt = mhc_b200.AdamW([p], state_bits=bits, master_weights=True, **HYPER)
    loss = (p * p).sum()
    loss.backward(retain_graph=True)
    before = p._version, opt.state[p]["exp_avg"]._version
    opt.step()
    assert p._version > before[0] and opt.state[p]["exp_avg"]._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    q = torch.nn.Parameter(torch.ones(4, device=DEV))  # no gradient: left alone
    version = q._version
    mhc_b200.AdamW([q]).step()
    assert q._version == version


def test_a_step_between_two_backwards_of_a_linear_layer():
    lin = mhc_b200.FusedLinear(32, 48, activation="silu", device=DEV)
    x = torch.randn(20, 32, device=DEV).to(torch.bfloat16).requires_grad_()
    opt = mhc_b200.AdamW(lin.parameters())
    y = lin(x).float().sum()
    y.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_capture_is_refused():
    """A captured step would repeat one step's bias corrections and rounding."""
    (p,) = _params([(300,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], state_bits=8, **HYPER)
    _set_grads([p], 2)
    opt.step()
    before = p.detach().clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(g):
            opt.step()
    assert opt.state_dict()["state"][0]["step"] == 1 and torch.equal(p.detach(), before)
    opt.step()
    assert not torch.equal(p.detach(), before)


@pytest.mark.parametrize("eps", [0.0, 1e-8])
@pytest.mark.parametrize("size", [1e-21, 1e-20, 1e-19, 1e-18, 1e-15])
def test_8_bit_state_of_small_gradients(eps, size):
    """v down among fp32's subnormal numbers: codes as the formulas give them, and a
    parameter that moves by what m and the root of v come to."""
    h = dict(HYPER, eps=eps)
    (p,) = _params([(600,)], torch.float32, 3)
    opt = mhc_b200.AdamW([p], state_bits=8, seed=7, **h)
    buf = opt.state_buffers()
    b1, b2 = h["betas"]
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    for t in range(1, 4):
        sign = torch.where(torch.arange(600, device=DEV) % 3 == 0, -1.0, 1.0)
        p.grad = size * sign * (1 + torch.arange(600, device=DEV) % 7 / 8)
        wide = lambda k: buf[k].float().view(-1, 256) * buf[k + "_scale"][:, None]  # noqa: E731
        g = torch.zeros(768, device=DEV)
        g[:600] = p.grad
        g = g.view(-1, 256)
        m = wide("exp_avg") * f32(b1) + g * f32(1 - b1)
        r = wide("exp_avg_sq_root")
        r = (r * r * f32(b2) + g * g * f32(1 - b2)).sqrt()
        base = p.detach().double()
        opt.step()
        k = _hash(torch.arange(768, device=DEV), (7 * 0x9E3779B9 + t * 0x85A308D3) & 0xFFFFFFFF)
        for key, x, u, floor in (("exp_avg", m, k & 0xFFFF, False),
                                 ("exp_avg_sq_root", r, k >> 16, True)):
            q, scale = _quantise(x, u, floor)
            assert torch.equal(buf[key + "_scale"], scale), key
            assert torch.equal(buf[key].float().view(-1, 256), q), key
        mm, rr = (x.view(-1)[:600].double() for x in (m, r))
        u = h["lr"] / (1 - b1 ** t) * mm / (rr / math.sqrt(1 - b2 ** t) + eps)
        _check_p(p, base * (1 - h["lr"] * h["weight_decay"]) - u, u)


@pytest.mark.parametrize("size", [2e19, 3e38])
def test_a_gradient_whose_square_overflows(size):
    """v is infinite: the element stays where it is but for the decay, with 8-bit state as
    with 32."""
    ps = [torch.nn.Parameter(torch.ones(512, device=DEV)) for _ in range(2)]
    opts = [mhc_b200.AdamW([p], state_bits=b, lr=0.5, weight_decay=0.25) for p, b in zip(ps, (32, 8))]
    rest = torch.arange(512, device=DEV) != 300
    for t in range(20):
        for p, opt in zip(ps, opts):
            p.grad = torch.ones_like(p)
            if t == 0:
                p.grad[300] = size
            opt.step()
            assert torch.isfinite(p).all()
            if t == 0:  # a decay of 1/8 and, elsewhere, a first step of lr
                assert float(p.detach()[300]) == 0.875
                assert ((p.detach()[rest] - 0.375).abs() <= 2.0 ** -20).all()
        assert torch.equal(ps[0].detach()[300], ps[1].detach()[300])
    # a gradient that is itself infinite is NaN for good
    (p,) = ps[1:]
    p.grad[300] = float("inf")
    for _ in range(3):
        opts[1].step()
        p.grad = torch.ones_like(p)
        assert torch.isnan(p[300]) and torch.isfinite(p[:256]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_new_values_of_a_parameter_with_a_master(bits, dtype):
    """Values written into the parameter between steps are what the next step starts from;
    elements that were left alone, or given the value that they had, keep their master's
    digits."""
    shapes = [(33, 50), (7,)]
    params = _params(shapes, dtype, 1)
    opt = mhc_b200.AdamW(params, state_bits=bits, master_weights=True, **HYPER)
    _set_grads(params, 2)
    opt.step()
    fresh = torch.randn(33, 50, device=DEV, generator=_gen(4)).to(dtype)
    fresh[0, :10] = params[0].detach()[0, :10]
    with torch.no_grad():
        params[0][:20].copy_(fresh[:20])
        params[1].data = torch.full_like(params[1], 3.0)
    start = [opt.state[p]["master"].double() for p in params]
    kept = params[0].detach()[20:].clone()
    assert torch.equal(start[0][20:].to(dtype), kept) and not torch.equal(start[0][20:], kept.double())
    given = start[0][:20].to(dtype) != fresh[:20]
    assert not given[0, :10].any() and given.sum() > 900
    start[0][:20][given], start[1][:] = fresh[:20][given].double(), 3.0
    own = [opt.state[p] for p in params]
    if bits == 32:
        m = [s["exp_avg"].double() for s in own]
        v = [s["exp_avg_sq"].double() for s in own]
    else:
        b = opt.state_buffers()
        wide = lambda k: (b[k].float().view(-1, 256) * b[k + "_scale"][:, None]).view(-1)  # noqa: E731
        cut = lambda x: [x[:1650].view(33, 50).double(), x[1792:1799].double()]  # noqa: E731
        m, v = cut(wide("exp_avg")), [r.square() for r in cut(wide("exp_avg_sq_root"))]
    _set_grads(params, 3)
    opt.step()
    for p, x, mm, vv, s in zip(params, start, m, v, own):
        want, _, _, u = _ref_step(x, p.grad.double(), mm, vv, 2, HYPER)
        _check_p(p, want, u)
        tol = 2.0 ** -22 * want.abs() + 2.0 ** -19 * u.abs()
        assert ((s["master"].double() - want).abs() <= tol).all()


def test_grad_scale_is_one_number():
    (p,) = _params([(30,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    _set_grads([p], 2)
    for bad in (torch.ones(0, device=DEV), torch.ones(2, device=DEV)):
        with pytest.raises(ValueError, match="grad_scale"):
            opt.step(grad_scale=bad)
    with pytest.raises(ValueError, match="grad_scale"):
        opt.step(grad_scale=0.5)
    assert opt.state_dict()["state"][0]["step"] == 0
    opt.step(grad_scale=torch.ones(1, dtype=torch.float64, device=DEV))


def test_a_step_that_raises_does_not_count():
    (p,) = _params([(30,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    _set_grads([p], 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step(grad_scale=torch.ones(1))
    assert opt.state_dict()["state"][0]["step"] == 0


def test_parameters_that_share_memory_are_refused():
    """Blocks of one launch would write the same values."""
    p = torch.nn.Parameter(torch.zeros(10, device=DEV))
    with pytest.warns(UserWarning, match="duplicate"), pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([p, p])
    flat = torch.zeros(100, device=DEV)
    part = lambda a, b: torch.nn.Parameter(flat[a:b])  # noqa: E731
    with pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([part(50, 100), part(0, 10), part(9, 20)])
    with pytest.raises(ValueError, match="share memory"):
        mhc_b200.AdamW([part(0, 100), part(10, 20), torch.nn.Parameter(flat[30:30])])
    mhc_b200.AdamW([part(50, 100), part(10, 50), part(0, 10), torch.nn.Parameter(flat[30:30])])


def test_8_bit_state_of_another_layout_is_refused():
    """Its scales go by blocks of memory, which hold other elements there."""
    w = torch.randn(40, 30, device=DEV)
    a, b = torch.nn.Parameter(w.t()), torch.nn.Parameter(w.t().contiguous())
    for bits in (8, 32):
        oa, ob = (mhc_b200.AdamW([x], state_bits=bits) for x in (a, b))
        a.grad = torch.randn(30, 40, device=DEV)
        oa.step()
        saved = oa.state_dict()
        if bits == 8:
            with pytest.raises(ValueError, match="laid out"):
                ob.load_state_dict(saved)
            assert ob.state_dict()["state"][0]["step"] == 0
        else:
            ob.load_state_dict(saved)
            assert torch.equal(ob.state[b]["exp_avg"], oa.state[a]["exp_avg"])
    # an axis of one element has any stride
    c = torch.nn.Parameter(torch.zeros(1, 8, device=DEV).t())
    d = torch.nn.Parameter(torch.zeros(8, 1, device=DEV))
    oc, od = (mhc_b200.AdamW([x], state_bits=8) for x in (c, d))
    od.load_state_dict(oc.state_dict())


def test_state_hooks_and_walks():
    params = _params([(30,), (4, 4)], torch.float32, 1)
    opt = mhc_b200.AdamW(params, **HYPER)
    assert len(opt.state) == 2 and list(opt.state) == params and params[0] in opt.state
    assert [s["exp_avg"].shape for s in opt.state.values()] == [p.shape for p in params]
    assert all(s is opt.state[p] for p, s in opt.state.items())
    _set_grads(params, 2)
    opt.step()
    seen = []
    opt.register_state_dict_pre_hook(lambda o: seen.append("pre"))

    def post(o, d):
        seen.append("post")
        d["note"] = 5

    opt.register_state_dict_post_hook(post)
    opt.register_state_dict_post_hook(lambda o, d: {**d, "other": 6})
    saved = opt.state_dict()
    assert seen == ["pre", "post"] and saved["note"] == 5 and saved["other"] == 6
    new = mhc_b200.AdamW(_params([(30,), (4, 4)], torch.float32, 9))

    def before(o, d):
        seen.append("before")
        d = {**d, "param_groups": [{**g, "lr": 0.125} for g in d["param_groups"]]}
        return d

    new.register_load_state_dict_pre_hook(before)
    new.register_load_state_dict_post_hook(lambda o: seen.append(("after", o.param_groups[0]["lr"])))
    new.load_state_dict(saved)
    assert seen == ["pre", "post", "before", ("after", 0.125)]
    assert saved["param_groups"][0]["lr"] == HYPER["lr"]
    for a, b in zip(opt.state.values(), new.state.values()):
        assert torch.equal(a["exp_avg"], b["exp_avg"])


def test_a_copy_with_a_scheduler_steps_its_own_parameters():
    (p,) = _params([(300,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda n: 0.5 ** n)
    _set_grads([p], 2)
    opt.step()
    schedule.step()
    twin = copy.deepcopy(opt)
    (q,) = twin.param_groups[0]["params"]
    q.grad = p.grad.clone()
    before = p.detach().clone()
    twin.step()
    assert torch.equal(p.detach(), before) and not torch.equal(q.detach(), before)
    opt.step()
    assert torch.equal(p.detach(), q.detach())


@pytest.mark.parametrize("bits", [32, 8])
def test_pickled(bits):
    params = _params([(50, 7), (4,)], torch.bfloat16, 1) + _params([(9,)], torch.float32, 2)
    opt = mhc_b200.AdamW([{"params": params[:2]}, {"params": params[2:], "lr": 0.5}],
                         state_bits=bits, master_weights=True, seed=3, **HYPER)
    torch.optim.lr_scheduler.LambdaLR(opt, lambda n: 1.0)
    for t in range(2):
        _set_grads(params, t)
        opt.step()
    twin = pickle.loads(pickle.dumps(opt))
    own = [p for g in twin.param_groups for p in g["params"]]
    assert all(torch.equal(p, q) and p is not q for p, q in zip(params, own))
    assert twin.state_bits == bits and twin.seed == 3 and twin.param_groups[1]["lr"] == 0.5
    for t in range(2, 4):
        for ps, o in ((params, opt), (own, twin)):
            _set_grads(ps, t)
            o.step()
    assert all(torch.equal(p, q) for p, q in zip(params, own))
    for k in (0, 1):
        for a, b in zip(opt.state_buffers(k).values(), twin.state_buffers(k).values()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
