"""AdamW over many tensors against the formulas in float64.

Tolerances, from the arithmetic and before any run: m and v are two products
and a sum in fp32, |error| <= 2^-22 (|m| + |g|) and 2^-22 (v + g^2).  The
update is a quotient of those (square root and division to 2 units of 2^-23):
2^-19 of its size before b1 m and (1 - b1) g cancel, plus the parameter's own rounding: half a unit of its type, and
2^-23 of it for the decay.  8-bit codes are compared bit for bit with the
formulas in fp32."""

from __future__ import annotations

import math

import pytest
import torch

import mhc_b200

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _params(shapes, dtype, seed):
    g = _gen(seed)
    return [torch.nn.Parameter(torch.randn(s, device=DEV, generator=g).to(dtype)) for s in shapes]


def _set_grads(params, seed):
    g = _gen(seed)
    for p in params:
        p.grad = (0.1 * torch.randn(p.shape, device=DEV, generator=g)).to(p.dtype)


def _ref_step(p, g, m, v, t, h):
    """One update in float64: (p, m, v, the update's size were m's two terms of one sign)."""
    b1, b2 = h["betas"]
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    per = h["lr"] / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + h["eps"])
    return p * (1 - h["lr"] * h["weight_decay"]) - m * per, m, v, size * per


def _check_p(p, want, u):
    tol = HALF_ULP[p.dtype] * want.abs() + TINY[p.dtype] + 2.0 ** -22 * want.abs() + 2.0 ** -19 * u.abs()
    bad = (p.detach().double() - want).abs() > tol
    assert not bad.any(), ((p.detach().double() - want).abs() / tol.clamp(min=1e-300)).max()


SHAPES = [(1,), (4,), (4, 4), (7, 9), (256,), (257,), (2048,), (2049,), (3, 0), (33, 1000), (5, 4097)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("master", [False, True])
def test_32_bit_state(dtype, master):
    params = _params(SHAPES, dtype, 1)
    opt = mhc_b200.AdamW(params, master_weights=master, **HYPER)
    m = [torch.zeros(p.shape, dtype=torch.float64, device=DEV) for p in params]
    v = [torch.zeros_like(x) for x in m]
    for t in range(1, 4):
        _set_grads(params, 10 + t)
        # each step from the kernel's own state: one step's error at a time
        own = [opt.state[p] for p in params]
        m = [s["exp_avg"].double() for s in own]
        v = [s["exp_avg_sq"].double() for s in own]
        base = [(s["master"] if "master" in s else p.detach()).double() for p, s in zip(params, own)]
        opt.step()
        for p, s, b, mm, vv in zip(params, own, base, m, v):
            g = p.grad.double()
            want, m2, v2, u = _ref_step(b, g, mm, vv, t, HYPER)
            _check_p(p, want, u)
            assert ((s["exp_avg"].double() - m2).abs() <= 2.0 ** -22 * (mm.abs() + g.abs())).all()
            assert ((s["exp_avg_sq"].double() - v2).abs() <= 2.0 ** -22 * (vv + g * g)).all()
            if "master" in s:
                tol = 2.0 ** -22 * want.abs() + 2.0 ** -19 * u.abs()
                assert ((s["master"].double() - want).abs() <= tol).all()
                assert torch.equal(s["master"].to(dtype), p.detach())


def _scale_of(x):
    """Least power of two s >= 2^-126 with max |x| <= 448 s, per block, by logarithm."""
    top = x.abs().amax(dim=1).double()
    e = torch.where(top > 0, (top / 448).log2().ceil(), torch.full_like(top, -126.0))
    return torch.pow(2.0, e.clamp(min=-126)).float()


def _hash(pos, key):
    m = 0xFFFFFFFF
    h = ((pos * 0x9E3779B9) & m) ^ key
    h = ((h ^ (h >> 16)) * 0x6A09E667) & m
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & m
    return h ^ (h >> 16)


def _quantise(x, u16, floor):
    """(values on the e4m3 grid in units of the scale, scale), x [blocks, 256] fp32."""
    scale = _scale_of(x)
    y0 = (x / scale[:, None]).abs()
    y = torch.where(y0 < 2.0 ** -6, (y0 + 2.0 ** -6) - 2.0 ** -6, y0)  # there it counts to 2^-29
    # spacing: 2^-9 below 2^-6, else 2^(exponent - 3)
    step = torch.pow(2.0, (torch.floor(torch.log2(y.clamp(min=2.0 ** -6).double())) - 3)).float()
    low = torch.floor(y / step) * step
    part = (y - low) / step  # in [0, 1), exact
    # the same 20 bits of a fraction, and of 16 bits of chance above them
    up = torch.floor(part * 2 ** 20) + u16.view_as(x).float() * 16 >= 2 ** 20
    q = torch.where(up, low + step, low)
    if floor:
        q = torch.where((y0 > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return torch.where(x < 0, -q, q), scale


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("master", [False, True])
def test_8_bit_state(dtype, master):
    shapes = [(3,), (256,), (700,), (41, 100)]
    params = _params(shapes, dtype, 3)
    opt = mhc_b200.AdamW(params, state_bits=8, master_weights=master, seed=7, **HYPER)
    buf = opt.state_buffers()
    b1, b2 = HYPER["betas"]
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    for t in range(1, 6):
        _set_grads(params, 20 + t)
        if t == 2:
            params[1].grad.zero_()
            params[2].grad[:300] *= 1e-6  # far below the block's largest
        n = buf["exp_avg"].numel()
        wide = lambda k: buf[k].float().view(-1, 256) * buf[k + "_scale"][:, None]  # noqa: E731
        g = torch.zeros(n, device=DEV)
        o = 0
        for p in params:
            g[o:o + p.numel()] = p.grad.float().view(-1)
            o += -(-p.numel() // 256) * 256
        g = g.view(-1, 256)
        m = wide("exp_avg") * f32(b1) + g * f32(1 - b1)
        r = wide("exp_avg_sq_root")
        r = (r * r * f32(b2) + g * g * f32(1 - b2)).sqrt()
        base = [(opt.state[p]["master"] if "master" in opt.state[p] else p.detach()).double()
                for p in params]
        opt.step()
        h = _hash(torch.arange(n, device=DEV), (7 * 0x9E3779B9 + t * 0x85A308D3) & 0xFFFFFFFF)
        for key, x, u, floor in (("exp_avg", m, h & 0xFFFF, False),
                                 ("exp_avg_sq_root", r, h >> 16, True)):
            q, scale = _quantise(x, u, floor)
            assert torch.equal(buf[key + "_scale"], scale), key
            assert torch.equal(buf[key].float().view(-1, 256), q), key
        o = 0
        for p, b in zip(params, base):
            mm, rr = (x.view(-1)[o:o + p.numel()].view(p.shape).double() for x in (m, r))
            u = HYPER["lr"] / (1 - b1 ** t) * mm / (rr / math.sqrt(1 - b2 ** t) + HYPER["eps"])
            _check_p(p, b * (1 - HYPER["lr"] * HYPER["weight_decay"]) - u, u)
            o += -(-p.numel() // 256) * 256


def test_8_bit_moments_keep_their_mean():
    """A constant |g| = 1: v goes to 1 - b2^t although a step moves it by a tenth of
    a code.  4096 elements: the mean's own spread is far below the 4 % that the
    rounding of a square root adds to a square."""
    p = torch.nn.Parameter(torch.zeros(4096, device=DEV))
    opt = mhc_b200.AdamW([p], lr=0.0, betas=(0.9, 0.99), state_bits=8)
    p.grad = torch.where(torch.arange(4096, device=DEV) % 2 == 0, 1.0, -1.0)
    for t in range(1, 301):
        opt.step()
    b = opt.state_buffers()
    r = b["exp_avg_sq_root"].float().view(-1, 256) * b["exp_avg_sq_root_scale"][:, None]
    m = b["exp_avg"].float().view(-1, 256) * b["exp_avg_scale"][:, None]
    assert abs(float(r.square().mean()) / (1 - 0.99 ** 300) - 1) < 0.06
    assert abs(float((m * p.grad.view(-1, 256)).mean()) - 1) < 0.02


def test_moments_of_one_follow_32_bits():
    """8-bit and 32-bit runs of the same gradients end near each other: a code is off by
    3 to 6 % (half its spacing), the moments' memory adds up two or three of those."""
    a = _params([(64, 64), (300,)], torch.float32, 5)
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa, ob = mhc_b200.AdamW(a, **HYPER), mhc_b200.AdamW(b, state_bits=8, **HYPER)
    start = [p.detach().clone() for p in a]
    for t in range(30):
        _set_grads(a, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        oa.step(), ob.step()
    for p, q, s in zip(a, b, start):
        moved = (p - s).double().norm()
        assert (p - q).double().norm() < 0.25 * moved


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts_and_alignment(bits):
    """Transposed parameters, views at odd offsets, gradients laid out otherwise: the
    same updates as plain copies of them."""
    flat = torch.randn(5000, device=DEV, generator=_gen(1))
    views = [flat[1:1 + 999], flat[1003:1003 + 64 * 33].view(64, 33).t(), flat[4001:4002]]
    plain = [v.clone(memory_format=torch.contiguous_format) for v in views]
    grads = [torch.randn(v.shape, device=DEV, generator=_gen(i)) for i, v in enumerate(views)]
    a = [torch.nn.Parameter(v) for v in views]
    b = [torch.nn.Parameter(v) for v in plain]
    assert a[1].stride() == (1, 33)
    # one parameter at a time, so that both see the same places in the state
    for p, q, g in zip(a, b, grads):
        oa, ob = (mhc_b200.AdamW([x], state_bits=bits, **HYPER) for x in (p, q))
        for _ in range(2):
            p.grad, q.grad = g, g.clone()
            oa.step(), ob.step()
        if bits == 32:
            assert torch.equal(p.detach(), q.detach())
            assert torch.equal(oa.state[p]["exp_avg"], ob.state[q]["exp_avg"])
        else:  # the dither goes by the place in memory, which a transpose changes
            assert (p - q).abs().max() < 0.3 * HYPER["lr"]
    assert torch.equal(flat[1000:1003], torch.randn(5000, device=DEV, generator=_gen(1))[1000:1003])


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_missing_gradients(bits):
    """More tensors than one launch takes, types mixed in a group, some without gradients."""
    shapes = [(4,), (4, 4), (64,)] * 400
    params = _params(shapes, torch.float32, 1) + _params([(8, 8), (300,)], torch.bfloat16, 2)
    opt = mhc_b200.AdamW([{"params": params[:600]}, {"params": params[600:], "lr": 2e-2}],
                         state_bits=bits, **HYPER)
    with pytest.raises(ValueError, match="dtype"):
        opt.state_buffers(1)
    assert opt.state_buffers(1, torch.bfloat16)["exp_avg"].numel() == 256 + 512
    _set_grads(params, 9)
    for p in params[::7]:
        p.grad = None
    before = [p.detach().clone() for p in params]
    opt.step()
    lrs = [HYPER["lr"]] * 600 + [2e-2] * (len(params) - 600)
    steps = [0] * len(params)
    for i, (p, b, lr) in enumerate(zip(params, before, lrs)):
        if p.grad is None:
            assert torch.equal(p.detach(), b)
            continue
        steps[i] = 1
        z = torch.zeros_like(b, dtype=torch.float64)
        want, _, _, u = _ref_step(b.double(), p.grad.double(), z, z, 1, dict(HYPER, lr=lr))
        _check_p(p, want, u)
    # now all have one: each with its own count of steps
    for p in params:
        if p.grad is None:
            p.grad = torch.ones_like(p)
    before = [p.detach().clone() for p in params]
    opt.step()
    for i in range(0, len(params), 7):
        z = torch.zeros_like(before[i], dtype=torch.float64)
        want, _, _, u = _ref_step(before[i].double(), z + 1, z, z, 1, dict(HYPER, lr=lrs[i]))
        _check_p(params[i], want, u)
    assert opt.state_dict()["state"][0]["step"] == 1 and opt.state_dict()["state"][1]["step"] == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_save_and_resume(bits):
    a = _params([(50, 7), (4,)], torch.bfloat16, 1)
    oa = mhc_b200.AdamW(a, state_bits=bits, master_weights=True, seed=3, **HYPER)
    for t in range(3):
        _set_grads(a, t)
        oa.step()
    saved = oa.state_dict()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = mhc_b200.AdamW(b, state_bits=bits, master_weights=True, lr=1.0)
    ob.load_state_dict(saved)
    for t in range(3, 5):
        _set_grads(a, t)
        _set_grads(b, t)
        oa.step(), ob.step()
    assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(a, b))
    for k, v in oa.state_buffers().items():
        u = ob.state_buffers()[k]
        assert torch.equal(v.view(torch.uint8), u.view(torch.uint8)), k
    with pytest.raises(ValueError, match="bits"):
        mhc_b200.AdamW(b, state_bits=40 - bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="groups"):
        mhc_b200.AdamW(b[:1], state_bits=bits).load_state_dict(saved)
    with pytest.raises(ValueError, match="fit"):
        mhc_b200.AdamW(b[::-1], state_bits=bits, master_weights=True).load_state_dict(saved)


def test_grad_scale_closure_and_streams():
    p, q = _params([(1000,)], torch.float32, 1) + _params([(1000,)], torch.float32, 1)
    a, b = mhc_b200.AdamW([p], **HYPER), mhc_b200.AdamW([q], **HYPER)
    g = torch.randn(1000, device=DEV, generator=_gen(2))
    p.grad, q.grad = g * 4, g.clone()
    out = a.step(lambda: 5.0, grad_scale=torch.tensor(0.25, device=DEV))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step()
    torch.cuda.current_stream().wait_stream(s)
    assert out == 5.0 and torch.equal(p.detach(), q.detach())


def test_grad_scaler_skips_what_overflowed():
    (p,) = _params([(500,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    scaler = torch.amp.GradScaler("cuda", init_scale=8.0)
    before = p.detach().clone()
    scaler.scale((p * float("inf")).sum()).backward()
    scaler.step(opt)
    scaler.update()
    assert torch.equal(p.detach(), before) and opt.state_dict()["state"][0]["step"] == 0
    opt.zero_grad()
    scaler.scale((p * 2).sum()).backward()
    scaler.step(opt)
    z = torch.zeros(500, dtype=torch.float64, device=DEV)
    want, _, _, u = _ref_step(before.double(), z + 2, z, z, 1, HYPER)
    _check_p(p, want, u)


@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_gradients_stay_where_they_are(bits):
    p = torch.nn.Parameter(torch.ones(1024, device=DEV))
    opt = mhc_b200.AdamW([p], state_bits=bits, **HYPER)
    p.grad = torch.ones_like(p)
    p.grad[300] = float("nan")
    opt.step()
    assert torch.isnan(p[300]) and torch.isfinite(p[torch.arange(1024, device=DEV) != 300]).all()
    p.grad = torch.ones_like(p)
    opt.step()
    ok = torch.ones(1024, dtype=torch.bool, device=DEV)
    ok[256:512] = bits == 32  # 8 bits: its block of 256 is spoilt
    ok[300] = False
    assert torch.isfinite(p[ok]).all() and torch.isnan(p[300])


def test_a_tensor_past_32_bits():
    """2^31 + 300 elements: what lies past 2^31 is updated as what lies before."""
    n = 2 ** 31 + 300
    p = torch.nn.Parameter(torch.ones(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.full((n,), 0.5, dtype=torch.bfloat16, device=DEV)
    p.grad[-1] = -0.5
    opt = mhc_b200.AdamW([p], state_bits=8, lr=0.25, weight_decay=0.0)
    opt.step()
    assert float(p[0]) == 0.75 and float(p[2 ** 31 + 298]) == 0.75 and float(p[-1]) == 1.25
    assert bool((p[::4099] == 0.75).all())
    del p, opt
    torch.cuda.empty_cache()


def test_repeatable_and_captured():
    runs = []
    for k in range(2):
        params = _params([(77, 100), (5,)], torch.bfloat16, 1)
        opt = mhc_b200.AdamW(params, state_bits=8, seed=5, **HYPER)
        for t in range(3):
            _set_grads(params, t)
            opt.step()
        runs.append([p.detach().clone() for p in params] +
                    [b.view(torch.uint8).clone() for b in opt.state_buffers().values()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_parameters_given_other_memory():
    """New memory of the same form is followed; another type or size is refused."""
    (p,) = _params([(300,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    _set_grads([p], 2)
    opt.step()
    p.data = p.data.clone()
    before = p.detach().clone()
    opt.step()
    assert not torch.equal(p.detach(), before)
    p.data = p.data.half()
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="another type"):
        opt.step()
    p.grad = None
    p.data = torch.zeros(200, device=DEV)
    p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="another type"):
        opt.step()


def test_copied_optimizer_steps_its_own_parameters():
    import copy

    (p,) = _params([(300,)], torch.float32, 1)
    opt = mhc_b200.AdamW([p], **HYPER)
    _set_grads([p], 2)
    opt.step()
    twin = copy.deepcopy(opt)
    (q,) = twin.param_groups[0]["params"]
    q.grad = p.grad.clone()
    before = p.detach().clone()
    twin.step()
    assert torch.equal(p.detach(), before) and not torch.equal(q.detach(), before)
    opt.step()
    assert torch.equal(p.detach(), q.detach())
