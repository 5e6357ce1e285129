"""Cases that measure the fine-tuning operators: the preference and policy losses on logits, the
AdamW step over many tensors and the linear layer with its epilogue, each with its gradient.

A case is a dict of plain values.  `prepare` makes what a training program has in hand before the
call, `run` makes one pass (the plain form in torch, or the framework's kernels where `own` is
true) and `exact` gives the outputs in 64 bits.  Sizes: the patched decoder of the examples (4096
channels, 11008 in its MLP, 32000 tokens, 4 streams, 32 layers), the tests' small vocabulary of
512, and odd and ragged ones around them.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100
BLOCK = 256  # elements that share a scale in the 8-bit optimizer state
BETA, LR, B1, B2, EPS, DECAY, STEP = 0.1, 1e-3, 0.9, 0.95, 1e-8, 0.1, 100
CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "mhc-mlx_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mhc_b200

    return mhc_b200


# ------------------------------------------------------------------- cases --
def listed():
    return [
        # a unit test's or a toy model's step: launch latency is all there is
        dict(name="preference small", op="preference", pairs=2, tokens=16, vocab=512,
             dtype="bf16", smoothing=0.0, scale=1.0),
        # eight pairs of answers from the decoder of the examples, lengths ragged, prompts masked
        dict(name="preference bf16", op="preference", pairs=8, tokens=512, vocab=32000,
             dtype="bf16", smoothing=0.0, scale=1.0),
        # 32-bit logits of a vocabulary with one added token: rows that no vector load fits
        dict(name="preference f32 odd", op="preference", pairs=3, tokens=101, vocab=32001,
             dtype="f32", smoothing=0.1, scale=1.0),
        # the tail of a micro-batch: a few tokens of a long vocabulary
        dict(name="policy few tokens", op="policy", tokens=7, vocab=131072, dtype="bf16",
             kl=0.05, masked=0.0, scale=1.0),
        # a policy-gradient micro-batch of the decoder of the examples
        dict(name="policy bf16", op="policy", tokens=8192, vocab=32000, dtype="bf16", kl=0.05,
             masked=0.3, scale=1.0),
        # mixed-precision training with a loss scale, odd rows
        dict(name="policy f16 odd", op="policy", tokens=1000, vocab=50001, dtype="f16", kl=0.0,
             masked=0.2, scale=65536.0),
        # the mHC parameters of the patched decoder: 512 small tensors
        dict(name="adamw streams", op="adamw", layers=32, streams=4, channels=1024, dims=0, mlp=0,
             dtype="f32", bits=32, master=False),
        # one decoder block's weights with 32-bit states
        dict(name="adamw block 32", op="adamw", layers=0, streams=4, channels=1024, dims=4096,
             mlp=11008, dtype="bf16", bits=32, master=False),
        # the same with 8-bit states
        dict(name="adamw block 8", op="adamw", layers=0, streams=4, channels=1024, dims=4096,
             mlp=11008, dtype="bf16", bits=8, master=False),
        # one token through an output projection that adds the residual stream
        dict(name="linear one token", op="linear", tokens=1, ins=4096, outs=4096, dtype="bf16",
             act="none", bias=True, residual=True, train=False),
        # the MLP's input projection in training
        dict(name="linear train", op="linear", tokens=8192, ins=4096, outs=11008, dtype="bf16",
             act="silu", bias=True, residual=False, train=True),
        # sizes that fit no tile
        dict(name="linear odd", op="linear", tokens=777, ins=1001, outs=1500, dtype="f16",
             act="gelu", bias=True, residual=True, train=True),
    ]


MOST_LOGITS = 8192 * 32000
MOST_PRODUCTS = 8192 * 4096 * 11008


def _log(rng, low, high):
    """A whole number between low and high, even over the logarithm; one in two is odd."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v % 2 == 0 and v > low:
        v -= 1
    v = max(low, min(high, v))
    return v - 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["preference", "policy", "adamw", "linear"])
    if op == "preference":
        vocab = _log(rng, 512, 131072)
        pairs = rng.randint(1, 16)
        most = max(4, min(512, MOST_LOGITS // (2 * pairs * vocab)))
        return dict(op=op, pairs=pairs, tokens=_log(rng, 4, most), vocab=vocab,
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    smoothing=rng.choice([0.0, 0.1]), scale=rng.choice([1.0, 1024.0]))
    if op == "policy":
        vocab = _log(rng, 512, 131072)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = min(8192, MOST_LOGITS // vocab // (2 if dtype == "f32" else 1))
        return dict(op=op, tokens=_log(rng, 1, most), vocab=vocab, dtype=dtype,
                    kl=rng.choice([0.0, 0.05]), masked=rng.choice([0.0, 0.3]),
                    scale=1024.0 if dtype == "f16" else 1.0)
    if op == "adamw":
        streams = rng.random() < 0.4
        dtype = "f32" if streams else rng.choice(["bf16", "bf16", "f16", "f32"])
        bits = rng.choice([32, 8])
        dims = 0 if streams else _log(rng, 64, 2048)
        return dict(op=op, layers=rng.randint(1, 48) if streams else 0,
                    streams=rng.choice([1, 2, 4, 8]), channels=_log(rng, 64, 4096), dims=dims,
                    mlp=0 if streams else 3 * dims - 1, dtype=dtype, bits=bits,
                    master=dtype != "f32" and rng.random() < 0.4)
    tokens, ins = _log(rng, 1, 8192), _log(rng, 64, 11008)
    outs = _log(rng, 64, max(64, min(11008, MOST_PRODUCTS // (tokens * ins))))
    return dict(op=op, tokens=tokens, ins=ins, outs=outs, dtype=rng.choice(["bf16", "f16"]),
                act=rng.choice(["none", "relu", "silu", "gelu"]), bias=rng.random() < 0.7,
                residual=rng.random() < 0.5, train=rng.random() < 0.6)


# ------------------------------------------------------------------ inputs --
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _lengths(pairs, tokens):
    """Ragged lengths of 2 * pairs sequences, 2 * pairs * tokens rows in all."""
    w = [0.4 + 1.2 * ((7 * i * i + 3 * i) % 11) / 10 for i in range(2 * pairs)]
    total, out = 2 * pairs * tokens, []
    for i in range(2 * pairs - 1):
        out.append(max(1, int(total * w[i] / sum(w))))
    return out + [max(0, total - sum(out))]


def _logits(g, rows, vocab, dtype):
    """Logits of a model that has learnt something: the target stands out."""
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    x = _randn(g, rows, vocab).mul_(2.0)
    x[torch.arange(rows, device="cuda"), targets] += 9.0
    logp = x.gather(1, targets[:, None])[:, 0] - torch.logsumexp(x, dim=1)
    return x.to(dtype), targets, logp


def _prepare_preference(case, g):
    dtype, pairs = DTYPES[case["dtype"]], case["pairs"]
    lengths = _lengths(pairs, case["tokens"])
    rows = sum(lengths)
    logits, targets, logp = _logits(g, rows, case["vocab"], dtype)
    # a fifth of each sequence is the prompt; the reference model is a little apart
    starts = [sum(lengths[:i]) for i in range(2 * pairs + 1)]
    pos = torch.arange(rows, device="cuda")
    prompt = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for s, n in zip(starts, lengths):
        prompt |= (pos >= s) & (pos < s + n // 5)
    targets = torch.where(prompt, torch.full_like(targets, IGNORE), targets)
    ref = logp + 0.1 * _randn(g, rows)
    return dict(logits=logits, targets=targets, ref=ref,
                cu_seqlens=torch.tensor(starts, dtype=torch.int32, device="cuda"))


def _prepare_policy(case, g):
    rows = case["tokens"]
    logits, targets, logp = _logits(g, rows, case["vocab"], DTYPES[case["dtype"]])
    advantages = 0.3 + _randn(g, rows)
    old = logp + 0.3 * _randn(g, rows)
    # keep clear of the two kinks of the clip, where the gradient jumps
    ratio = logp - old
    for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        old = torch.where((ratio - edge).abs() < 0.02, old - 0.05, old)
        ratio = logp - old
    ref = logp + 0.3 * _randn(g, rows)
    drop = torch.rand(rows, generator=g, device="cuda") < case["masked"]
    drop[0] = False
    targets = torch.where(drop, torch.full_like(targets, IGNORE), targets)
    return dict(logits=logits, targets=targets, old=old, ref=ref, advantages=advantages)


def _shapes(case):
    if case["layers"]:
        n, c = case["streams"], case["channels"]
        return [(n,), (n,), (n, n), (c,)] * (4 * case["layers"])
    d, m = case["dims"], case["mlp"]
    return [(d, d)] * 4 + [(m, d), (d, m), (m, d), (d,), (d,)]


def _power_of_two_scale(top):
    """The least power of two s (2^-126 at least) with top <= 448 s, by the bits of `top`."""
    e = ((top.view(torch.int32) + 0x1FFFFF) >> 23) - 8
    return (e.clamp(min=1) << 23).view(torch.float32)


def _prepare_adamw(case, g):
    shapes, dtype = _shapes(case), DTYPES[case["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    offsets = [0]
    for n in sizes:
        offsets.append(offsets[-1] + -(-n // BLOCK) * BLOCK)
    total = offsets[-1]
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    for o, n in zip(offsets, sizes):
        used[o:o + n] = True
    master = (0.05 * _randn(g, total)).mul_(used)
    flat = master.to(dtype)
    grad = (1e-3 * _randn(g, total)).mul_(used).to(dtype)
    m = (3e-4 * _randn(g, total)).mul_(used)
    root = (1e-3 * (0.3 + torch.rand(total, generator=g, device="cuda"))).mul_(used)
    s = dict(flat=flat, grad=grad, step=STEP,
             padded=[b - a for a, b in zip(offsets, offsets[1:])])
    if case["master"]:
        s["master"] = master
    if case["bits"] == 8:
        for key, x in (("exp_avg", m), ("exp_avg_sq_root", root)):
            b = x.view(-1, BLOCK)
            scale = _power_of_two_scale(b.abs().amax(dim=1))
            s[key] = (b / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            s[key + "_scale"] = scale
    else:
        s["exp_avg"], s["exp_avg_sq"] = m, root.square_()
    views = lambda x: [x[o:o + n].view(sh) for o, n, sh in zip(offsets, sizes, shapes)]  # noqa: E731
    if own:
        params = [torch.nn.Parameter(v) for v in views(flat)]
        for p, v in zip(params, views(grad)):
            p.grad = v
        opt = _package().AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY,
                               state_bits=case["bits"], master_weights=case["master"], seed=1)
        for key, buffer in opt.state_buffers(0).items():
            buffer.copy_(s[key])
            s[key] = buffer
        opt.set_step(STEP)
        s["opt"] = opt
    return s


def _prepare_linear(case, g):
    dtype, rows, k, n = DTYPES[case["dtype"]], case["tokens"], case["ins"], case["outs"]
    s = dict(x=_randn(g, rows, k).to(dtype), weight=(_randn(g, n, k) / math.sqrt(k)).to(dtype))
    s["bias"] = (0.1 * _randn(g, n)).to(dtype) if case["bias"] else None
    s["residual"] = _randn(g, rows, n).to(dtype) if case["residual"] else None
    if case["train"]:
        s["dy"] = _randn(g, rows, n).to(dtype)
        if own:
            for key in ("x", "weight", "bias"):
                if s[key] is not None:
                    s[key].requires_grad_(True)
    return s


PREPARE = dict(preference=_prepare_preference, policy=_prepare_policy, adamw=_prepare_adamw,
               linear=_prepare_linear)


def prepare(case, seed):
    state = PREPARE[case["op"]](case, _generator(seed))
    state["case"] = case
    if own:
        state["package"] = _package()
    return state


# ------------------------------------------------------------- plain forms --
def _plain_logprobs(logits, targets):
    """The 32-bit log probability of each row's target (0 where it is ignored) and softmax."""
    x = logits.float()
    x = x - x.amax(dim=1, keepdim=True)
    p = x.exp()
    total = p.sum(dim=1, keepdim=True)
    valid = targets != IGNORE
    index = torch.where(valid, targets, torch.zeros_like(targets))
    logp = x.gather(1, index[:, None])[:, 0] - total[:, 0].log()
    return torch.where(valid, logp, torch.zeros_like(logp)), p.div_(total), valid, index


def _plain_dlogits(p, index, coef, dtype):
    """coef * (one-hot - softmax), rounded once."""
    d = p.mul_(-coef[:, None])
    d[torch.arange(d.shape[0], device=d.device), index] += coef
    return d.to(dtype)


def _plain_preference(s):
    case, targets = s["case"], s["targets"]
    logp, p, valid, index = _plain_logprobs(s["logits"], targets)
    pos = torch.arange(targets.shape[0], device=targets.device)
    starts = s["cu_seqlens"].long()
    member = ((pos >= starts[:-1, None]) & (pos < starts[1:, None]) & valid).float()
    ratio = (member * (logp - s["ref"])).sum(dim=1).view(-1, 2)
    margin = BETA * (ratio[:, 0] - ratio[:, 1])
    soft = torch.log1p(torch.exp(-margin.abs()))
    eps = case["smoothing"]
    # -log sigmoid(z) = max(-z, 0) + log(1 + exp(-|z|))
    loss = ((1 - eps) * ((-margin).clamp(min=0) + soft)
            + eps * (margin.clamp(min=0) + soft)).sum() / margin.shape[0]
    dmargin = (torch.sigmoid(margin) - (1 - eps)) * (case["scale"] / margin.shape[0])
    per_seq = BETA * torch.stack([dmargin, -dmargin], dim=1).view(-1)
    coef = (member * per_seq[:, None]).sum(dim=0)
    return dict(loss=loss, logprobs=logp, margins=margin,
                dlogits=_plain_dlogits(p, index, coef, s["logits"].dtype))


def _plain_policy(s):
    case = s["case"]
    logp, p, valid, index = _plain_logprobs(s["logits"], s["targets"])
    count, mask = valid.sum(), valid.float()
    ratio = torch.exp(logp - s["old"])
    free = ratio * s["advantages"]
    held = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * s["advantages"]
    d = s["ref"] - logp
    kl = torch.expm1(d) - d
    loss = (mask * (case["kl"] * kl - torch.minimum(free, held))).sum() / count
    slope = torch.where(free <= held, -free, torch.zeros_like(free)) - case["kl"] * torch.expm1(d)
    coef = mask * slope * (case["scale"] / count)
    return dict(loss=loss, logprobs=logp, kl=(mask * kl).sum() / count,
                dlogits=_plain_dlogits(p, index, coef, s["logits"].dtype))


def _hash32(pos, key):
    """A 32-bit mix of an element's place in the state and the step's key."""
    m = 0xFFFFFFFF
    h = ((pos * 0x9E3779B9) & m) ^ key
    h = ((h ^ (h >> 16)) * 0x6A09E667) & m
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & m
    return h ^ (h >> 16)


def _to_e4m3(x, dither, floor):
    """x in blocks of 256 as 8-bit floats (4 bits of exponent, 3 of mantissa) times a power of
    two, rounded up or down by 16 bits of `dither`; `floor`: what is not 0 stays so."""
    b = x.view(-1, BLOCK)
    scale = _power_of_two_scale(b.abs().amax(dim=1))
    inverse = ((254 << 23) - scale.view(torch.int32)).view(torch.float32)
    y = b * inverse[:, None]
    a = y.abs()
    low = (a < 2.0 ** -6).float() * 2.0 ** -6  # below the smallest normal the grid is even
    bits = (a + low).view(torch.int32) + (dither.view_as(b) << 4).to(torch.int32)
    a2 = (bits & -(1 << 20)).view(torch.float32) - low
    if floor:
        a2 = torch.maximum(a2, (a > 0).float() * 2.0 ** -9)
    return torch.where(y < 0, -a2, a2).to(torch.float8_e4m3fn).view(-1), scale


def _plain_adamw(s):
    s["step"] += 1
    return _plain_adamw_8(s) if s["case"]["bits"] == 8 else _plain_adamw_32(s)


def _plain_adamw_32(s):
    """Tensor by tensor, as a model has its parameters, with the list forms of torch's products,
    sums and roots, in place where the state is."""
    t, wide = s["step"], "master" not in s and s["flat"].dtype != torch.float32
    each = lambda x: torch.split(x, s["padded"])  # noqa: E731
    g, m, v = each(s["grad"].float()), each(s["exp_avg"]), each(s["exp_avg_sq"])
    torch._foreach_mul_(m, B1)
    torch._foreach_add_(m, g, alpha=1 - B1)
    torch._foreach_mul_(v, B2)
    torch._foreach_add_(v, torch._foreach_mul(g, g), alpha=1 - B2)
    root = torch._foreach_sqrt(v)
    torch._foreach_mul_(root, 1 / math.sqrt(1 - B2 ** t))
    torch._foreach_add_(root, EPS)
    flat = s["flat"].float() if wide else s.get("master", s["flat"])
    p = each(flat)
    torch._foreach_mul_(p, 1 - LR * DECAY)
    torch._foreach_add_(p, torch._foreach_div(m, root), alpha=-LR / (1 - B1 ** t))
    if flat is not s["flat"]:
        s["flat"].copy_(flat)
    out = dict(params=s["flat"], exp_avg=s["exp_avg"], exp_avg_sq=s["exp_avg_sq"])
    return out | ({"master": s["master"]} if "master" in s else {})


def _plain_adamw_8(s):
    """On the whole state at once: its blocks of 256 belong to one tensor each."""
    t, g = s["step"], s["grad"].float()
    widen = lambda k: (s[k].float().view(-1, BLOCK) * s[k + "_scale"][:, None]).view(-1)  # noqa: E731
    m, r = widen("exp_avg"), widen("exp_avg_sq_root")
    m = m * B1 + g * (1 - B1)
    r = ((r * r) * B2 + (g * g) * (1 - B2)).sqrt()
    p = s["master"] if "master" in s else s["flat"].float()
    step = LR / (1 - B1 ** t)
    p = p * (1 - LR * DECAY) - step * (m / (r * (1 / math.sqrt(1 - B2 ** t)) + EPS))
    s["flat"].copy_(p)
    out = dict(params=s["flat"])
    if "master" in s:
        s["master"].copy_(p)
        out["master"] = s["master"]
    key = (1 * 0x9E3779B9 + t * 0x85A308D3) & 0xFFFFFFFF
    h = _hash32(torch.arange(m.shape[0], device=m.device), key)
    new = (_to_e4m3(m, h & 0xFFFF, False), _to_e4m3(r, h >> 16, True))
    for k, (code, scale) in zip(("exp_avg", "exp_avg_sq_root"), new):
        s[k].copy_(code)
        s[k + "_scale"].copy_(scale)
        out[k], out[k + "_scale"] = s[k], s[k + "_scale"]
    return out


def _activation(z, name):
    """(act(z), act'(z))"""
    if name == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if name == "silu":
        q = torch.sigmoid(z)
        return z * q, q * (1 + z * (1 - q))
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, None


def _linear(s, dtype):
    """y = act(x W^T + b) + residual and, in training, its gradients, in `dtype`."""
    case, x, w = s["case"], s["x"].to(dtype), s["weight"].to(dtype)
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].to(dtype)
    y, slope = _activation(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].to(dtype)
    out = dict(y=y)
    if case["train"]:
        dz = s["dy"].to(dtype)
        if slope is not None:
            dz = dz * slope
        out["dx"], out["dweight"] = dz @ w, dz.t() @ x
        if s["bias"] is not None:
            out["dbias"] = dz.sum(dim=0)
    return out


def _plain_linear(s):
    return {k: v.to(s["x"].dtype) for k, v in _linear(s, torch.float32).items()}


PLAIN = dict(preference=_plain_preference, policy=_plain_policy, adamw=_plain_adamw,
             linear=_plain_linear)


# ----------------------------------------------------------- own operators --
def _own_preference(s):
    r = s["package"].preference_loss_grad(
        s["logits"], s["targets"], s["ref"], s["cu_seqlens"], beta=BETA,
        label_smoothing=s["case"]["smoothing"], ignore_index=IGNORE, grad_scale=s["case"]["scale"])
    return dict(loss=r.loss, logprobs=r.logprobs, margins=r.margins, dlogits=r.dlogits)


def _own_policy(s):
    r = s["package"].policy_loss_grad(
        s["logits"], s["targets"], s["old"], s["advantages"], ref_logprobs=s["ref"],
        clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=s["case"]["kl"], ignore_index=IGNORE,
        grad_scale=s["case"]["scale"])
    return dict(loss=r.loss, logprobs=r.logprobs, kl=r.kl, dlogits=r.dlogits)


def _own_adamw(s):
    s["opt"].step()
    keys = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_root", "exp_avg_sq_root_scale",
            "master")
    return dict(params=s["flat"], **{k: s[k] for k in keys if k in s})


def _own_linear(s):
    x, w, b = s["x"], s["weight"], s["bias"]
    y = s["package"].linear_act(x, w, b, residual=s["residual"], activation=s["case"]["act"])
    if not s["case"]["train"]:
        return dict(y=y)
    wrt = [x, w] + ([b] if b is not None else [])
    grads = torch.autograd.grad(y, wrt, s["dy"])
    return dict(y=y.detach(), **dict(zip(("dx", "dweight", "dbias"), grads)))


OWN = dict(preference=_own_preference, policy=_own_policy, adamw=_own_adamw, linear=_own_linear)


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# --------------------------------------------------------------- 64 bits --
def _exact_rows(logits, targets):
    """Each row's log probability of its target, and a function that gives coef * (one-hot -
    softmax): from the log-sum-exp of the logits in 64 bits."""
    x = logits.double()
    lse = torch.logsumexp(x, dim=1)
    rows = torch.nonzero(targets != IGNORE)[:, 0]
    logp = torch.zeros_like(lse)
    logp[rows] = x[rows, targets[rows]] - lse[rows]

    def gradient(coef):
        d = x.sub_(lse[:, None]).exp_().mul_(-coef[:, None])
        d[rows, targets[rows]] += coef[rows]
        return d

    return logp, rows, gradient


def _exact_preference(case, s):
    logp, rows, gradient = _exact_rows(s["logits"], s["targets"])
    ends = s["cu_seqlens"].tolist()
    delta = torch.zeros_like(logp)
    delta[rows] = logp[rows] - s["ref"].double()[rows]
    margins, coef = [], torch.zeros_like(logp)
    live = (s["targets"] != IGNORE).double()
    loss, n = 0.0, case["pairs"]
    for i in range(n):
        a, b, c = ends[2 * i:2 * i + 3]
        z = BETA * float(delta[a:b].sum() - delta[b:c].sum())
        margins.append(z)
        up = 1 / (1 + math.exp(z))  # d(-log sigmoid(z)) / dz = -up
        loss += ((1 - case["smoothing"]) * math.log1p(math.exp(-z))
                 + case["smoothing"] * math.log1p(math.exp(z))) / n
        dz = (-(1 - case["smoothing"]) * up + case["smoothing"] * (1 - up)) * case["scale"] / n
        coef[a:b], coef[b:c] = BETA * dz, -BETA * dz
    return dict(loss=torch.tensor(loss, dtype=torch.float64), logprobs=logp,
                margins=torch.tensor(margins, dtype=torch.float64), dlogits=gradient(coef * live))


def _exact_policy(case, s):
    logp, rows, gradient = _exact_rows(s["logits"], s["targets"])
    lp, old, ref, adv = (v.double()[rows] for v in (logp, s["old"], s["ref"], s["advantages"]))
    ratio = (lp - old).exp()
    # the clip holds the surrogate where the ratio has gone past the edge in the gain's direction
    past = torch.where(adv > 0, ratio > 1 + CLIP_HIGH, ratio < 1 - CLIP_LOW)
    edge = torch.where(adv > 0, 1.0 + CLIP_HIGH, 1.0 - CLIP_LOW)
    gain = torch.where(past, edge, ratio) * adv
    kl = (ref - lp).exp() - 1 - (ref - lp)
    n = rows.shape[0]
    coef = torch.zeros_like(logp)
    coef[rows] = case["scale"] / n * (torch.where(past, 0.0, -ratio * adv)
                                      + case["kl"] * (1 - (ref - lp).exp()))
    return dict(loss=(case["kl"] * kl - gain).mean(), logprobs=logp, kl=kl.mean(),
                dlogits=gradient(coef))


def _exact_adamw(case, s):
    t, g = STEP + 1, s["grad"].double()
    if case["bits"] == 8:
        by_block = lambda k: s[k].double() * s[k + "_scale"].double().repeat_interleave(BLOCK)  # noqa: E731
        m, v = by_block("exp_avg"), by_block("exp_avg_sq_root") ** 2
    else:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    m = m.mul_(B1).add_(g, alpha=1 - B1)
    v = v.mul_(B2).addcmul_(g, g, value=1 - B2)
    p = (s["master"] if case["master"] else s["flat"]).double()
    p = p - LR * (DECAY * p + (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS))
    out = dict(params=p)
    if case["master"]:
        out["master"] = p
    if case["bits"] == 8:
        # what is stored is rounded at random to 8 bits: no 64-bit value
        out |= {k: None for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq_root",
                                  "exp_avg_sq_root_scale")}
    else:
        out["exp_avg"], out["exp_avg_sq"] = m, v
    return out


def _exact_linear(case, s):
    x = s["x"].double().requires_grad_(case["train"])
    w = s["weight"].double().requires_grad_(case["train"])
    b = s["bias"].double().requires_grad_(case["train"]) if case["bias"] else None
    f = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu,
         "gelu": torch.nn.functional.gelu}[case["act"]]
    y = f(torch.nn.functional.linear(x, w, b))
    out = dict(y=y.detach() + s["residual"].double() if case["residual"] else y.detach())
    if case["train"]:
        names = ["dx", "dweight"] + (["dbias"] if case["bias"] else [])
        out |= dict(zip(names, torch.autograd.grad(
            y, [x, w] + ([b] if case["bias"] else []), s["dy"].double())))
    return out


EXACT = dict(preference=_exact_preference, policy=_exact_policy, adamw=_exact_adamw,
             linear=_exact_linear)


def exact(case, seed):
    state = PREPARE[case["op"]](case, _generator(seed))
    return EXACT[case["op"]](case, state)


# -------------------------------------------------------------------- work --
def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if op in ("preference", "policy"):
        rows = case["tokens"] * (2 * case["pairs"] if op == "preference" else 1)
        # the logits once in, their gradient once out; a difference, an exponential, a sum and a
        # product for each, then three more for the gradient
        per_row = 8 + 4 + 4 if op == "preference" else 8 + 12 + 4
        return dict(bytes=2 * rows * case["vocab"] * size + rows * per_row,
                    flops=7 * rows * case["vocab"])
    if op == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        state = 16 if case["bits"] == 32 else 4 + 4 * 4 / BLOCK
        return dict(bytes=n * (3 * size + state + (8 - size if case["master"] else 0)),
                    flops=14 * n)
    m, k, n = case["tokens"], case["ins"], case["outs"]
    values = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
    if case["train"]:
        values += m * n + m * k + n * k + (n if case["bias"] else 0)
    return dict(bytes=values * size, flops=(6 if case["train"] else 2) * m * n * k)
