"""Timed cases of the trainable answer head: the norm in front of the vocabulary
projection, the projection's cross entropy with its gradients, and the AdamW
step that updates both.

A pass is what one training or scoring step of a program calls: the norm
(forward alone, or forward and backward), the loss of a batch of hidden states
against their next tokens (forward alone for scoring, forward and backward for
training), or one optimiser step over a list of tensors. Where ``own`` is false
the same mathematics is written with elementary torch operations in float32.

Definitions (all in float32 or wider, one rounding at the end):

  norm      mean = sum(x) / D (0 without centring), rstd = 1 / sqrt(sum((x - mean)^2) / D + eps),
            xhat = (x - mean) * rstd, y = xhat * w + b;
            with a = dy * w: dx = rstd * (a - [sum(a) / D] - xhat * sum(a * xhat) / D), the bracket with
            centring only; dw = sum over rows of dy * xhat, db = sum over rows of dy
  loss      z = h . W_v, l = c * tanh(z / c) (l = z without a softcap), lse = log(sum(exp(l))),
            loss = lse - l_target, 0 where the target is outside [0, V);
            dz = g * (exp(l - lse) - [v = target]) * (1 - (l / c)^2), 0 for such a row;
            dh = sum over v of dz * W_v, dW_v = sum over rows of dz * h
  AdamW     g = grad * grad_scale, m = b1 * m + (1 - b1) * g, v = b2 * v + (1 - b2) * g * g,
            p = p * (1 - lr * decay) - (lr / (1 - b1^t)) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
            States in 8 bits: blocks of 256 elements with a float32 scale each, m in e4m3 in units of
            (largest |m|) / 448, v in e5m2 in units of (largest v) / 57344, rounded up or down at random with
            the chance that keeps the mean; the random bits are a hash of the seed, the step and the
            element's place in the list. The step uses the values before they are rounded.
"""
import math

import torch

own = False

BLOCK = 256  # elements that share a scale of 8-bit states


def listed():
    return [
        # One token's log-probability under the full vocabulary: the weights are read once, latency counts.
        dict(name="score_1", kind="score", rows=1, dim=2816, vocab=262144, dtype="bf16", softcap=30.0, ignored=0.0),
        # A few candidate tokens scored by a small model with an odd vocabulary.
        dict(name="score_7_small", kind="score", rows=7, dim=640, vocab=32003, dtype="bf16", softcap=0.0, ignored=0.0),
        # The perplexity of a short text in float32.
        dict(name="score_96_f32", kind="score", rows=96, dim=1000, vocab=50257, dtype="f32", softcap=0.0, ignored=0.0),
        # A training step of a small model over ragged sequences whose prompt tokens carry no loss.
        dict(name="train_1021", kind="train", rows=1021, dim=1152, vocab=32003, dtype="bf16", softcap=30.0, ignored=0.3),
        # The same step in float32.
        dict(name="train_300_f32", kind="train", rows=300, dim=768, vocab=50257, dtype="f32", softcap=0.0, ignored=0.1),
        # The largest step: a batch of 4,096 tokens over the full vocabulary.
        dict(name="train_4096", kind="train", rows=4096, dim=2816, vocab=262144, dtype="bf16", softcap=30.0, ignored=0.1),
        # The norm of four sessions' newest tokens in a decode loop.
        dict(name="norm_4", kind="norm", rows=4, dim=2816, dtype="bf16", wdtype="bf16", center=False, bias=False),
        # The norm with its gradients, odd sizes, everything in float32.
        dict(name="norm_train_4099_f32", kind="norm_train", rows=4099, dim=1001, dtype="f32", wdtype="f32", center=True, bias=True),
        # The norm of a large training batch in bfloat16 with float32 weights.
        dict(name="norm_train_16384", kind="norm_train", rows=16384, dim=2816, dtype="bf16", wdtype="f32", center=True, bias=True),
        # The step of a small model's adapters: many tiny tensors, one launch's latency.
        dict(name="adamw_adapters", kind="adamw", tensors=24, most=20000, dtype="f32", gdtype="f32", master=False, bits=32),
        # Mixed training: bfloat16 weights with float32 masters, tensors of every size.
        dict(name="adamw_mixed", kind="adamw", tensors=150, most=4000000, dtype="bf16", gdtype="bf16", master=True, bits=32),
        # The head's own weights, whose states fit beside them in 8 bits.
        dict(name="adamw_head_8bit", kind="adamw", tensors=2, most=262144 * 2816, dtype="bf16", gdtype="bf16", master=False, bits=8),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("score", "train", "train", "norm", "norm_train", "adamw"))
    c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "f32")))
    if kind in ("score", "train"):
        c["rows"] = _spread(rng, 1, 512) if kind == "score" else _spread(rng, 16, 4096)
        c["vocab"] = 262144 if rng.random() < 0.2 else _spread(rng, 8000, 262144)
        c["dim"] = _spread(rng, 256, 2816)
        if rng.random() < 0.8:  # models' widths are round, with few exceptions
            c["dim"] = max(256, c["dim"] - c["dim"] % 64)
        if c["dtype"] == "f32" and kind == "train":  # float32 heads are small ones
            c["rows"], c["vocab"] = min(c["rows"], 1024), min(c["vocab"], 65536)
        c["softcap"] = rng.choice((30.0, 0.0))
        c["ignored"] = rng.choice((0.0, 0.1, 0.5))
    elif kind in ("norm", "norm_train"):
        c["rows"] = _spread(rng, 1, 512) if kind == "norm" else _spread(rng, 16, 16384)
        c["dim"] = _spread(rng, 64, 8192)
        if rng.random() < 0.7:
            c["dim"] = max(64, c["dim"] - c["dim"] % 64)
        c["wdtype"] = "f32" if c["dtype"] == "f32" else rng.choice(("bf16", "f32"))
        c["center"] = rng.random() < 0.6
        c["bias"] = c["center"] and rng.random() < 0.7
    else:
        c["tensors"] = _spread(rng, 1, 200)
        c["most"] = _spread(rng, 1000, 4000000)
        c["gdtype"] = "f32" if c["dtype"] == "f32" else rng.choice(("bf16", "f32"))
        c["master"] = c["dtype"] == "bf16" and rng.random() < 0.5
        c["bits"] = rng.choice((8, 32))
    return c


DTYPES = dict(f32=torch.float32, bf16=torch.bfloat16)
EPS = 1e-6
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01)
GRAD_SCALE = 0.5
STEPS = 100  # optimiser steps taken before the first timed one


def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _sizes(c):
    """The tensors' element counts: the largest first, the others spread over the logarithm, odd ones among them."""
    n, most = c["tensors"], c["most"]
    return [most] + [max(1, int(most ** (0.25 + 0.75 * ((i * 0.6180339887) % 1.0)))) for i in range(1, n)]


def _inputs(c, seed):
    gen, kind = _gen(seed), c["kind"]
    dt = DTYPES[c["dtype"]]
    if kind in ("score", "train"):
        n, d, v = c["rows"], c["dim"], c["vocab"]
        # logits of standard deviation 3, and the target's raised by up to 16: from unforeseen tokens to certain ones
        w = (_randn(gen, v, d, dtype=dt) * (3.0 / math.sqrt(d))).to(dt)
        targets = torch.randint(v, (n,), generator=gen, device="cuda")
        up = 16.0 * torch.rand(n, 1, generator=gen, device="cuda")
        h = (_randn(gen, n, d) + up / 9.0 * w[targets].float()).to(dt)
        skip = torch.rand(n, generator=gen, device="cuda") < c["ignored"]
        targets = torch.where(skip, -1, targets).int()
        g = torch.full((n,), 1.0 / n, device="cuda")
        return dict(h=h, w=w, targets=targets, g=g)
    if kind in ("norm", "norm_train"):
        n, d, wdt = c["rows"], c["dim"], DTYPES[c["wdtype"]]
        # hidden states: channels of different size and offset, a few of them far larger
        size = torch.exp(0.5 * _randn(gen, d)) * torch.where(torch.rand(d, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
        x = (size * _randn(gen, n, d) + 0.3 * _randn(gen, d)).to(dt)
        w = (1.0 + 0.2 * _randn(gen, d)).to(wdt)
        b = (0.2 * _randn(gen, d)).to(wdt) if c["bias"] else None
        dy = (_randn(gen, n, d) / n).to(dt)
        return dict(x=x, w=w, b=b, dy=dy)
    sizes = _sizes(c)
    starts, total = [], 0
    for s in sizes:  # each tensor begins at a block of its own in one buffer
        starts.append(total)
        total += -(-s // BLOCK) * BLOCK
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, s in zip(starts, sizes):
        live[a:a + s] = True
    p32 = torch.where(live, _randn(gen, total) * 0.02, 0.0)
    grad = torch.where(live, _randn(gen, total) * 1e-3, 0.0).to(DTYPES[c["gdtype"]])
    m = torch.where(live, _randn(gen, total) * 3e-4, 0.0)
    v = torch.where(live, (_randn(gen, total) * 5e-4).square_(), 0.0)
    s = dict(p=p32.to(dt), grad=grad, master=p32 if c["master"] else None, starts=starts, sizes=sizes)
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _first_codes(m, 448.0, torch.float8_e4m3fn)
        s["v"], s["v_scale"] = _first_codes(v, 57344.0, torch.float8_e5m2)
    else:
        s["m"], s["v"] = m, v
    return s


def _first_codes(x, top, dtype):
    """States as an earlier step left them: 8-bit values and their blocks' scales."""
    blocks = x.view(-1, BLOCK)
    scale = blocks.abs().amax(1) / top
    return (blocks / scale.clamp_min(1e-30)[:, None]).to(dtype).view(-1), scale


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"], s["steps"] = c, STEPS
    if own:
        from gemmaedge_amd import head as H

        if c["kind"] == "adamw":
            views = lambda t: [t[a:a + n] for a, n in zip(s["starts"], s["sizes"])]  # noqa: E731
            blocks = lambda t: [t[a // BLOCK:-(-(a + n) // BLOCK)] for a, n in zip(s["starts"], s["sizes"])]  # noqa: E731
            states = dict(m=views(s["m"]), v=views(s["v"]))
            if c["bits"] == 8:
                states.update(m_scale=blocks(s["m_scale"]), v_scale=blocks(s["v_scale"]))
            s["adamw"] = H.AdamW(views(s["p"]), views(s["grad"]), masters=views(s["master"]) if c["master"] else None,
                                 state_bits=c["bits"], seed=7, **states, **HYPER)
            s["adamw"].steps = STEPS
        else:
            train = c["kind"] in ("train", "norm_train")
            s["head"] = H.Head(c["rows"], c["dim"], c.get("vocab", 1), dtype=DTYPES[c["dtype"]], train=train)
    return s


# ---- plain forms --------------------------------------------------------------


def _norm_forward(x, w, b, center):
    x = x.float()
    mean = x.mean(1, keepdim=True) if center else torch.zeros_like(x[:, :1])
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + EPS)
    y = xc * rstd * w.float()
    return (y if b is None else y + b.float()), mean, rstd


def _norm_backward(dy, x, w, mean, rstd, center):
    dy = dy.float()
    xhat = (x.float() - mean) * rstd
    a = dy * w.float()
    t = a - xhat * (a * xhat).mean(1, keepdim=True)
    if center:
        t = t - a.mean(1, keepdim=True)
    return t * rstd, (dy * xhat).sum(0), dy.sum(0)


def _loss_forward(h, w, targets, softcap):
    z = h.float() @ w.float().t()
    l = softcap * torch.tanh(z / softcap) if softcap > 0 else z
    top = l.amax(1, keepdim=True)
    lse = top[:, 0] + torch.log(torch.exp(l - top).sum(1))
    kept = (targets >= 0) & (targets < w.shape[0])
    at = l.gather(1, targets.clamp(0, w.shape[0] - 1).long()[:, None])[:, 0]
    return torch.where(kept, lse - at, 0.0), lse, l, kept


def _loss_backward(g, h, w, targets, l, lse, kept, softcap):
    dz = torch.exp(l - lse[:, None])
    rows = torch.arange(h.shape[0], device=h.device)
    dz[rows, targets.clamp(0, w.shape[0] - 1).long()] -= 1.0
    if softcap > 0:
        dz *= 1.0 - (l / softcap) ** 2
    dz *= torch.where(kept, g, 0.0)[:, None]
    return (dz @ w.float()).to(h.dtype), (dz.t() @ h.float()).to(w.dtype)


def _i32(x):
    """x modulo 2^32 as a signed 32-bit number."""
    x &= 0xFFFFFFFF
    return x - (1 << 32) if x >> 31 else x


def _mix(x):
    """A 32-bit hash of int32 tensors: shifts without sign and products modulo 2^32."""
    x = (x ^ ((x >> 16) & 0xFFFF)) * _i32(0xBB67AE85)
    x = (x ^ ((x >> 15) & 0x1FFFF)) * _i32(0x6A09E667)
    return x ^ ((x >> 16) & 0xFFFF)


def _random_bits(blocks, seed, step):
    """32 random bits for every element: of the block's number, the seed and the step, then of the place in the block."""
    b = torch.arange(blocks, device="cuda", dtype=torch.int32)[:, None]
    i = torch.arange(BLOCK, device="cuda", dtype=torch.int32)[None, :]
    return _mix(_mix(_mix(b + _i32(0x9E3779B9 * seed)) + _i32(0x9E3779B9 * step)) + i * _i32(0x9E3779B9))


def _encode(x, bits, top, low, drop, dtype):
    """Blocks of values >= 0 in 8 bits: scale, random rounding of the bits below the format's, codes' values."""
    big = x.amax(1, keepdim=True)
    dead = big < 2.0 ** -100
    y = torch.clamp_max(x * (top / torch.where(dead, 1.0, big)), top)
    r = ((y.view(torch.int32) + (bits << (drop - 16))) >> drop << drop).view(torch.float32)
    small = torch.where((bits.float() * (low / 65536.0)) < y, low, 0.0) if dtype == torch.float8_e4m3fn else torch.where(y > 0, low, 0.0)
    r = torch.where(y < low, small, r)
    return torch.where(dead, 0.0, r), torch.where(dead, 0.0, big * (1.0 / top))[:, 0]


def _adamw(s, c):
    t = s["steps"] = s["steps"] + 1
    k = HYPER
    decay = 1.0 - k["lr"] * k["weight_decay"]
    size = k["lr"] / (1.0 - k["beta1"] ** t)
    root = 1.0 / math.sqrt(1.0 - k["beta2"] ** t)
    g = s["grad"].float() * GRAD_SCALE
    m, v = s["m"], s["v"]
    if c["bits"] == 8:
        m = (m.float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
    m = m * k["beta1"] + g * (1.0 - k["beta1"])
    v = v * k["beta2"] + g * g * (1.0 - k["beta2"])
    p = s["p"].float() if s["master"] is None else s["master"]
    p = p * decay - m / (torch.sqrt(v) * root + k["eps"]) * size
    s["p"].copy_(p)
    if s["master"] is not None:
        s["master"].copy_(p)
    if c["bits"] == 8:
        bits = _random_bits(m.numel() // BLOCK, 7, t)
        mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
        r, scale = _encode(mb.abs(), bits & 0xFFFF, 448.0, 2.0 ** -6, 20, torch.float8_e4m3fn)
        s["m"].copy_(torch.copysign(r, mb).view(-1).to(torch.float8_e4m3fn))
        s["m_scale"].copy_(scale)
        r, scale = _encode(vb, (bits >> 16) & 0xFFFF, 57344.0, 2.0 ** -14, 21, torch.float8_e5m2)
        s["v"].copy_(r.view(-1).to(torch.float8_e5m2))
        s["v_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)


# ---- the pass -----------------------------------------------------------------


def run(s):
    c = s["case"]
    kind = c["kind"]
    if kind in ("score", "train"):
        cap = c["softcap"]
        if own:
            loss, lse = s["head"].loss(s["h"], s["w"], s["targets"], softcap=cap)
            if kind == "score":
                return dict(loss=loss, lse=lse)
            dh, dw = s["head"].loss_backward(s["g"], s["h"], s["w"], s["targets"], lse, softcap=cap)
        else:
            loss, lse, l, kept = _loss_forward(s["h"], s["w"], s["targets"], cap)
            if kind == "score":
                return dict(loss=loss, lse=lse)
            dh, dw = _loss_backward(s["g"], s["h"], s["w"], s["targets"], l, lse, kept, cap)
        return dict(loss=loss, lse=lse, dh=dh, dw=dw)
    if kind in ("norm", "norm_train"):
        x, w, b, center = s["x"], s["w"], s["b"], c["center"]
        if own:
            y, mean, rstd = s["head"].norm(x, w, b, eps=EPS, center=center)
            if kind == "norm":
                return dict(y=y, rstd=rstd)
            dx, dw, db = s["head"].norm_backward(s["dy"], x, w, mean, rstd, bias=b is not None)
        else:
            y, mean, rstd = _norm_forward(x, w, b, center)
            y = y.to(x.dtype)
            if kind == "norm":
                return dict(y=y, rstd=rstd[:, 0])
            dx, dw, db = _norm_backward(s["dy"], x, w, mean, rstd, center)
            dx, dw, rstd = dx.to(x.dtype), dw.to(w.dtype), rstd[:, 0]
            db = db.to(w.dtype) if b is not None else None
        return dict(y=y, rstd=rstd, dx=dx, dw=dw, db=db)
    if own:
        s["adamw"].step(grad_scale=GRAD_SCALE)
    else:
        _adamw(s, c)
    return {k: s[k] for k in ("p", "master", "m", "v", "m_scale", "v_scale") if s.get(k) is not None}


def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] in ("score", "train"):
        n, d, v = c["rows"], c["dim"], c["vocab"]
        reads = (n + v) * d * size + 4 * n
        if c["kind"] == "score":
            return dict(bytes=reads + 8 * n, flops=2.0 * n * d * v)
        return dict(bytes=reads + 12 * n + (n + v) * d * size, flops=6.0 * n * d * v)
    if c["kind"] in ("norm", "norm_train"):
        n, d = c["rows"], c["dim"]
        ws = (2 if c["wdtype"] == "bf16" else 4) * d * (2 if c["bias"] else 1)
        if c["kind"] == "norm":
            return dict(bytes=2 * n * d * size + ws + 4 * n, flops=8.0 * n * d)
        return dict(bytes=4 * n * d * size + 2 * ws + 4 * n, flops=22.0 * n * d)
    total = sum(_sizes(c))
    gsize = 2 if c["gdtype"] == "bf16" else 4
    state = 16 if c["bits"] == 32 else 4 + 16.0 / BLOCK
    params = size + 8 if c["master"] else 2 * size
    return dict(bytes=total * (params + gsize + state), flops=14.0 * total)


# ---- the definitions in 64 bits -------------------------------------------------


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    kind = c["kind"]
    if kind in ("score", "train"):
        return _exact_loss(c, s)
    if kind in ("norm", "norm_train"):
        x, w = s["x"].double(), s["w"].double()
        d = x.shape[1]
        mean = x.sum(1) / d if c["center"] else torch.zeros(x.shape[0], device="cuda", dtype=torch.float64)
        x = x - mean[:, None]
        rstd = ((x ** 2).sum(1) / d + EPS) ** -0.5
        x *= rstd[:, None]
        y = x * w if s["b"] is None else torch.addcmul(s["b"].double(), x, w)
        if kind == "norm":
            return dict(y=y, rstd=rstd)
        dy = s["dy"].double()
        dw, db = torch.einsum("nd,nd->d", dy, x), dy.sum(0)
        dy *= w
        dx = dy - x * (torch.einsum("nd,nd->n", dy, x) / d)[:, None]
        if c["center"]:
            dx -= dy.sum(1, keepdim=True) / d
        return dict(y=y, rstd=rstd, dx=dx * rstd[:, None], dw=dw, db=db if c["bias"] else None)
    k, t = HYPER, STEPS + 1
    g = s["grad"].double() * GRAD_SCALE
    scaled = lambda q, z: q.double() if z is None else (q.float().double().view(-1, BLOCK) * z.double()[:, None]).view(-1)  # noqa: E731
    m = scaled(s["m"], s.get("m_scale")).lerp(g, 1.0 - k["beta1"])
    v = scaled(s["v"], s.get("v_scale")).lerp(g * g, 1.0 - k["beta2"])
    p = (s["p"] if s["master"] is None else s["master"]).double()
    p = p - k["lr"] * (k["weight_decay"] * p + (m / (1 - k["beta1"] ** t)) / ((v / (1 - k["beta2"] ** t)) ** 0.5 + k["eps"]))
    out = dict(p=p, master=None if s["master"] is None else p)
    if c["bits"] == 8:  # a value rounded at random has no counterpart in 64 bits; its block's scale has
        out.update(m=None, v=None, m_scale=m.view(-1, BLOCK).abs().amax(1) / 448.0, v_scale=v.view(-1, BLOCK).amax(1) / 57344.0)
    else:
        out.update(m=m, v=v)
    return out


def _exact_loss(c, s):
    h, targets, cap = s["h"].double(), s["targets"].long(), c["softcap"]
    n, v = c["rows"], c["vocab"]
    piece = max(1024, min(v, (1 << 28) // n))  # columns of the vocabulary at a time

    def logits(a):
        w = s["w"][a:a + piece].double()
        z = h @ w.t()
        return w, cap * torch.tanh(z / cap) if cap > 0 else z

    kept = (targets >= 0) & (targets < v)
    parts, at = [], torch.zeros(n, device="cuda", dtype=torch.float64)
    for a in range(0, v, piece):
        _, l = logits(a)
        parts.append(torch.logsumexp(l, 1))
        here = kept & (targets >= a) & (targets < a + l.shape[1])
        at[here] = l[here, targets[here] - a]
    lse = torch.logsumexp(torch.stack(parts), 0)
    out = dict(loss=torch.where(kept, lse - at, 0.0), lse=lse)
    if c["kind"] == "score":
        return out
    g = s["g"].double() * kept
    dh, dw = torch.zeros_like(h), torch.empty(s["w"].shape, device="cuda", dtype=torch.float64)
    for a in range(0, v, piece):
        w, l = logits(a)
        dz = (l - lse[:, None]).exp_()
        here = kept & (targets >= a) & (targets < a + l.shape[1])
        dz[here, targets[here] - a] -= 1.0
        if cap > 0:
            dz *= 1.0 - (l / cap).square_()
        dz *= g[:, None]
        dh += dz @ w
        dw[a:a + piece] = dz.t() @ h
    return dict(out, dh=dh, dw=dw)
