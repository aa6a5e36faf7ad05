"""The AdamW step on the GPU: float32 states against float64, 8-bit states
against the format's definition in numpy, bit for bit.

Tolerances of the float32 step, u = 2^-24: m and v are two products and a sum
(3 u of the sum of magnitudes), the update a square root, two quotients and two
products more; p itself is rounded twice. Stored in bf16 it is rounded once more."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HP = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1)
SIZES = (1, 2, 3, 255, 256, 257, 4095, 4096, 4097, 0, 70001, 5)


def rand(n, seed, scale, dtype=torch.float32, offset=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(n + offset, generator=g, device="cuda") * scale).to(dtype)
    return x[offset:]


def expected(p, g, m, v, step, scale, hp=HP):
    p, g, m, v = p.double(), g.double() * scale, m.double(), v.double()
    m1 = hp["beta1"] * m + (1 - hp["beta1"]) * g
    v1 = hp["beta2"] * v + (1 - hp["beta2"]) * g * g
    denom = torch.sqrt(v1) / (1 - hp["beta2"] ** step) ** 0.5 + hp["eps"]
    upd = hp["lr"] / (1 - hp["beta1"] ** step) * m1 / denom
    e_m = 4 * U * (hp["beta1"] * m.abs() + (1 - hp["beta1"]) * g.abs())
    p1 = p * (1 - hp["lr"] * hp["weight_decay"]) - upd
    e_p = 12 * U * upd.abs() + hp["lr"] / (1 - hp["beta1"] ** step) * e_m / denom + 3 * U * (p.abs() + p1.abs())
    return p1, m1, v1, e_p, e_m, 5 * U * v1


@pytest.mark.parametrize("dt,gdt,master", [("f32", "f32", False), ("bf16", "bf16", True), ("bf16", "f32", False), ("f32", "bf16", True),
                                           ("bf16", "bf16", False)])
@pytest.mark.parametrize("offset", (0, 1, 3))
def test_states_of_32_bits(dt, gdt, master, offset):
    from gemmaedge_amd import head as H

    ps = [rand(n, 10 + i, 0.05, DT[dt], offset) for i, n in enumerate(SIZES)]
    gs = [rand(n, 40 + i, 1e-3, DT[gdt], offset) for i, n in enumerate(SIZES)]
    masters = [rand(n, 70 + i, 0.05, offset=offset) if i % 3 else None for i, n in enumerate(SIZES)] if master else None
    opt = H.AdamW(ps, gs, masters=masters, **HP)
    for step in range(1, 4):
        for i, g in enumerate(gs):
            if step == 2:
                g.mul_(-0.5)
            if step == 3:
                g.zero_()
        src = [(masters[i] if masters and masters[i] is not None else p).clone() for i, p in enumerate(ps)]
        was = [(m.clone(), v.clone()) for m, v in zip(opt.m, opt.v)]
        opt.step(grad_scale=0.25)
        assert opt.steps == step
        for i, p in enumerate(ps):
            p1, m1, v1, e_p, e_m, e_v = expected(src[i], gs[i], *was[i], step, 0.25)
            assert ((opt.m[i].double() - m1).abs() <= e_m + 1e-40).all(), (i, step)
            assert ((opt.v[i].double() - v1).abs() <= e_v + 1e-40).all(), (i, step)
            if masters and masters[i] is not None:
                assert ((masters[i].double() - p1).abs() <= e_p).all(), (i, step)
                assert torch.equal(p, masters[i].to(p.dtype))
            else:
                r = torch.finfo(p.dtype).eps / 2
                assert ((p.double() - p1).abs() <= e_p + r * (p1.abs() + e_p)).all(), (i, step)


# ---- 8-bit states: the definition in numpy ------------------------------------


def mix(x):
    x = ((x ^ (x >> np.uint32(16))) * np.uint32(0xBB67AE85)).astype(np.uint32)
    x = ((x ^ (x >> np.uint32(15))) * np.uint32(0x6A09E667)).astype(np.uint32)
    return x ^ (x >> np.uint32(16))


def encode(x, bits, top, man, bias, up):
    """Codes of |x| for one block (float32), 16 random bits each, and the scale."""
    f = np.float32
    big = x.max() if x.size else f(0)
    if big < f(2.0 ** -100):
        return np.zeros(x.size, np.uint8), f(0)
    y = np.minimum(x * ((f(1) / big) * f(top)), f(top)).astype(np.float32)
    low = f(2.0 ** (1 - bias))
    drop = 23 - man
    r = ((y.view(np.uint32) + (bits << np.uint32(drop - 16))) >> np.uint32(drop)) - np.uint32((127 - bias) << man)
    keep = y > 0 if up else bits.astype(np.float32) * (low / f(65536)) < y
    return np.where(y < low, np.where(keep, 1 << man, 0), r).astype(np.uint8), big * (f(1) / f(top))


def step8(p, g, m, ms, v, vs, first_block, step, scale, seed):
    f = np.float32
    hp = HP
    b1, r1, b2, r2 = f(hp["beta1"]), f(1 - hp["beta1"]), f(hp["beta2"]), f(1 - hp["beta2"])
    out_m, out_v = np.zeros(p.size, np.uint8), np.zeros(p.size, np.uint8)
    for b in range(-(-p.size // 256)):
        at = slice(b * 256, min(p.size, b * 256 + 256))
        gg = g[at] * f(scale)
        mm = m[at] * ms[b] * b1 + gg * r1
        vv = v[at] * vs[b] * b2 + gg * gg * r2
        with np.errstate(over="ignore"):
            key = mix(mix(np.uint32([first_block + b]) + np.uint32(seed * 0x9E3779B9 & 0xFFFFFFFF)) + np.uint32(step * 0x9E3779B9 & 0xFFFFFFFF))
            bits = mix(key + (np.arange(mm.size, dtype=np.uint64) * 0x9E3779B9 & 0xFFFFFFFF).astype(np.uint32))
        q, ms[b] = encode(np.abs(mm), bits & np.uint32(0xFFFF), 448.0, 3, 7, False)
        out_m[at] = q | np.where(mm < 0, 0x80, 0).astype(np.uint8)
        out_v[at], vs[b] = encode(vv, bits >> np.uint32(16), 57344.0, 2, 15, True)
        denom = np.sqrt(vv) * f(1 / np.sqrt(1 - hp["beta2"] ** step)) + f(hp["eps"])
        p[at] = p[at] * f(1 - hp["lr"] * hp["weight_decay"]) - mm / denom * f(hp["lr"] / (1 - hp["beta1"] ** step))
    return out_m, out_v


def values(codes, dtype):
    return torch.from_numpy(codes.copy()).view(dtype).float().numpy()


@pytest.mark.parametrize("offset", (0, 1))
@pytest.mark.parametrize("gdt", ("f32", "bf16"))
def test_states_of_8_bits(offset, gdt):
    from gemmaedge_amd import head as H

    ps = [rand(n, 10 + i, 0.05, offset=offset) for i, n in enumerate(SIZES)]
    gs = [rand(n, 40 + i, 1e-3, DT[gdt], offset) for i, n in enumerate(SIZES)]
    for i, g in enumerate(gs):  # blocks with far apart values, and some of zeros
        if g.numel() > 300:
            g[:200] *= 1e-4
            g[100:150] = 0
            g[256:512] = 0
            g[-1] = 3.0
    opt = H.AdamW(ps, gs, state_bits=8, seed=99, **HP)
    want = [[p.cpu().numpy().copy(), np.zeros(p.numel(), np.float32), np.zeros(-(-p.numel() // 256), np.float32),
             np.zeros(p.numel(), np.float32), np.zeros(-(-p.numel() // 256), np.float32)] for p in ps]
    for step in range(1, 5):
        opt.step(grad_scale=0.5)
        first = 0
        for i, p in enumerate(ps):
            w = want[i]
            qm, qv = step8(w[0], gs[i].float().cpu().numpy(), w[1], w[2], w[3], w[4], first, step, 0.5, 99)
            first += -(-p.numel() // 256)
            w[1], w[3] = values(qm, torch.float8_e4m3fn), values(qv, torch.float8_e5m2)
            assert np.array_equal(opt.m[i].cpu().view(torch.uint8).numpy(), qm), (i, step)
            assert np.array_equal(opt.v[i].cpu().view(torch.uint8).numpy(), qv), (i, step)
            assert np.array_equal(opt.m_scale[i].cpu().numpy(), w[2]) and np.array_equal(opt.v_scale[i].cpu().numpy(), w[4])
            # square root and quotients: 1 ulp each of the update, and p's own rounding
            got = p.double().cpu().numpy()
            assert np.all(np.abs(got - w[0]) <= 4 * U * np.abs(w[0]) + 8 * U * 0.05)
            w[0] = p.cpu().numpy().copy()


def test_random_rounding_keeps_the_mean():
    from gemmaedge_amd import head as H

    # A constant gradient: every step moves v by (1 - beta2) of its distance, far less than a code's step. The mean over
    # 65,536 elements must follow; each element's variance is below (step / 2)^2 a step, and beta2 forgets it.
    n = 65536
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1.0, device="cuda")
    g[::256] = 4.0  # the blocks' scale
    opt = H.AdamW([p], [g], state_bits=8, beta2=0.999, lr=0.0, weight_decay=0.0)
    for _ in range(300):
        opt.step()
    v = opt.v[0].float().view(-1, 256) * opt.v_scale[0][:, None]
    want = 1 - 0.999 ** 300
    mean = float(v[:, 1:].double().mean())
    # steps of a code are at most a quarter of the value: standard deviation below sqrt(300) / 8 of it, over sqrt(65280) elements
    assert abs(mean - want) < 5 * want * (300 ** 0.5 / 8) / 65280 ** 0.5
    m = opt.m[0].float().view(-1, 256) * opt.m_scale[0][:, None]
    assert abs(float(m[:, 1:].double().mean()) - 1.0) < 5 * 0.25 / 65280 ** 0.5


def test_a_non_finite_value_poisons_its_block_only():
    from gemmaedge_amd import head as H

    p, g = rand(2000, 1, 1.0), rand(2000, 2, 1e-3)
    g[300], g[1999] = float("inf"), float("nan")
    opt = H.AdamW([p], [g], state_bits=8)
    opt.step()
    bad = torch.zeros(8, dtype=torch.bool, device="cuda")
    bad[1] = bad[7] = True
    assert torch.equal(torch.isnan(opt.m_scale[0]), bad) and torch.equal(torch.isnan(opt.v_scale[0]), bad)
    assert int((~torch.isfinite(p)).sum()) == 2
    g.zero_()
    opt.step()
    assert torch.isfinite(p[:256]).all() and torch.isnan(p[256:512]).all()


def test_replayed_steps_read_their_parameters_from_the_device():
    from gemmaedge_amd import head as H

    for bits in (8, 32):
        make = lambda: ([rand(n, 3 + i, 0.05) for i, n in enumerate((5000, 77))], [rand(n, 9 + i, 1e-3) for i, n in enumerate((5000, 77))])  # noqa: E731
        (pa, ga), (pb, gb) = make(), make()
        a, b = H.AdamW(pa, ga, state_bits=bits, seed=5), H.AdamW(pb, gb, state_bits=bits, seed=5)
        hp = b.device_params()
        b.step(device_params=hp)  # a launch before the capture
        a.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b.step(device_params=hp)
        for step in range(4):
            lr = 1e-3 / (step + 1)
            a.step(lr=lr, grad_scale=0.5)
            b.device_params(lr=lr, grad_scale=0.5, out=hp)
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(pa + a.m + a.v, pb + b.m + b.v):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), (bits, step)
        assert a.steps == b.steps == 5


def test_refusals():
    from gemmaedge_amd import head as H
    from gemmaedge_amd import sampler as S

    p, g = rand(300, 1, 1.0), rand(300, 2, 1.0)
    for bad in (lambda: H.AdamW([p], []), lambda: H.AdamW([p], [g[:10]]), lambda: H.AdamW([p.double()], [g]), lambda: H.AdamW([p], [g.cpu()]),
                lambda: H.AdamW([p[::2]], [g[::2]]), lambda: H.AdamW([p], [g], masters=[p.bfloat16()]), lambda: H.AdamW([p], [g], m=[g.bfloat16()]),
                lambda: H.AdamW([p], [g], state_bits=8, m_scale=[g])):
        with pytest.raises(ValueError):
            bad()
    opt = H.AdamW([p], [g])
    for kw in (dict(lr=float("inf")), dict(grad_scale=float("nan"))):
        with pytest.raises(S.SamplerError) as e:
            opt.step(**kw)
        assert e.value.code == S.GE_ERR_INVALID_ARG
    assert opt.steps == 0
