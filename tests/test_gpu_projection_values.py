"""What the projection holds between its sums: the rows' low-rank values u and du.

Inputs are chosen so that every float32 sum of them is exact in any order (integers below 2^24
times a power of two), and so that an output is one value's product with a power of two. What
comes out is then the value as it was held, in float32 outputs bit by bit, and
in bf16 ones by the side of a halfway point on which it lies: the tolerance is 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def values(rows, halfway, seed):
    """[rows, 3] whole numbers whose sum with 2^16, 2^8 and 1 has 24 bits, and that sum with a sign a row.
    halfway: 2^-16 of the first 8 bits' last away from the middle of two bf16 numbers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.randint(256, (rows, 3), generator=g, device="cuda")
    c[:, 0] = c[:, 0] | 128
    if halfway:
        above = torch.arange(rows, device="cuda") % 2 == 0
        c[:, 1], c[:, 2] = torch.where(above, 128, 127), torch.where(above, 1, 255)
    sign = 1 - 2 * torch.randint(2, (rows, 1), generator=g, device="cuda")
    c = c * sign
    return c, (c * torch.tensor([65536, 256, 1], device="cuda")).sum(1).double()


POWERS = torch.tensor([2.0 ** -4, 2.0 ** -12, 2.0 ** -20])


def table(adapters, rank, cols):
    """[adapters, rank, cols]: 2^16, 2^8, 1 in three columns times 2^-20 and a power of two of the rank and the adapter; and those powers."""
    p = 2.0 ** -(torch.arange(rank)[None, :] % 5).double() * 2.0 ** (torch.arange(adapters)[:, None] % 3)
    t = torch.zeros(adapters, rank, cols, dtype=torch.float64)
    t[:, :, :3] = p[:, :, None] * POWERS.double()
    return t.cuda(), (p * 2.0 ** -20).cuda()


SHAPES = [(1, 8, 40, 1, 1), (5, 72, 300, 8, 2), (40, 64, 513, 5, 9), (64, 128, 256, 33, 4), (100, 33, 129, 20, 3), (300, 96, 515, 16, 5),
          (700, 130, 260, 64, 2), (130, 64, 700, 100, 3)]


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,out,rank,adapters", SHAPES)
def test_u(rows, dim, out, rank, adapters, dt):
    """u in the projection's float32 output, and in dB."""
    from gemmaedge_amd import projection as P

    d = DT[dt]
    ids = (torch.arange(rows, device="cuda") * 7 % (adapters + 1)).int()  # the last: none
    p = P.Projection(rows, dim, out, rank, adapters, dtype=d, train=True)
    a, unit = table(adapters, rank, dim)
    weight = torch.zeros(out, dim, device="cuda", dtype=d)
    b = torch.zeros(adapters, out, rank, device="cuda", dtype=d)
    at = torch.arange(out, device="cuda")
    b[:, at, at % rank] = torch.where(at % 3 == 0, -2.0, 0.5).to(d)
    scale = torch.ones(adapters, device="cuda")
    have = ids < adapters
    k = ids.clamp_max(adapters - 1).long()

    c, number = values(rows, False, rows)
    hidden = torch.zeros(rows, dim, device="cuda", dtype=d)
    hidden[:, :3] = c.to(d)
    u = number[:, None] * unit[k] * have[:, None]
    want = u[:, at % rank] * torch.where(at % 3 == 0, -2.0, 0.5)
    got = p.project(hidden, weight, a.to(d), b, scale, ids, out_dtype=torch.float32)
    assert torch.equal(got.double(), want)

    # dB: one row of each adapter has a gradient, a power of two
    c, number = values(rows, True, rows + 1)
    hidden[:, :3] = c.to(d)
    u = number[:, None] * unit[k]
    dout = torch.zeros(rows, out, device="cuda", dtype=d)
    want = torch.zeros(adapters, out, rank, device="cuda", dtype=torch.float64)
    for i in range(adapters):
        mine = torch.nonzero(ids == i)[:, 0]
        if len(mine):
            n = int(mine[len(mine) * 2 // 3])
            dout[n] = torch.where(at % 2 == 0, 0.25, -1.0).to(d)
            want[i] = torch.where(at % 2 == 0, 0.25, -1.0).double()[:, None] * u[n]
    _, _, db = p.project_backward(dout, hidden, weight, a.to(d), b, scale, ids)
    assert torch.equal(db, want.to(torch.float32).to(d))


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,out,rank,adapters", SHAPES)
def test_du(rows, dim, out, rank, adapters, dt):
    """du in dhidden and in dA."""
    from gemmaedge_amd import projection as P

    d = DT[dt]
    ids = (torch.arange(rows, device="cuda") * 7 % (adapters + 1)).int()
    p = P.Projection(rows, dim, out, rank, adapters, dtype=d, train=True)
    b, unit = table(adapters, rank, out)
    weight = torch.zeros(out, dim, device="cuda", dtype=d)
    a = torch.zeros(adapters, rank, dim, device="cuda", dtype=d)
    at = torch.arange(dim, device="cuda")
    a[:, at % rank, at] = torch.where(at % 3 == 0, -2.0, 0.5).to(d)
    scale = torch.ones(adapters, device="cuda")
    have = ids < adapters
    k = ids.clamp_max(adapters - 1).long()

    c, number = values(rows, True, rows)
    dout = torch.zeros(rows, out, device="cuda", dtype=d)
    dout[:, :3] = c.to(d)
    du = number[:, None] * unit[k] * have[:, None]
    hidden = torch.zeros(rows, dim, device="cuda", dtype=d)
    want = torch.zeros(adapters, rank, dim, device="cuda", dtype=torch.float64)
    for i in range(adapters):
        mine = torch.nonzero(ids == i)[:, 0]
        if len(mine):
            n = int(mine[len(mine) * 2 // 3])
            hidden[n] = torch.where(at % 2 == 0, 0.25, -1.0).to(d)
            want[i] = du[n][:, None] * torch.where(at % 2 == 0, 0.25, -1.0).double()
    dh, da, _ = p.project_backward(dout, hidden, weight, a, b.transpose(1, 2).contiguous().to(d), scale, ids)
    assert torch.equal(dh, (du[:, at % rank] * torch.where(at % 3 == 0, -2.0, 0.5)).to(torch.float32).to(d))
    assert torch.equal(da, want.to(torch.float32).to(d))


def whole(g, *shape):
    """Whole numbers of 1 to 3 and their negatives: every sum of their products is exact."""
    return torch.randint(1, 4, shape, generator=g) * (1 - 2 * torch.randint(2, shape, generator=g))


def definition(s, dout):
    """The formulas, a product and a sum at a time, in float64 on the CPU."""
    h, w, g = s["hidden"].double(), s["weight"].double(), dout.double()
    def mm(x, y):  # noqa: E306
        return (x[:, :, None] * y[None]).sum(1)
    out, dh = mm(h, w.t()), mm(g, w)
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    for k in range(len(s["scale"])):
        at = torch.nonzero(s["adapter"] == k)[:, 0]
        a, b, c = s["a"][k].double(), s["b"][k].double(), s["scale"][k].double()
        u, du = c * mm(h[at], a.t()), c * mm(g[at], b)
        out[at] += mm(u, b.t())
        dh[at] += mm(du, a)
        da[k], db[k] = mm(du.t(), h[at]), mm(g[at].t(), u)
    return dict(out=out, dh=dh, da=da, db=db)


@pytest.mark.parametrize("where", ("a", "b", "hidden", "dout", "scale"))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,out,rank", [(4, 24, 33, 1), (40, 17, 130, 3), (130, 40, 70, 1), (300, 30, 65, 20)])
def test_an_infinity_gives_what_the_definition_gives(rows, dim, out, rank, dt, where):
    """One infinity in an operand: infinities and NaN of the definition, where it has them, and its numbers elsewhere."""
    from gemmaedge_amd import projection as P

    d = DT[dt]
    g = torch.Generator().manual_seed(rows + rank)
    s = dict(hidden=whole(g, rows, dim), weight=whole(g, out, dim), a=whole(g, 3, rank, dim), b=whole(g, 3, out, rank))
    s = {k: v.to(d) for k, v in s.items()}
    s["scale"], s["adapter"] = torch.tensor([1.0, 2.0, 0.5]), (torch.arange(rows) % 4).int()
    dout = whole(g, rows, out).to(d)
    t = dout if where == "dout" else s[where]
    if where == "scale":
        t[1] = -float("inf")
    elif t.dim() == 2:
        t[1, 5] = -float("inf")
    else:
        t[1, t.shape[1] // 2, t.shape[2] // 3] = float("inf")
    want = definition(s, dout)
    p = P.Projection(rows, dim, out, rank, 3, dtype=d, train=True)
    on = {k: v.cuda() for k, v in s.items()}
    got = dict(out=p.project(**on, out_dtype=torch.float32))
    got["dh"], got["da"], got["db"] = (x for x in p.project_backward(dout.cuda(), **on))
    for k, x in got.items():
        x, y = x.cpu(), want[k].to(torch.float32).to(x.dtype)
        if dt == "f32" and (where, k) in (("hidden", "out"), ("dout", "dh")):  # through the weight's product: NaN
            assert not torch.isfinite(x[1]).any(), k
            x, y = x.clone(), y.clone()
            x[1] = y[1] = 0
        assert torch.equal(torch.isnan(x), torch.isnan(y)), k
        assert torch.equal(torch.nan_to_num(x, nan=0.0, posinf=float("inf"), neginf=-float("inf")),
                           torch.nan_to_num(y, nan=0.0, posinf=float("inf"), neginf=-float("inf"))), k
    assert not all(torch.isfinite(v).all() for v in want.values())


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("out", (1, 1001, 1008))
def test_no_rows(out, dt):
    from gemmaedge_amd import projection as P

    d = DT[dt]
    p = P.Projection(3, 65, 1008, 5, 2, dtype=d, train=True)
    s = dict(hidden=torch.empty(0, 65), weight=torch.randn(out, 65), a=torch.randn(2, 5, 65), b=torch.randn(2, out, 5))
    s = {k: v.to(d).cuda() for k, v in s.items()}
    s.update(scale=torch.ones(2, device="cuda"), adapter=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert p.project(**s).shape == (0, out)
    dh, da, db = p.project_backward(torch.empty(0, out, dtype=d, device="cuda"), **s, da=torch.ones_like(s["a"]), db=torch.ones_like(s["b"]))
    assert dh.shape == (0, 65) and not da.any() and not db.any()
    assert p.project_backward(torch.empty(0, out, dtype=d, device="cuda"), s["hidden"], s["weight"])[0].shape == (0, 65)


def test_outputs_apart_from_all_else():
    """An output over an operand is refused and leaves everything as it was; columns of one buffer are apart."""
    from gemmaedge_amd import projection as P
    from gemmaedge_amd import sampler as S

    g = torch.Generator().manual_seed(2)
    s = dict(hidden=whole(g, 40, 64), weight=whole(g, 64, 64), a=whole(g, 3, 4, 64), b=whole(g, 3, 64, 4))
    s = {k: v.bfloat16().cuda() for k, v in s.items()}
    s.update(scale=torch.ones(3, device="cuda"), adapter=(torch.arange(40, device="cuda") % 4).int())
    dout = whole(g, 40, 64).bfloat16().cuda()
    p = P.Projection(40, 64, 64, 4, 3, train=True)
    before = {k: v.clone() for k, v in s.items()}
    for out in (s["hidden"], s["weight"][24:], s["a"].view(-1)[:512].view(8, 64)):
        n = out.shape[0]
        with pytest.raises(S.SamplerError, match="overlaps"):
            p.project(s["hidden"][:n], s["weight"], s["a"], s["b"], s["scale"], s["adapter"][:n], out=out)
    for kw in (dict(dhidden=s["hidden"]), dict(dhidden=dout), dict(da=s["a"]), dict(db=s["b"]), dict(da=s["weight"].view(-1)[:768].view(3, 4, 64))):
        with pytest.raises(S.SamplerError, match="overlaps"):
            p.project_backward(dout, **s, **kw)
    both = torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(S.SamplerError, match="overlaps"):
        p.project_backward(dout, **s, da=both, db=both.view(3, 64, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(s[k], before[k]) for k in s)
    wide = torch.zeros(40, 192, device="cuda", dtype=torch.bfloat16)
    wide[:, :64] = s["hidden"]
    wide[:, 128:] = dout
    want, got = p.project(**s), p.project(**dict(s, hidden=wide[:, :64]), out=wide[:, 64:128])
    assert torch.equal(got, want)
    dh = p.project_backward(wide[:, 128:], **dict(s, hidden=wide[:, :64]), dhidden=wide[:, 64:128])[0]
    assert torch.equal(dh, p.project_backward(dout, **s)[0])
