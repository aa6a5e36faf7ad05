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
