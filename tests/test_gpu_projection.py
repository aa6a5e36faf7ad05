"""The projection with adapters and its gradients on the GPU against float64.

Tolerances, u = 2^-24. A sum of K products is off by at most 2 (K + 64) u of the
sum of their magnitudes (float32 adds, whose order is the hardware's; operands of
float32 leave out 4 u of a product). u and du carry that error and their
own rounding, 2^-17 where bf16 operands hold them in two bf16 numbers; both go
through the sums they enter. Outputs are rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(rows, dim, out, rank, adapters, dt, seed=1, pad=0, runs=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(hidden=rn(max(rows, 1), dim + pad).to(dt)[:rows, :dim], weight=(rn(out, dim + pad) / dim ** 0.5).to(dt)[:, :dim])
    if adapters:
        s.update(a=(rn(adapters, rank, dim) / dim ** 0.5).to(dt), b=(rn(adapters, out, rank) / rank ** 0.5).to(dt), scale=0.5 + rn(adapters).abs())
        ids = torch.randint(adapters + 2, (rows // runs + 1,), generator=g, device="cuda", dtype=torch.int32)
        wild = torch.tensor([-1, -2 ** 31, adapters, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
        ids = torch.where(ids < adapters, ids, wild[torch.arange(len(ids), device="cuda") % 4])
        s["adapter"] = ids.repeat_interleave(runs)[:rows].contiguous()
    dout = (rn(max(rows, 1), out + pad) / max(rows, 1)).to(dt)[:rows, :out]
    return s, dout


def mm(x, y, xe, ye):
    """x @ y, and its error for operands off by xe and ye (None: exact), summed in float32."""
    size = x.abs() @ y.abs()
    e = 2 * (x.shape[1] + 64) * U * size + 4 * U * size
    if xe is not None:
        e = e + xe @ y.abs()
    if ye is not None:
        e = e + x.abs() @ ye
    return x @ y, e


def reference(s, dout, dtype):
    h, w, g = s["hidden"].double(), s["weight"].double(), dout.double()
    out, e_out = mm(h, w.t(), None, None)
    dh, e_dh = mm(g, w, None, None)
    ref = {}
    if "a" in s:
        half = 2.0 ** -17 if dtype == torch.bfloat16 else U
        da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
        e_da, e_db = torch.zeros_like(da), torch.zeros_like(db)
        for k in range(s["a"].shape[0]):
            at = torch.nonzero(s["adapter"] == k)[:, 0]
            a, b, c = s["a"][k].double(), s["b"][k].double(), float(s["scale"][k])
            u, e_u = mm(h[at], a.t(), None, None)
            u, e_u = c * u, c * e_u
            e_u = e_u + (half + U) * (u.abs() + e_u)
            du, e_du = mm(g[at], b, None, None)
            du, e_du = c * du, c * e_du
            e_du = e_du + (half + U) * (du.abs() + e_du)
            y, e = mm(u, b.t(), e_u, None)
            out[at] += y
            e_out[at] += e + 2 * U * (e + y.abs())
            y, e = mm(du, a, e_du, None)
            dh[at] += y
            e_dh[at] += e + 2 * U * (e + y.abs())
            da[k], e_da[k] = mm(du.t(), h[at], e_du.t(), None)
            db[k], e_db[k] = mm(g[at].t(), u, None, e_u)
        ref.update(da=(da, e_da), db=(db, e_db))
    e_out = e_out + 2 * U * out.abs()
    e_dh = e_dh + 2 * U * dh.abs()
    return dict(ref, out=(out, e_out), dh=(dh, e_dh))


def close(got, ref, what):
    want, err = ref
    assert got.shape == want.shape, what
    tol = err + torch.finfo(got.dtype).eps / 2 * (want.abs() + err) + 1e-37
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((off / tol).max()):.3g} tolerances"


def check(rows, dim, out, rank, adapters, dt, odt=None, pad=0, seed=1, handle=None, runs=1, train=True):
    from gemmaedge_amd import projection as P

    s, dout = inputs(rows, dim, out, rank, adapters, DT[dt], seed, pad, runs)
    p = handle or P.Projection(max(rows, 1), dim, out, rank if adapters else 0, adapters, dtype=DT[dt], train=train)
    got = dict(out=p.project(**s, out_dtype=DT[odt] if odt else None))
    if train:
        got["dh"], got["da"], got["db"] = p.project_backward(dout, **s)
    torch.cuda.synchronize()
    assert got["out"].dtype == DT[odt or dt]
    ref = reference(s, dout, DT[dt])
    for k, t in got.items():
        if t is not None:
            close(t, ref[k], k)
    assert not train or (got["da"] is None) == (adapters == 0)
    return p


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,dim,out,rank,adapters,pad", [
    (1, 1, 1, 1, 1, 0), (1, 8, 2, 0, 0, 0), (2, 64, 127, 4, 1, 0), (7, 33, 255, 5, 3, 0), (16, 72, 256, 8, 2, 8), (17, 100, 257, 16, 5, 4),
    (33, 64, 1000, 17, 9, 1), (64, 136, 1003, 32, 40, 0), (65, 64, 512, 12, 4, 64), (129, 200, 300, 64, 7, 0), (255, 96, 5003, 33, 3, 0),
    (256, 64, 256, 65, 2, 0), (257, 328, 999, 7, 30, 0), (300, 1001, 700, 16, 6, 0), (600, 257, 2049, 100, 2, 3), (40, 512, 640, 256, 3, 0),
    (1000, 96, 1025, 0, 0, 0)])
def test_projection(rows, dim, out, rank, adapters, pad, dt):
    check(rows, dim, out, rank, adapters, dt, pad=pad)


@pytest.mark.parametrize("dt,odt", (("bf16", "f32"), ("f32", "bf16")))
@pytest.mark.parametrize("rows,out", ((3, 1001), (100, 520), (300, 777)))
def test_other_output_type(rows, out, dt, odt):
    check(rows, 160, out, 8, 3, dt, odt, train=False)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_sequences_and_smaller_calls_on_a_larger_handle(dt):
    from gemmaedge_amd import projection as P

    p = P.Projection(700, 512, 3000, 64, 20, dtype=DT[dt], train=True)
    for rows, dim, out, rank, adapters, runs in ((700, 512, 3000, 64, 20, 40), (3, 40, 2000, 8, 2, 1), (65, 512, 77, 20, 20, 13), (1, 7, 3000, 3, 1, 1),
                                                 (200, 129, 300, 0, 0, 1), (513, 256, 640, 33, 4, 100)):
        check(rows, dim, out, rank, adapters, dt, handle=p, seed=rows, runs=runs)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_packed_pieces(dt):
    # Rows of 1,001 elements: 32,768 rows of the weight are packed at a time.
    check(5, 1001, 33333, 6, 3, dt, seed=4)


def test_pieces_of_dout():
    # 256 MiB of packed rows hold 32,768 outputs of 4,096 rows: two pieces.
    check(4096, 64, 40001, 8, 3, "bf16", seed=9, runs=50)


def test_pieces_of_more_rows_than_a_grid_has():
    # dhidden's parts of 70,001 rows, whose dout is packed 1,792 outputs at a time.
    check(70001, 36, 1801, 4, 2, "bf16", seed=5, runs=700)


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_rows_far_apart(dt):
    """Rows whose offsets in a tile pass 31 bits are packed first."""
    from gemmaedge_amd import projection as P

    far = (1 << 21) + 16
    s, dout = inputs(20, 64, 70, 8, 3, DT[dt])
    p = P.Projection(20, 64, 70, 8, 3, dtype=DT[dt], train=True)
    want = [p.project(**s), *p.project_backward(dout, **s)]
    apart = dict(s)
    for k in ("hidden", "weight"):
        wide = torch.empty(s[k].shape[0], far, device="cuda", dtype=DT[dt])
        wide[:, :64] = s[k]
        apart[k] = wide[:, :64]
    wide = torch.empty(20, far, device="cuda", dtype=DT[dt])
    wide[:, :70] = dout
    got = [p.project(**apart), *p.project_backward(wide[:, :70], **apart)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_many_adapters():
    check(500, 128, 400, 4, 700, "bf16")
    check(300, 64, 200, 4, 700, "f32")


@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows", (5, 70, 300))
def test_no_number_stays_with_its_request(rows, dt):
    """Infinities and NaN in one adapter and in one row: the other rows' results are what they are without."""
    from gemmaedge_amd import projection as P

    s, dout = inputs(rows, 96, 500, 8, 4, DT[dt], seed=3)
    s["adapter"] = (torch.arange(rows, device="cuda") % 5).int()  # 4: none
    p = P.Projection(rows, 96, 500, 8, 4, dtype=DT[dt], train=True)
    out = p.project(**s).clone()
    dh, da, db = p.project_backward(dout, **s)
    bad = {k: v.clone() for k, v in s.items()}
    bad["a"][2, :, ::3] = float("inf")
    bad["b"][2, ::7] = float("nan")
    bad["hidden"][2, 5] = float("nan")  # a row of that adapter
    dbad = dout.clone()
    dbad[2, 11] = float("inf")
    out2 = p.project(**bad)
    dh2, da2, db2 = p.project_backward(dbad, **bad)
    mine = s["adapter"] == 2
    assert torch.equal(out[~mine], out2[~mine]) and torch.equal(dh[~mine], dh2[~mine])
    keep = [0, 1, 3]
    assert torch.equal(da[keep], da2[keep]) and torch.equal(db[keep], db2[keep])
    assert torch.isnan(out2[2]).any() and not torch.isfinite(dh2[2]).all()


def test_no_rows_and_no_adapters():
    from gemmaedge_amd import projection as P

    s, dout = inputs(0, 65, 300, 5, 3, torch.float32)
    p = P.Projection(7, 65, 300, 5, 3, dtype=torch.float32, train=True)
    assert p.project(**s).shape == (0, 300)
    da, db = torch.full_like(s["a"], 7.0), torch.full_like(s["b"], 7.0)
    dh, da, db = p.project_backward(dout, **s, da=da, db=db)
    assert dh.shape == (0, 65) and not da.any() and not db.any()
    # every row without an adapter
    s, dout = inputs(6, 65, 300, 5, 3, torch.float32)
    s["adapter"].fill_(-1)
    plain = {k: s[k] for k in ("hidden", "weight")}
    assert torch.equal(p.project(**s), p.project(**plain))
    dh, da, db = p.project_backward(dout, **s)
    assert torch.equal(dh, p.project_backward(dout, **plain)[0]) and not da.any() and not db.any()
    assert p.project_backward(dout, **plain)[1:] == (None, None)


def test_wanted_gradients_alone():
    from gemmaedge_amd import projection as P

    s, dout = inputs(70, 64, 300, 5, 3, torch.bfloat16)
    p = P.Projection(70, 64, 300, 5, 3, train=True)
    dh, da, db = p.project_backward(dout, **s)
    assert torch.equal(p.project_backward(dout, **s, need_adapters=False)[0], dh)
    none, da2, db2 = p.project_backward(dout, **s, need_hidden=False)
    assert none is None and torch.equal(da, da2) and torch.equal(db, db2)
    only = torch.empty_like(db)
    assert p.project_backward(dout, **s, need_hidden=False, need_adapters=False, db=only)[1] is None and torch.equal(only, db)


def test_strided_outputs_leave_what_lies_between():
    from gemmaedge_amd import projection as P

    s, dout = inputs(70, 64, 300, 5, 3, torch.bfloat16)
    p = P.Projection(70, 64, 300, 5, 3, train=True)
    wide = torch.full((70, 331), 9.0, device="cuda")
    out = p.project(**s, out=wide[:, :300])
    assert torch.equal(out, p.project(**s, out_dtype=torch.float32)) and bool((wide[:, 300:] == 9).all())
    wide = torch.full((70, 75), 9.0, device="cuda", dtype=torch.bfloat16)
    dh = p.project_backward(dout, **s, dhidden=wide[:, :64])[0]
    assert torch.equal(dh, p.project_backward(dout, **s)[0]) and bool((wide[:, 64:] == 9).all())


def test_gradients_against_differences():
    from gemmaedge_amd import projection as P

    s, dout = inputs(6, 24, 60, 4, 2, torch.float32, seed=8)
    s["adapter"] = torch.tensor([0, 1, -1, 1, 0, 1], device="cuda", dtype=torch.int32)
    p = P.Projection(6, 24, 60, 4, 2, dtype=torch.float32, train=True)
    grads = dict(zip(("hidden", "a", "b"), p.project_backward(dout, **s)))

    def value(**kw):
        return float((p.project(**dict(s, **kw)).double() * dout.double()).sum())

    for name, grad in grads.items():
        g = torch.Generator(device="cuda").manual_seed(5)
        step = torch.randn(s[name].shape, generator=g, device="cuda")
        h = 2.0 ** -4  # the objective is at most quadratic along a step in one operand: differences are exact but for rounding
        got = (value(**{name: s[name] + h * step}) - value(**{name: s[name] - h * step})) / (2 * h)
        want = float((grad.double() * step.double()).sum())
        # float32 sums of 24 + 4 and rounded operands, over the step: 2^-24 x 100 x the objective's magnitudes / h
        size = float((p.project(**{k: (v.abs() if v.is_floating_point() else v) for k, v in s.items()}).double() * dout.double().abs()).sum())
        assert abs(got - want) <= 100 * U * size * 4 / h, name


def test_graph():
    """A captured forward and backward pass over new inputs in the same memory."""
    from gemmaedge_amd import projection as P

    rows, dim, out = 130, 96, 700
    s, dout = inputs(rows, dim, out, 8, 5, torch.bfloat16)
    p = P.Projection(rows, dim, out, 8, 5, train=True)
    q = P.Projection(rows, dim, out, 8, 5, train=True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        p.project(**s)
        p.project_backward(dout, **s)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [p.project(**s), *p.project_backward(dout, **s)]
    for seed in range(2, 6):
        new, dnew = inputs(rows, dim, out, 8, 5, torch.bfloat16, seed=seed)
        for k in s:
            s[k].copy_(new[k])
        dout.copy_(dnew)
        want = [q.project(**new), *q.project_backward(dnew, **new)]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_another_stream_and_dropped_tensors():
    from gemmaedge_amd import projection as P

    s, dout = inputs(200, 256, 3000, 8, 5, torch.bfloat16)
    p = P.Projection(200, 256, 3000, 8, 5, train=True)
    want = [p.project(**s), *p.project_backward(dout, **s)]
    torch.cuda.synchronize()
    copies, dcopy = {k: v.clone() for k, v in s.items()}, dout.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    got = [p.project(**copies, stream=side), *p.project_backward(dcopy, **copies, stream=side)]
    del copies, dcopy
    junk = [torch.full((600_000,), 7.0, device="cuda") for _ in range(8)]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert len(junk) == 8


def test_refusals():
    from gemmaedge_amd import projection as P
    from gemmaedge_amd import sampler as S

    s, dout = inputs(8, 64, 300, 5, 3, torch.bfloat16)
    p = P.Projection(8, 64, 300, 5, 3)
    t = P.Projection(8, 64, 300, 5, 3, train=True)
    for kw in (dict(adapter=None), dict(a=s["a"][:, :, :63]), dict(a=s["a"].float()), dict(b=s["b"][:2]), dict(b=s["b"].transpose(1, 2)),
               dict(scale=s["scale"].bfloat16()), dict(scale=s["scale"][:2]), dict(adapter=s["adapter"].long()), dict(adapter=s["adapter"][:7]),
               dict(hidden=s["hidden"].float()), dict(hidden=s["hidden"][0]), dict(weight=s["weight"][:, :60]), dict(hidden=s["hidden"].t()),
               dict(hidden=s["hidden"].cpu())):
        with pytest.raises(ValueError):
            p.project(**dict(s, **kw))
    for kw in (dict(out_dtype=torch.float16), dict(out=torch.empty(8, 299, device="cuda")),
               dict(out=torch.empty(8, 300, device="cuda"), out_dtype=torch.bfloat16), dict(out=torch.empty(300, 8, device="cuda").t())):
        with pytest.raises(ValueError):
            p.project(**s, **kw)
    with pytest.raises(S.SamplerError, match="without train"):
        p.project_backward(dout, **s)
    for kw in (dict(dhidden=torch.empty(8, 64, device="cuda")), dict(da=torch.empty_like(s["b"])),
               dict(db=torch.empty(3, 5, 300, device="cuda", dtype=torch.bfloat16).transpose(1, 2))):
        with pytest.raises(ValueError):
            t.project_backward(dout, **s, **kw)
    with pytest.raises(ValueError):
        t.project_backward(dout.float(), **s)
    with pytest.raises(ValueError):
        t.project_backward(dout, s["hidden"], s["weight"], da=torch.empty_like(s["a"]))
    big, _ = inputs(9, 64, 300, 5, 3, torch.bfloat16)
    with pytest.raises(S.SamplerError, match="capacity"):
        p.project(**big)
    with pytest.raises(S.SamplerError, match="capacity"):
        P.Projection(8, 64, 300).project(**s)
