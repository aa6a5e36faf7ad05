"""Penalties, biases and masks on the GPU against float64, and against the sampler's
own softcap and penalty bit for bit.

Tolerance, u = 2^-24: the softcap is a quotient, a tanh within 1 ulp and a product
(4 u of its value), the repetition penalty one operation, f * c, the two
subtractions and the bias one each: 8 u of the sum of the magnitudes they take,
and one rounding to the output's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
INF = math.inf


def lists(gen, rows, most, vocab, wild=True):
    """Offsets and ids of ragged rows, some empty, some ids outside the vocabulary."""
    n = torch.randint(most + 1, (rows,), generator=gen, device="cuda")
    n[0] = most
    if rows > 2:
        n[2] = 0
    offs = torch.cat([torch.zeros(1, device="cuda", dtype=torch.long), torch.cumsum(n, 0)]).int()
    total = int(offs[-1])
    ids = (vocab * torch.rand(total, generator=gen, device="cuda") ** 3).int().clamp_max(vocab - 1)
    if wild and total:
        ids[::11] = torch.tensor([-1, vocab, 2 ** 31 - 1, -2 ** 31], device="cuda", dtype=torch.int32)[
            torch.arange((total + 10) // 11, device="cuda") % 4]
    return offs, ids


def reference(x, cfgs, hist, prompt, bias, ok):
    """(value, magnitude) in float64 for rows of ids and (id, bias) pairs."""
    x = x.double()
    rows, v = x.shape
    want, size = torch.empty_like(x), torch.empty_like(x)
    for i in range(rows):
        c = cfgs[i]
        y = c.softcap * torch.tanh(x[i] / c.softcap) if c.softcap > 0 else x[i].clone()
        seen, count = torch.zeros(v, dtype=torch.bool), torch.zeros(v, dtype=torch.float64)
        for k, t in enumerate(hist[i]):
            if 0 <= t < v:
                seen[t] = True
                count[t] += k >= prompt[i]
        seen, count = seen.to(x.device), count.to(x.device)
        y = torch.where(seen, torch.where(y > 0, y / c.repetition_penalty, y * c.repetition_penalty), y)
        s = y.abs()
        y = torch.where(count > 0, y - c.frequency_penalty * count - c.presence_penalty, y)
        s = s + count * abs(c.frequency_penalty) + abs(c.presence_penalty)
        last = {t: b for t, b in bias[i] if 0 <= t < v}
        if last:
            at = torch.tensor(list(last), device=x.device)
            b = torch.tensor(list(last.values()), device=x.device, dtype=torch.float64)
            y[at] += b
            s[at] += b.abs()
        want[i] = torch.where(ok[i], y, -INF)
        size[i] = s
    return want, size


def close(got, want, size):
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got.double()[rest], want[rest])
    err = 8 * U * size[fine]
    tol = err + torch.finfo(got.dtype).eps / 2 * (want[fine].abs() + err) + 1e-44
    off = (got.double()[fine] - want[fine]).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def config(i, cap):
    from gemmaedge_amd import rules as R

    return R.RuleConfig(cap * (1 + i % 3), (1.0, 1.3, 0.7)[i % 3], (0.0, 0.5, -0.25)[i % 3], (0.2, 0.0, 1.5)[i % 3])


def make(rows, vocab, dt, history=0, bias=0, masks=False, cap=0.0, per_row=False, pad=0, seed=1):
    from gemmaedge_amd import rules as R

    g = torch.Generator(device="cuda").manual_seed(seed)
    base = (4 * torch.randn(rows, vocab + pad, generator=g, device="cuda")).to(DT[dt])
    kw, ref = {}, dict(hist=[[]] * rows, bias=[[]] * rows, prompt=[0] * rows)
    if history:
        offs, ids = lists(g, rows, history, vocab)
        prompt = torch.randint(history + 2, (rows,), generator=g, device="cuda", dtype=torch.int32)
        kw.update(history=ids, history_offsets=offs, prompt_len=prompt)
        o, t = offs.tolist(), ids.tolist()
        ref["hist"], ref["prompt"] = [t[o[i]:o[i + 1]] for i in range(rows)], prompt.tolist()
    if bias:
        offs, ids = lists(g, rows, bias, vocab)
        vals = 3 * torch.randn(ids.numel(), generator=g, device="cuda")
        vals[::7] = -INF
        vals[5::13] = INF
        kw.update(bias_ids=ids, bias_values=vals, bias_offsets=offs)
        o, t, b = offs.tolist(), ids.tolist(), vals.tolist()
        ref["bias"] = [list(zip(t[o[i]:o[i + 1]], b[o[i]:o[i + 1]])) for i in range(rows)]
    ok = torch.ones(rows, vocab, dtype=torch.bool, device="cuda")
    if masks:
        n, words = rows + 1, -(-vocab // 32)
        m = torch.randint(-2 ** 31, 2 ** 31, (n, words + 2), generator=g, device="cuda").int()
        m[1] = -1                                           # everything
        m[2 % n] = 0                                        # nothing
        if vocab % 32 and n > 3:
            m[3] = 0
            m[3, vocab // 32] = -1 << (vocab % 32)          # bits behind the vocabulary alone: nothing
        m = m[:, :words]                                    # words apart in memory
        which = (torch.arange(rows, device="cuda") * 3 + 1) % (n + 2) - 1  # -1 and n: none
        kw.update(mask=m, mask_rows=which.int())
        bits = (m[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().reshape(n, -1)[:, :vocab]
        none = (which < 0) | (which >= n)
        ok = bits[which.clamp(0, n - 1)] | none[:, None]
    cfgs = [config(i if per_row else 1, cap) for i in range(rows)]
    if per_row:
        kw["row_params"] = R.row_params(cfgs)
    else:
        kw["config"] = cfgs[0]
    return base, kw, ref, ok, cfgs


@pytest.mark.parametrize("to", ("new", "inplace", "f32", "bf16"))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
@pytest.mark.parametrize("rows,vocab,history,bias,masks,cap,per_row,pad", [
    (1, 1, 3, 2, True, 0.0, False, 0), (1, 7, 0, 0, False, 30.0, False, 0), (3, 8, 9, 0, False, 0.0, True, 1),
    (5, 33, 40, 9, True, 2.0, True, 0), (4, 2048, 0, 5, False, 0.0, False, 0), (6, 2049, 700, 0, True, 0.0, False, 3),
    (9, 4100, 5000, 300, True, 0.0, True, 8), (2, 50257, 9000, 70, True, 30.0, False, 0), (7, 20001, 0, 0, True, 0.0, False, 0),
    (150, 33001, 90, 20, True, 0.0, True, 0), (70, 70000, 40, 0, False, 0.0, False, 2), (65, 66000, 300, 30, True, 30.0, True, 0),
    (3, 262144, 4097, 40, False, 0.0, False, 0), (100, 70001, 6001, 20, True, 0.0, True, 0), (90, 70001, 50, 6001, False, 0.0, False, 0)])
def test_rules(rows, vocab, history, bias, masks, cap, per_row, pad, dt, to):
    from gemmaedge_amd import rules as R

    base, kw, ref, ok, cfgs = make(rows, vocab, dt, history, bias, masks, cap, per_row, pad)
    x = base[:, :vocab]
    before = base.clone()
    want, size = reference(x, cfgs, ref["hist"], ref["prompt"], ref["bias"], ok)
    flags = torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    if to == "inplace":
        got = R.apply(x, out=x, flags=flags, **kw)
        assert got.data_ptr() == x.data_ptr()
        assert torch.equal(base[:, vocab:], before[:, vocab:])
    else:
        got = R.apply(x, out_dtype=None if to == "new" else DT[to], flags=flags, **kw)
        assert torch.equal(base, before)
        assert got.dtype == (DT[dt] if to == "new" else DT[to])
    torch.cuda.synchronize()
    close(got, want, size)
    assert torch.equal(flags, torch.where(ok.any(1), 0, R.GE_RULE_EMPTY).int())


@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_values_that_are_no_numbers(dt):
    from gemmaedge_amd import rules as R

    base, kw, ref, ok, cfgs = make(4, 1001, dt, history=300, bias=40, masks=True)
    base[:, 0::5] = INF
    base[:, 1::5] = -INF
    base[:, 2::5] = math.nan
    base[:, 3::10] = torch.finfo(DT[dt]).min
    want, size = reference(base, cfgs, ref["hist"], ref["prompt"], ref["bias"], ok)
    for to in (None, base):
        got = R.apply(base, out=to, **kw)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        inf = torch.isinf(want)
        assert torch.equal(got.double()[inf], want[inf])


@pytest.mark.parametrize("cap", (0.0, 30.0))
@pytest.mark.parametrize("length", (0, 1, 5, 8, 9, 24, 1000003))
def test_ring(length, cap):
    """The ring's places hold the last of the appended tokens; the prompt's are known by their number."""
    from gemmaedge_amd import rules as R

    rows, vocab, capacity = 3, 500, 8
    base = make(rows, vocab, "f32")[0]
    g = torch.Generator().manual_seed(length)
    # of a long history only the last 2 x capacity ids can matter
    first = max(0, length - 2 * capacity)
    tail = torch.randint(0, 40, (rows, length - first), generator=g)
    ring = torch.full((rows, capacity), 499, dtype=torch.int32)
    for k in range(first, length):
        ring[:, k % capacity] = tail[:, k - first].int()
    prompts = [0, length // 2, max(0, length - 3)]
    cfgs = [config(1, cap)] * rows
    kept = max(0, length - capacity)
    hist = [tail[r, kept - first:].tolist() for r in range(rows)]
    want, size = reference(base, cfgs, hist, [max(0, p - kept) for p in prompts], [[]] * rows,
                           torch.ones(rows, vocab, dtype=torch.bool, device="cuda"))
    ring_d, lens = ring.cuda(), torch.full((rows,), length, dtype=torch.int32, device="cuda")
    got = R.apply(base, cfgs[0], ring=ring_d, ring_len=lens, prompt_len=torch.tensor(prompts, dtype=torch.int32, device="cuda"))
    close(got, want, size)
    assert torch.equal(ring_d.cpu(), ring) and bool((lens == length).all())


def test_mask_without_rows_and_one_row_of_logits():
    from gemmaedge_amd import rules as R

    x = torch.randn(300, device="cuda")
    m = torch.zeros(1, 12, dtype=torch.int32, device="cuda")
    m[0, 3] = 1 << 4
    flags = torch.empty(1, dtype=torch.int32, device="cuda")
    got = R.apply(x, mask=m, flags=flags)
    assert got.shape == (300,) and int(flags) == 0
    assert torch.isfinite(got).nonzero().tolist() == [[100]] and got[100] == x[100]
    y = x.clone()
    assert R.apply(y, out=y, mask=m).data_ptr() == y.data_ptr() and torch.equal(y, got)


def test_no_rows_and_empty_lists():
    from gemmaedge_amd import rules as R

    none = torch.empty(0, dtype=torch.int32, device="cuda")
    x = torch.empty(0, 50, device="cuda")
    assert R.apply(x, R.RuleConfig(presence_penalty=1.0)).shape == (0, 50)
    y = torch.randn(3, 50, device="cuda")
    offs = torch.zeros(4, dtype=torch.int32, device="cuda")
    got = R.apply(y, R.RuleConfig(presence_penalty=1.0), history=none, history_offsets=offs, bias_ids=none,
                  bias_values=torch.empty(0, device="cuda"), bias_offsets=offs)
    assert torch.equal(got, y)


@pytest.mark.parametrize("to", ("new", "inplace"))
def test_longest_lists(to):
    """A history and a list of biases whose lengths add up to more than 31 bits, in one of so many rows
    that a slice of the vocabulary has more tokens than are counted by a word each."""
    from gemmaedge_amd import rules as R

    rows, vocab, n, m = 512, 8200, 4999, 2 ** 31 - 1
    x = torch.randn(rows, vocab, device="cuda")
    ids = (torch.arange(n, device="cuda") % 4999).int()
    offs = torch.full((rows + 1,), n, dtype=torch.int32, device="cuda")
    offs[0] = 0
    bias_ids = torch.arange(vocab, device="cuda", dtype=torch.int32).repeat(m // vocab + 1)[:m]
    values = torch.full((m,), math.nan, device="cuda")
    last = torch.randn(vocab, device="cuda")
    values[m - vocab:] = last
    bias_offs = torch.full((rows + 1,), m, dtype=torch.int32, device="cuda")
    bias_offs[0] = 0
    want = x.clone()
    want[0, :n] -= 1.5
    want[0, bias_ids[m - vocab:].long()] += last
    got = R.apply(x, R.RuleConfig(presence_penalty=1.5), out=x if to == "inplace" else None, history=ids, history_offsets=offs,
                  bias_ids=bias_ids, bias_values=values, bias_offsets=bias_offs)
    assert torch.equal(got, want)


def test_more_rows_than_a_launch():
    from gemmaedge_amd import rules as R

    rows = (1 << 22) + 5
    x = torch.randn(rows, 33, device="cuda", dtype=torch.bfloat16)
    ids = torch.arange(rows, device="cuda", dtype=torch.int32) % 33
    offs = torch.arange(rows + 1, device="cuda", dtype=torch.int32)
    want = x.clone()
    want[torch.arange(rows, device="cuda"), ids.long()] -= 1.0
    assert torch.equal(R.apply(x, R.RuleConfig(presence_penalty=1.0), history=ids, history_offsets=offs), want)


@pytest.mark.parametrize("cap", (0.0, 30.0))
@pytest.mark.parametrize("dt", ("bf16", "f32"))
def test_sampling_after_the_rules_is_the_samplers_own(dt, cap):
    """Softcap and repetition penalty here, or in the sampler: the same tokens and probabilities."""
    import numpy as np

    from gemmaedge_amd import rules as R
    from gemmaedge_amd import sampler as S

    rows, vocab = 9, 50021
    base, kw, _, _, _ = make(rows, vocab, dt, history=2000, seed=3)
    uni = torch.rand(rows, device="cuda")
    hist = dict(history=kw["history"], history_offsets=kw["history_offsets"])
    with S.Sampler(rows, vocab, 2000) as s:
        for k in (64, 0):
            full = s.sample(base, S.SamplingConfig(0.9, k, 0.95, 0.01, softcap=cap, repetition_penalty=1.2), uniforms=uni, **hist)
            y = R.apply(base, R.RuleConfig(softcap=cap, repetition_penalty=1.2), out_dtype=torch.float32, **hist)
            mine = s.sample(y, S.SamplingConfig(0.9, k, 0.95, 0.01), uniforms=uni)
            for a, b in zip(full[:2], mine[:2]):
                assert np.array_equal(a.cpu().numpy().view(np.uint32), b.cpu().numpy().view(np.uint32))


def test_graph():
    """A captured call on new logits, a longer ring and other masks in the same memory."""
    from gemmaedge_amd import rules as R

    rows, vocab, capacity = 3, 9001, 64
    base, kw, _, _, _ = make(rows, vocab, "bf16", bias=20, masks=True, seed=5)
    ring = torch.zeros(rows, capacity, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    kw.update(ring=ring, ring_len=lens)
    x, flags = base.clone(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        R.apply(x, out=x, flags=flags, **kw)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        R.apply(x, out=x, flags=flags, **kw)
    for step in range(4):
        torch.manual_seed(step)
        new = (4 * torch.randn(rows, vocab, device="cuda")).bfloat16()
        ring.copy_(torch.randint(vocab, (rows, capacity), device="cuda"))
        lens.fill_(20 * step)
        kw["mask"].copy_(torch.randint(-2 ** 31, 2 ** 31, kw["mask"].shape, device="cuda"))
        x.copy_(new)
        want_flags = torch.zeros_like(flags)
        want = R.apply(new, flags=want_flags, **kw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(flags, want_flags)


def test_another_stream_and_dropped_tensors():
    from gemmaedge_amd import rules as R

    base, kw, ref, ok, cfgs = make(40, 30000, "f32", history=500, bias=20, masks=True)
    want = R.apply(base, **kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    copies = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    got = R.apply(base, stream=side, **copies)
    del copies
    junk = [torch.full((400_000,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]
    side.synchronize()
    assert torch.equal(got, want) and len(junk) == 8


def test_refusals():
    from gemmaedge_amd import rules as R

    x = torch.randn(4, 100, device="cuda")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    bad = [dict(out=x.bfloat16(), out_dtype=torch.float32), dict(out=torch.empty(4, 99, device="cuda")), dict(out_dtype=torch.float16),
           dict(history=i32(5)), dict(history=i32(5), history_offsets=i32(4)), dict(history=i32(5).long(), history_offsets=i32(5)),
           dict(ring=i32(4, 8)), dict(ring=i32(3, 8), ring_len=i32(4)), dict(ring=i32(4, 8), ring_len=i32(3)),
           dict(ring=i32(4, 8), ring_len=i32(4), history=i32(5), history_offsets=i32(5)), dict(prompt_len=i32(3)),
           dict(bias_ids=i32(5)), dict(bias_ids=i32(5), bias_values=torch.zeros(4, device="cuda"), bias_offsets=i32(5)),
           dict(mask=i32(4, 3)), dict(mask=i32(3, 4)), dict(mask=i32(4)), dict(mask=i32(4, 4), mask_rows=i32(5)), dict(mask_rows=i32(4)),
           dict(flags=i32(5)), dict(flags=torch.zeros(4, device="cuda")), dict(row_params=torch.zeros(63, dtype=torch.uint8, device="cuda")),
           dict(config=R.RuleConfig(repetition_penalty=0.0)), dict(history=i32(5).cpu(), history_offsets=i32(5)), dict(out=x[:, :100].t())]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError)):
            R.apply(x, **kw)
    with pytest.raises(ValueError):
        R.apply(x.half())
    with pytest.raises(ValueError):
        R.apply(x[:, ::2])
    with pytest.raises(ValueError):
        R.apply(torch.empty(2, 0, device="cuda"))
    with pytest.raises(RuntimeError, match="overlaps"):
        big = torch.zeros(500, device="cuda")
        R.apply(big[:400].view(4, 100), out=big[100:].view(4, 100))
