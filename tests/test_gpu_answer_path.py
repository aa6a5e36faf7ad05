"""From hidden states to tokens as a decode loop runs it: norm, projection with each
request's adapter, the request's rules, and the sampler, which appends to the ring that
the rules count; captured once and replayed, against the same steps in float64.

Greedy tokens are compared where the two largest logits are further apart than 1e-3, far
above what bf16 operands with float32 sums leave (a logit is a sum of 128 products of
rounded operands, which the float64 steps take as they are)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ROWS, DIM, VOCAB, CAPACITY, STEPS = 6, 128, 2001, 8, 12


def setup():
    g = torch.Generator(device="cuda").manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    m = dict(embed=rn(VOCAB, DIM).bfloat16(), norm=(1 + 0.1 * rn(DIM)).bfloat16(), weight=(rn(VOCAB, DIM) / 4).bfloat16(),
             a=(rn(3, 8, DIM) / 8).bfloat16(), b=(rn(3, VOCAB, 8) / 2).bfloat16(), scale=torch.tensor([1.0, 0.5, 2.0], device="cuda"),
             adapter=torch.tensor([0, 2, -1, 1, 2, 0], device="cuda", dtype=torch.int32))
    words = -(-VOCAB // 32)
    mask = torch.full((2, words), -1, dtype=torch.int32, device="cuda")
    mask[1, : words // 2] = 0x55555555
    m.update(mask=mask, mask_rows=torch.tensor([1, -1, 0, 1, -1, 1], device="cuda", dtype=torch.int32),
             bias_ids=torch.tensor([5, 6, 7, 5], device="cuda", dtype=torch.int32),
             bias_values=torch.tensor([3.0, -float("inf"), 1.0, 4.0], device="cuda"),
             bias_offsets=torch.tensor([0, 2, 2, 3, 3, 4, 4], device="cuda", dtype=torch.int32),
             first=torch.arange(ROWS, device="cuda", dtype=torch.int32) * 100 + 3)
    return m


def test_decode_loop():
    from gemmaedge_amd import head as H
    from gemmaedge_amd import projection as P
    from gemmaedge_amd import rules as R
    from gemmaedge_amd import sampler as S

    m = setup()
    cfgs = [R.RuleConfig(30.0, 1.0 + 0.2 * i, 0.5 * i, 0.25) for i in range(ROWS)]
    params = R.row_params(cfgs)
    head, proj, sampler = H.Head(ROWS, DIM, 1), P.Projection(ROWS, DIM, VOCAB, 8, 3), S.Sampler(ROWS, VOCAB, CAPACITY)
    ring = torch.zeros(ROWS, CAPACITY, dtype=torch.int32, device="cuda")
    lens = torch.zeros(ROWS, dtype=torch.int32, device="cuda")
    ring[:, 0], lens[:] = m["first"], 1
    prompt = torch.ones(ROWS, dtype=torch.int32, device="cuda")
    tokens, flags = m["first"].clone(), torch.zeros(ROWS, dtype=torch.int32, device="cuda")
    logits = torch.empty(ROWS, VOCAB, device="cuda")

    def step():
        x = m["embed"].index_select(0, tokens)
        y, _, _ = head.norm(x, m["norm"], center=False)
        proj.project(y, m["weight"], m["a"], m["b"], m["scale"], m["adapter"], out=logits)
        R.apply(logits, out=logits, row_params=params, ring=ring, ring_len=lens, prompt_len=prompt, bias_ids=m["bias_ids"],
                bias_values=m["bias_values"], bias_offsets=m["bias_offsets"], mask=m["mask"], mask_rows=m["mask_rows"], flags=flags)
        sampler.sample(logits, S.SamplingConfig(temperature=0.0), ring=ring, ring_len=lens, tokens=tokens)
        return y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    ring.zero_()
    ring[:, 0], lens[:] = m["first"], 1
    tokens.copy_(m["first"])

    d = {k: v.double() if v.is_floating_point() else v for k, v in m.items()}
    bits = (m["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32) & 1).bool().reshape(2, -1)[:, :VOCAB]
    history = [[int(t)] for t in m["first"]]
    compared = 0
    for n in range(STEPS):
        graph.replay()
        torch.cuda.synchronize()
        assert not flags.any() and int(lens[0]) == n + 2
        h = y.double()  # the norm's own output: what follows is compared
        for r in range(ROWS):
            z = d["weight"] @ h[r]
            k = int(m["adapter"][r])
            if k >= 0:
                z = z + d["b"][k] @ (d["scale"][k] * (d["a"][k] @ h[r]))
            c = cfgs[r]
            z = c.softcap * torch.tanh(z / c.softcap)
            kept = history[r][-CAPACITY:]
            generated = kept if len(history[r]) > CAPACITY else history[r][1:]
            for t in set(kept):
                z[t] = z[t] / c.repetition_penalty if z[t] > 0 else z[t] * c.repetition_penalty
            for t in set(generated):
                z[t] = z[t] - c.frequency_penalty * generated.count(t) - c.presence_penalty
            lo, hi = int(m["bias_offsets"][r]), int(m["bias_offsets"][r + 1])
            for i in range(lo, hi):
                z[int(m["bias_ids"][i])] += float(m["bias_values"][i])
            q = int(m["mask_rows"][r])
            if q >= 0:
                z[~bits[q]] = -float("inf")
            fine = torch.isfinite(z)
            assert torch.equal(torch.isfinite(logits[r]), fine)
            assert float((logits[r].double()[fine] - z[fine]).abs().max()) < 1e-3
            top = torch.topk(z, 2).values
            got = int(tokens[r])
            if float(top[0] - top[1]) > 1e-3:
                assert got == int(z.argmax())
                compared += 1
            history[r].append(got)
            assert int(ring[r, (n + 1) % CAPACITY]) == got
    assert compared > STEPS * ROWS // 2


@pytest.mark.parametrize("cfg", (dict(temperature=0.0), dict(temperature=0.8, top_k=40), dict(temperature=0.8, top_k=0, top_p=1.0)))
def test_a_row_that_may_answer_nothing_is_done(cfg):
    """The rules' flags as the sampler's done state: the sampler leaves those rows alone."""
    from gemmaedge_amd import rules as R
    from gemmaedge_amd import sampler as S

    rows, vocab = 3, 5003
    logits = torch.randn(rows, vocab, device="cuda")
    mask = torch.zeros(rows, -(-vocab // 32), dtype=torch.int32, device="cuda")
    mask[0, 3], mask[2, 100] = 1 << 7, 0b11
    done, flags = torch.zeros(2, rows, dtype=torch.int32, device="cuda")
    ring, lens = torch.zeros(rows, 4, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    R.apply(logits, out=logits, mask=mask, flags=flags)
    done |= flags
    sampler = S.Sampler(rows, vocab, 4)
    tokens, _, got = sampler.sample(logits, S.SamplingConfig(**cfg), torch.tensor([0.5, 0.5, 0.25], device="cuda"), ring=ring, ring_len=lens, done=done)
    torch.cuda.synchronize()
    assert done.tolist() == [0, 1, 0] and lens.tolist() == [1, 0, 1]
    assert int(tokens[0]) == 103 and int(tokens[1]) == -1 and int(tokens[2]) in (3200, 3201)
    assert int(got[1]) & S.GE_FLAG_DONE
