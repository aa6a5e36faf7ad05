"""Tensors that are dropped right after a call on another stream: their memory stays theirs
until the call is done, whatever their size, small blocks and large ones alike.

New tensors of the same sizes get none of it while the stream is busy; without a call
they get all of it, which shows that they would."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def blocks(tensors):
    return [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors]


def anew(shapes):
    return [torch.empty(s, dtype=d, device="cuda") for _ in range(3) for s, d in shapes]


def check(operands, call):
    """`call` with copies of the operands on a busy stream, dropped after it."""
    want = call(operands, None)
    torch.cuda.synchronize()
    shapes = [(t.shape, t.dtype) for t in operands.values()]

    copies = {k: v.clone() for k, v in operands.items()}
    old = blocks(copies.values())
    del copies
    new = anew(shapes)
    assert all(any(a < d and c < b for c, d in blocks(new)) for a, b in old)
    del new

    copies = {k: v.clone() for k, v in operands.items()}
    old = blocks(copies.values())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
    got = call(copies, side)
    del copies
    new = anew(shapes)
    assert not side.query(), "the stream was done before the new tensors were there"
    assert not any(a < d and c < b for c, d in blocks(new) for a, b in old)
    side.synchronize()
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("rows,vocab", ((3, 1000), (200, 40000)))
def test_rules(rows, vocab):
    from gemmaedge_amd import rules as R

    g = torch.Generator(device="cuda").manual_seed(rows)
    ids = lambda most, *s: torch.randint(most, s, generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
    x = dict(logits=torch.randn(rows, vocab, generator=g, device="cuda"), history=ids(vocab, rows * 300), bias_ids=ids(vocab, rows * 10),
             history_offsets=torch.arange(rows + 1, device="cuda", dtype=torch.int32) * 300, prompt_len=ids(300, rows),
             bias_offsets=torch.arange(rows + 1, device="cuda", dtype=torch.int32) * 10, bias_values=torch.randn(rows * 10, generator=g, device="cuda"),
             mask=ids(2 ** 31 - 1, rows, -(-vocab // 32)), mask_rows=ids(rows, rows),
             row_params=R.row_params([R.RuleConfig(20.0 + i, 1.1, 0.5, 0.1) for i in range(rows)]))

    def call(t, stream):
        flags = torch.empty(rows, dtype=torch.int32, device="cuda")
        return [R.apply(stream=stream, flags=flags, **t), flags]

    check(x, call)


@pytest.mark.parametrize("rows,dim,out", ((5, 64, 300), (300, 512, 4000)))
def test_projection(rows, dim, out):
    from gemmaedge_amd import projection as P

    g = torch.Generator(device="cuda").manual_seed(rows)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    x = dict(hidden=rn(rows, dim), weight=rn(out, dim), a=rn(3, 8, dim), b=rn(3, out, 8), scale=torch.rand(3, generator=g, device="cuda"),
             adapter=torch.randint(4, (rows,), generator=g, device="cuda", dtype=torch.int32))
    p = P.Projection(rows, dim, out, 8, 3, train=True)
    check(x, lambda t, stream: [p.project(**t, stream=stream)])
    x["dout"] = rn(rows, out)
    check(x, lambda t, stream: list(p.project_backward(**t, stream=stream)))
