"""Calls whose vocabulary is worked on in more than one piece (which sizes those are is
asserted on the host, in tests/cpp/head_plan_check.cpp). References and tolerances are
those of the loss's own tests (float64)."""
import pytest
import torch

import test_gpu_head_loss as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", (0.0, 30.0))
def test_two_pieces_of_256_wide_tiles(cap):
    # 512 MiB hold the gradient of 65,472 logits for each of 4,096 rows.
    L.check(4096, 64, 70001, "bf16", cap, seed=9)


def test_a_short_last_piece():
    # 512 MiB hold 130,944 logits of 2,000 rows: pieces of 65,792 and 65,283 words.
    L.check(2000, 128, 131075, "bf16", 0.0, seed=10)


def test_two_pieces_of_float32():
    # 512 MiB hold the gradient of 32,704 logits for each of 4,096 rows.
    L.check(4096, 64, 40001, "f32", 30.0, seed=11)


def test_three_pieces_of_float32_in_narrow_rows():
    L.check(3000, 33, 100003, "f32", 0.0, seed=12)


def test_packed_float32_weights_in_pieces():
    # Rows too far apart for a tile's 31-bit offsets are packed, 512 of this width at a time.
    from gemmaedge_amd import head as H

    rows, dim, vocab, stride = 5, 65536, 601, (1 << 21) + 8
    h, small, t, grad = L.inputs(rows, dim, vocab, torch.float32, seed=13)
    w = torch.empty(vocab, stride, device="cuda")[:, 3:3 + dim]
    w.copy_(small)
    hd = H.Head(rows, dim, vocab, dtype=torch.float32, train=True)
    loss, lse = hd.loss(h, w, t)
    dh, dw = hd.loss_backward(grad, h, w, t, lse)
    ref = L.reference(h, small, t, grad, 0.0, torch.float32)
    for k, got in dict(loss=loss, lse=lse, dh=dh, dw=dw).items():
        L.close(got, ref[k], k)
