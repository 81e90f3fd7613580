"""Losses where hidden needs no gradient, which take kernels of their own (and for one token the product
inside the decoder), against their formulas in 64 bits."""

import math

import pytest
import torch

import cuzipnn_b200 as z
from test_ops_gpu import (BF, DEV, HF, LOSS_SIZES, assert_within, distribution, reference_loss, rnd, sum_bound, teacher,
                          weight)

pytestmark = pytest.mark.gpu


def check_loss_only(call, h, w, ids, q, counts, temperature, reduction):
    """As the losses with a gradient are held: a logit is off by its sum's bound over T, lse by as much
    and 2^-20 of its terms; T^2 scales both."""
    assert not h.requires_grad
    loss = call(h)
    assert loss.dtype == torch.float32 and not loss.requires_grad
    want, *_, lse = reference_loss(h, w, ids, q, counts, temperature, reduction)
    smax = (h.double().abs() @ w.double().abs().t()).amax(1) / temperature
    tol = temperature**2 * (2 * sum_bound(w.shape[1]) * smax + 2.0**-20 * (1 + lse[:, 0].abs() + smax))
    tol = torch.where(counts, tol, 0.0)
    tol = {"mean": tol.sum() / max(1, int(counts.sum())), "sum": tol.sum(), "none": tol}[reduction]
    assert_within(loss, want, tol + 2.0**-23 * want.abs())
    assert z.last_decode_status() == 0
    return loss


# One token: multiplied inside the decoder where cols is a multiple of 16 from 128 on.
ONE = [(1, 300, 128, 1024), (1, 1, 128, 1024), (1, 5000, 144, 4096), (1, 65, 512, 131072), (1, 700, 3584, 8192),
       (1, 40000, 256, 1024), (1, 40, 20000, 1024), (1, 513, 640, 65536), (1, 1000, 75, 4096), (1, 900, 64, 4096)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", LOSS_SIZES + ONE)
def test_cross_entropy_only(tokens, vocab, cols, chunk, dtype):
    w, blob = weight(vocab, cols, dtype, chunk=chunk)
    h = rnd(tokens, cols, dtype=dtype, scale=2.0)
    t = torch.randint(vocab, (tokens,), generator=torch.Generator(device=DEV).manual_seed(tokens), device=DEV)
    t[::3] = vocab - 1
    t[1::5] = -100
    counts = t >= 0
    for reduction in ("mean", "sum", "none"):
        check_loss_only(lambda x: z.blob_cross_entropy(x, blob, t, reduction=reduction), h, w, t[:, None],
                        counts[:, None].double(), counts, 1.0, reduction)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", LOSS_SIZES + ONE)
@pytest.mark.parametrize("top,temperature", [(1, 1.0), (5, 2.0), (256, 0.5)])
def test_distillation_only(tokens, vocab, cols, chunk, top, temperature, dtype):
    w, blob = weight(vocab, cols, dtype, chunk=chunk)
    h = rnd(tokens, cols, dtype=dtype, scale=2.0)
    ids, logits = teacher(tokens, vocab, top)
    if tokens > 3:
        ids[1] = -1
        logits[2] = -math.inf
        logits[3] = torch.finfo(torch.float32).min
        ids[3] = vocab - 1
    else:
        ids[0, 0] = vocab - 1
        logits[0, 0] = 1.0
    q, counts = distribution(ids, logits, temperature)
    for reduction in ("mean", "sum", "none"):
        check_loss_only(lambda x: z.blob_distillation(x, blob, logits, ids, temperature=temperature, reduction=reduction),
                        h, w, ids, q, counts, temperature, reduction)


@pytest.mark.parametrize("tokens", [1, 6, 40])
@pytest.mark.parametrize("kind", ["both", "raw", "stored"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_loss_only_blob_kinds(tokens, kind, dtype):
    w, blob = weight(201, 272, dtype, kind=kind, chunk=4096)
    h = rnd(tokens, 272, dtype=dtype)
    t = torch.arange(tokens, device=DEV) * 5
    ones = torch.ones(tokens, dtype=torch.bool, device=DEV)
    check_loss_only(lambda x: z.blob_cross_entropy(x, blob, t, reduction="none"), h, w, t[:, None],
                    ones[:, None].double(), ones, 1.0, "none")


@pytest.mark.parametrize("tokens", [1, 20])
@pytest.mark.parametrize("std", [30.0, 300.0])
def test_loss_only_steep_logits(tokens, std):
    w, blob = weight(3000, 256, BF, chunk=4096)
    h = rnd(tokens, 256, scale=std / (0.05 * 16))
    t = torch.randint(3000, (tokens,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    ones = torch.ones(tokens, dtype=torch.bool, device=DEV)
    check_loss_only(lambda x: z.blob_cross_entropy(x, blob, t, reduction="none"), h, w, t[:, None],
                    ones[:, None].double(), ones, 1.0, "none")


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("grad", [False, True])
def test_small_losses_keep_their_digits(tokens, grad):
    """Logits that are exact in 32 bits (sums of multiples of 1 / 64), all above 120 and each row's target
    12 to 15 above the others: the loss log(1 + rest) is off by a few roundings of numbers around 1
    (2^-21) and by those of the logits times log2(e) (2^-24 of up to 205, four of them) relative to the
    rest, not by the roundings of the logits themselves, which are thousands of times as large."""
    vocab, cols = 2000, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    w = (torch.randint(-4, 5, (vocab, cols), generator=g, device=DEV) / 8).to(BF)
    h = (torch.randint(-2, 3, (tokens, cols), generator=g, device=DEV) / 8).to(BF)
    t = torch.randperm(vocab, generator=g, device=DEV)[:tokens]
    m = torch.arange(tokens, device=DEV)
    w[:, : tokens + 1] = 0.0
    h[:, : tokens + 1] = 0.0
    w[:, 0], h[:, 0] = 0.125, 1000.0
    w[t, m + 1], h[m, m + 1] = 4.0, (3.0 + m % 4 / 4).to(BF)
    blob = z.compress_tensor(w, chunk_bytes=4096, min_compress_bytes=0, readback_to_cpu=False)
    s = h.double() @ w.double().t()
    assert torch.equal(s, s.float().double()) and 120 < float(s.min()) and float(s.max()) < 142
    gap = s.gather(1, t[:, None])
    want = torch.log1p(torch.where(m.new_tensor(range(vocab)) == t[:, None], 0.0, torch.exp(s - gap)).sum(1))
    assert float(want.max()) < 0.1
    loss = z.blob_cross_entropy(h.requires_grad_(grad), blob, t, reduction="none")
    assert_within(loss, want, 2.0**-21 + 4 * 2.0**-24 * 205 * want)


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("grad", [False, True])
def test_infinite_logit_that_the_teacher_excludes(tokens, grad):
    """An entry of probability 0 adds nothing to the loss, also where the student's logit is -inf."""
    w = rnd(700, 128, scale=0.05)
    w[9] = -math.inf
    blob = z.compress_tensor(w, chunk_bytes=4096, min_compress_bytes=0, readback_to_cpu=False)
    h = rnd(tokens, 128).abs() + 0.1
    ids = torch.tensor([[3, 9, 600]], device=DEV).repeat(tokens, 1)
    logits = torch.tensor([[1.0, -math.inf, 2.0]], device=DEV).repeat(tokens, 1)
    loss = z.blob_distillation(h.requires_grad_(grad), blob, logits, ids, reduction="none")
    logp = torch.log_softmax(h.detach().double() @ w.double().t(), 1)[:, [3, 600]]
    q = torch.softmax(torch.tensor([1.0, 2.0], device=DEV).double(), 0)
    want = (q * (q.log() - logp)).sum(1)
    smax = (h.detach().double() @ rnd(700, 128, scale=0.05).double().abs().t()).amax(1)
    assert_within(loss, want, 2 * sum_bound(128) * smax + 2.0**-20 * (10 + smax))


@pytest.mark.parametrize("grad", [False, True])
def test_teacher_logits_in_64_bits(grad):
    """Large ones with small differences, and entries masked by the type's lowest value, all of a row's
    among them (uniform then, as in any other type)."""
    w, blob = weight(700, 128, BF)
    ids, _ = teacher(8, 700, 5)
    ids[:, 0] = torch.arange(8, device=DEV)
    logits = torch.randn((8, 5), device=DEV, dtype=torch.double, generator=torch.Generator(device=DEV).manual_seed(2)) + 3e9
    low = torch.finfo(torch.double).min
    logits[1] = low
    logits[2, 1:] = low
    logits[3, 2] = -math.inf
    logits[4] = -math.inf
    logits[5] = 1e300
    logits[6, 0] = -1e300
    q, counts = distribution(ids, logits, 1.0)
    assert bool(counts[1]) and not bool(counts[4])
    h = rnd(8, 128)
    want, *_, lse = reference_loss(h, w, ids, q, counts, 1.0, "none")
    smax = (h.double().abs() @ w.double().abs().t()).amax(1)
    loss = z.blob_distillation(h.requires_grad_(grad), blob, logits, ids, reduction="none")
    assert_within(loss, want, torch.where(counts, 2 * sum_bound(128) * smax + 2.0**-20 * (10 + smax), 0.0))
