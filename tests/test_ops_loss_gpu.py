"""Losses on a compressed head: gradients of confident rows, held to the difference of softmax and target."""

import math

import pytest
import torch

import cuzipnn_b200 as z
from test_ops_gpu import BF, DEV, HF, assert_within, rnd, sum_bound, u_of

pytestmark = pytest.mark.gpu


def head(vocab, cols, dtype, chunk, seed=1):
    """A head whose rows have a common mean as large as their deviation: what is lost from the softmax's
    tail is then a direction of its own in the gradient."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn((vocab, cols), generator=g, device=DEV) + torch.randn((1, cols), generator=g, device=DEV)) * 0.05
    w = w.to(dtype)
    return w, z.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=chunk // 16, min_compress_bytes=0, readback_to_cpu=False)


def confident(w, targets, nats, dtype, seed=5):
    """Hidden rows whose target's logit is about `nats` above the mean of the others."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    wd = w.double()
    up = wd[targets] - wd.mean(0)
    noise = torch.randn(up.shape, generator=g, device=DEV).double()
    noise = noise - up * ((noise * up).sum(1) / (up * up).sum(1))[:, None]
    return (noise + up * (nats.double() / (up * up).sum(1))[:, None]).to(dtype)


def bounds(h, w, p, q, d, dtype):
    """What the gradient's elements may be off by, for a gradient of one per row.

    A logit is off by el: its product's sum and a few roundings of it (2^-22 each).  Relative to itself a
    weight of the softmax is then off by 2 el (its own logit and lse), by its evaluation (2^-18: ex2, the
    sums) and by its rounding (u); in fp16 one below the others by more than 2^-22 loses up to 2^-33 of
    their sum besides.  At an id, p is off by 2 el p (1 - p) and both by 2^-18 of themselves; where there
    is one id, p - q is the others' sum, as exact as that."""
    u, smax = u_of(dtype), (h.abs() @ w.abs().t()).amax(1, keepdim=True)
    el = (sum_bound(w.shape[1]) + 2.0**-20) * smax
    other = torch.where(q > 0, 0.0, p)
    rel = u + 2.0**-18 + 4 * el
    one = (q > 0).sum(1, keepdim=True) == 1
    at_id = torch.where(q > 0, torch.where(one, rel * d.abs(), 4 * el * p * (1 - p) + 2.0**-18 * (p + q)), 0.0)
    flush = other.sum(1, keepdim=True) * 2.0**-33 * w.shape[0] if dtype == HF else 0.0
    e = (rel * other + at_id) @ w.abs() + flush * w.abs().amax(0)
    return e + sum_bound(w.shape[0]) * (d.abs() @ w.abs())


def check_rows(call, h, w, q, dtype, rows):
    """The gradient of every row, scaled to be of the order of one, against p - q in 64 bits; `rows`:
    1 - sum of p over the ids."""
    h = h.detach().clone().requires_grad_()
    gain = (1.0 / rows).float()
    loss = call(h)
    dh, = torch.autograd.grad(loss, [h], gain)
    hd, wd = h.detach().double(), w.double()
    logp = torch.log_softmax(hd @ wd.t(), 1)
    p = logp.exp()
    others = torch.where(q > 0, 0.0, p)
    one = (q > 0).sum(1, keepdim=True) == 1
    d = torch.where(q > 0, torch.where(one, -others.sum(1, keepdim=True), p - q), p)
    want = (d @ wd) * gain.double()[:, None]
    bound = bounds(hd, wd, p, q, d, dtype) * gain.double()[:, None] + (u_of(dtype) + 2.0**-22) * want.abs() + 2.0**-24
    assert_within(dh, want, bound)
    want_loss = (torch.special.xlogy(q, q) - torch.where(q > 0, q * logp, 0.0)).sum(1)
    return loss.detach(), want_loss


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", [(64, 20000, 256, 1024), (40, 51866, 128, 8192), (300, 4000, 320, 8192)])
@pytest.mark.parametrize("place", ["first 512", "first piece", "anywhere"])
def test_confident_rows(tokens, vocab, cols, chunk, place, dtype):
    """Targets among the first 512 ids (where the first reference is taken from), later in the first
    piece (where they might raise it) and anywhere, with 1 - p from about 0.1 to 1e-6."""
    w, blob = head(vocab, cols, dtype, chunk)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    low, high = {"first 512": (0, 512), "first piece": (512, 2900), "anywhere": (0, vocab)}[place]
    t = torch.randint(low, high, (tokens,), generator=g, device=DEV)
    nats = torch.linspace(13.0, 27.0, tokens, device=DEV)
    h = confident(w, t, nats, dtype)
    q = torch.zeros(tokens, vocab, dtype=torch.double, device=DEV).scatter_(1, t[:, None], 1.0)
    p = torch.softmax(h.double() @ w.double().t(), 1)
    rest = torch.where(q > 0, 0.0, p).sum(1)
    assert rest.min() < 1e-5 and rest.max() > 1e-2
    check_rows(lambda x: z.blob_cross_entropy(x, blob, t, reduction="none"), h, w, q, dtype, rest)
    one = torch.zeros(tokens, 1, device=DEV)
    check_rows(lambda x: z.blob_distillation(x, blob, one, t[:, None], reduction="none"), h, w, q, dtype, rest)


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("nats", [15.0, 40.0, 90.0, 300.0])
def test_confident_students(nats, dtype):
    """Several ids, one of them far above all else: the others' weights stay beside it, and past 100
    powers of two the reference is raised for it."""
    tokens, vocab, cols = 48, 20000, 256
    w, blob = head(vocab, cols, dtype, 1024)
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(vocab, (tokens, 6), generator=g, device=DEV)
    ids[:16, 0] = torch.arange(16, device=DEV)  # in the sample
    ids[16:32, 0] = 15000 + torch.arange(16, device=DEV)  # in a later piece
    logits = torch.randn((tokens, 6), generator=g, device=DEV) * 2
    h = confident(w, ids[:, 0], torch.full((tokens,), nats, device=DEV), dtype)
    q = torch.zeros(tokens, vocab, dtype=torch.double, device=DEV)
    q.scatter_add_(1, ids, torch.softmax(logits.double(), 1))
    loss, want = check_rows(lambda x: z.blob_distillation(x, blob, logits, ids, reduction="none"), h, w, q, dtype,
                            torch.ones(tokens, device=DEV))
    smax = (h.double().abs() @ w.double().abs().t()).amax(1)
    assert_within(loss, want, 2 * (sum_bound(cols) + 2.0**-20) * smax + 2.0**-20 * (10 + want.abs()))


@pytest.mark.parametrize("dtype", [HF, BF])
def test_ids_are_all_columns(dtype):
    """No column, or none of the sample, is left beside the ids."""
    for vocab, top in ((1, 1), (3, 3), (250, 250), (2000, 250)):
        w, blob = head(vocab, 64, dtype, 1024)
        ids = torch.arange(top, device=DEV).repeat(7, 1)
        logits = rnd(7, top, dtype=torch.float32)
        h = rnd(7, 64, dtype=dtype, scale=3.0)
        q = torch.zeros(7, vocab, dtype=torch.double, device=DEV).scatter_(1, ids, torch.softmax(logits.double(), 1))
        check_rows(lambda x: z.blob_distillation(x, blob, logits, ids, reduction="none"), h, w, q, dtype, torch.ones(7, device=DEV))
    w, blob = head(1, 64, dtype, 1024)
    for scale in (1.0, 300.0):
        h = rnd(5, 64, dtype=dtype, scale=scale).requires_grad_()
        loss = z.blob_cross_entropy(h, blob, torch.zeros(5, dtype=torch.int64, device=DEV), reduction="sum")
        dh, = torch.autograd.grad(loss, [h])
        assert loss.item() == 0 and bool((dh == 0).all())
