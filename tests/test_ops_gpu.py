"""Operators on compressed weights against their formulas in 64 bits.

Tolerances.  u = finfo.eps / 2 is the largest relative rounding of a 16-bit value.  A product of 16-bit
numbers is exact in 32 bits; a sum of n products of absolute sum S is off by at most
(n / 16 + 32) * 2^-22 * S when 16 products are added at a time into a 32-bit accumulator that may
truncate (one unit of the last place, 2^-23, for the aligned addends and one for the sum), n added
one by one by rounding (2^-24 each) staying below it as well.
Outputs are rounded once (u).  Where 16-bit intermediates enter a sum (the slope and dz of a
linear layer: 2u; softmax - q of a loss: u), every term is off by that fraction at most; the bound
over the sum is that fraction of the sum of absolute terms, and since the roundings are independent
the error's 2-norm stays near that fraction of the 2-norm of what is summed (checked with a factor 2).
"""

import math

import pytest
import torch

import cuzipnn_b200 as z

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
DEV = "cuda"
F = torch.nn.functional


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(*shape, dtype=BF, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * sum(shape))
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def weight(rows, cols, dtype, kind="coded", chunk=8192, seed=1):
    """(weight, blob).  kinds: coded (exponent plane coded), both (both planes coded), raw (every
    unit raw), stored (the stored path)."""
    if kind == "both":
        g = torch.Generator(device=DEV).manual_seed(seed)
        w = (torch.randint(-4, 5, (rows, cols), generator=g, device=DEV) * 0.125).to(dtype)
    else:
        w = rnd(rows, cols, dtype=dtype, scale=0.05, seed=seed)
    args = {"coded": {}, "both": {}, "raw": {"passthrough_threshold": 0.001}, "stored": {}}[kind]
    blob = z.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=max(8, chunk // 16), readback_to_cpu=False,
                             min_compress_bytes=1 << 30 if kind == "stored" else 0, **args)
    return w, blob


def sum_bound(n):
    return (n / 16 + 32) * 2.0**-22


def assert_within(got, want, tol):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    worst = int(off.argmax()) if off.numel() else 0
    assert bool((off <= 0).all()), (
        f"element {worst}: {got.flatten()[worst].item()} for {want.flatten()[worst].item()}, "
        f"{(off > 0).sum().item()} of {off.numel()} outside")


ACTS = {None: lambda v: v, "relu": F.relu, "gelu": F.gelu, "silu": F.silu,
        "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}


def check_linear(x, w, blob, bias=None, act=None, res=None):
    y = z.blob_linear(x, blob, bias=bias, activation=act, residual=res)
    assert y.dtype == x.dtype and y.is_contiguous()
    xd, wd = x.detach().double(), w.double()
    zz = F.linear(xd, wd, None if bias is None else bias.double())
    want = ACTS[act](zz)
    # An activation's slope is at most 1.13 and its own 32-bit evaluation is off by 2^-19 of the sum.
    s = xd.abs() @ wd.abs().t() + (0 if bias is None else bias.double().abs())
    tol = (1.13 * sum_bound(w.shape[1]) + 2.0**-19) * s
    if res is not None:
        want = want + res.double()
    tol = tol + (u_of(x.dtype) + 2.0**-22) * want.abs() + 2.0**-25  # 2^-25: half of fp16's smallest step
    assert_within(y, want, tol)
    assert z.last_decode_status() == 0
    return y


# tokens, rows, cols, chunk: one row and one token; rows inside sub-chunks, rows across sub-chunks,
# rows across many chunks, rows that end with their chunk; columns of no round size; more tokens
# than the decoder takes; ragged tiles.
SIZES = [
    (1, 1, 128, 1024), (1, 1, 1, 1024), (1, 48, 16, 1024), (1, 5000, 128, 1024), (2, 333, 144, 4096),
    (3, 97, 3584, 8192), (4, 40, 20000, 1024), (5, 9, 8192, 8192), (7, 640, 1280, 16384), (8, 31, 4096, 131072),
    (8, 700, 272, 1000 * 16), (9, 257, 64, 1024), (6, 1001, 517, 8192), (33, 129, 1000, 8192), (128, 128, 64, 1024),
    (129, 257, 63, 1024), (300, 700, 1016, 32768), (513, 1111, 333, 32768), (17, 5, 30000, 131072), (1000, 3, 8, 1024),
    (2100, 2503, 136, 32768),  # pairs of CTAs, ragged on both sides
    (2100, 2503, 4104, 65536),  # and the last tiles in parts of the contraction
    (20, 16000, 256, 1024),  # in pieces
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,rows,cols,chunk", SIZES)
def test_linear_sizes(tokens, rows, cols, chunk, dtype):
    w, blob = weight(rows, cols, dtype, chunk=chunk)
    check_linear(rnd(tokens, cols, dtype=dtype), w, blob)


@pytest.mark.parametrize("tokens", [1, 6, 40])
@pytest.mark.parametrize("kind", ["both", "raw", "stored"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_blob_kinds(tokens, kind, dtype):
    w, blob = weight(201, 272, dtype, kind=kind, chunk=4096)
    check_linear(rnd(tokens, 272, dtype=dtype), w, blob)


@pytest.mark.parametrize("sub", [64, 256, 1024, 1 << 20])
def test_linear_sub_chunk_counts(sub):
    w = rnd(100, 640, scale=0.05)
    for chunk in (2048, 65536):
        blob = z.compress_tensor(w, chunk_bytes=chunk, sub_chunk_bytes=sub, min_compress_bytes=0, readback_to_cpu=False)
        check_linear(rnd(2, 640), w, blob)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("tokens,rows,cols", [(1, 300, 256), (70, 333, 96), (600, 512, 64)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_epilogue(act, tokens, rows, cols, dtype):
    w, blob = weight(rows, cols, dtype)
    check_linear(rnd(tokens, cols, dtype=dtype, scale=4.0), w, blob, bias=rnd(rows, dtype=dtype), act=act,
                 res=rnd(tokens, rows, dtype=dtype, scale=3.0))


def test_linear_strides_and_shapes():
    w, blob = weight(77, 256, BF)
    base = rnd(2, 12, 3, 512)
    for x in (base[..., :256], base[..., 1:257], base.transpose(1, 2)[..., 256:], base[..., ::2], base[0, 0, 0, :256],
              base[0, 0, :1, 3:259], base[:1, :1, :1, :256].expand(2, 5, 1, 256)):
        check_linear(x, w, blob)
    res = rnd(77, 24).t()
    check_linear(base[0, :8, :, :256].reshape(24, 256), w, blob, res=res)
    assert z.blob_linear(base[:0, 0, 0, :256], blob).shape == (0, 77)
    b2 = torch.cat([torch.zeros(3, dtype=torch.uint8, device=DEV), blob])[3:]  # misaligned, no record
    check_linear(base[0, 0, :, :256], w, b2)
    b3 = torch.stack([blob, blob], 1)[:, 0]  # strided
    check_linear(base[0, 0, :, :256], w, b3)


def grads(y, leaves, g):
    return torch.autograd.grad(y, leaves, g)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("tokens,rows,cols,chunk", [(1, 64, 128, 1024), (5, 333, 75, 4096), (200, 130, 264, 8192),
                                                    (777, 1000, 520, 32768), (64, 5000, 256, 1024), (2100, 72, 2504, 32768), (2100, 4104, 2104, 65536),
                                                    (64, 16000, 256, 1024)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_linear_gradients(act, tokens, rows, cols, chunk, dtype):
    w, blob = weight(rows, cols, dtype, chunk=chunk)
    leaves = [rnd(tokens, cols, dtype=dtype, scale=2.0), rnd(rows, dtype=dtype), rnd(tokens, rows, dtype=dtype, seed=3)]
    g = rnd(tokens, rows, dtype=dtype, seed=5)
    for t in leaves:
        t.requires_grad_()
    y = z.blob_linear(leaves[0], blob, bias=leaves[1], activation=act, residual=leaves[2])
    dx, db, dr = grads(y, leaves, g)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    yr = ACTS[act](F.linear(ref[0], w.double(), ref[1])) + ref[2]
    rx, rb, rr = grads(yr, ref, g.double())
    zz = F.linear(ref[0], w.double(), ref[1]).detach().requires_grad_()
    dz = torch.autograd.grad(ACTS[act](zz).sum(), zz)[0] * g.double()
    assert torch.equal(dr, g)
    u = u_of(dtype)
    # The slope's own error: 2^-12 covers z's 32-bit sum (its slope changes by at most 1.2 per unit).
    # relu's slope jumps at 0: rows with a |z| within the sum's error are left out.
    ez = sum_bound(cols) * (ref[0].detach().abs() @ w.double().abs().t() + ref[1].detach().abs())
    near = (zz.detach().abs() <= ez) if act == "relu" else torch.zeros_like(dz, dtype=torch.bool)
    edz = (2 * u + u * u) * dz.abs() + 1.2 * ez * g.double().abs() + 2.0**-19 * g.double().abs() + 2.0**-24 * (dtype == HF)
    edz = torch.where(near, g.double().abs(), edz)
    tol = edz @ w.double().abs() + sum_bound(rows) * (dz.abs() @ w.double().abs()) + u * rx.abs() + 2.0**-25
    assert_within(dx, rx, tol)
    edb = u * dz.abs() + 1.2 * ez * g.double().abs() + 2.0**-19 * g.double().abs() + 2.0**-25
    edb = torch.where(near, g.double().abs(), edb)
    assert_within(db, rb, edb.sum(0) + sum_bound(tokens) * dz.abs().sum(0) + u * rb.abs() + 2.0**-25)
    assert float((dx.double() - rx).norm()) <= 2 * 2 * u * float(rx.norm()) + float((edz * near).norm())


def test_linear_gradient_against_differences():
    """The gradient is the formula's; against central differences of the operator itself the step h
    balances truncation (h^2 f'''/6) and the rounding of y (u |y| / h)."""
    w, blob = weight(40, 64, HF)
    x = rnd(3, 64, dtype=HF).requires_grad_()
    g = rnd(3, 40, dtype=HF, seed=2)
    dx, = grads(z.blob_linear(x, blob, activation="gelu"), [x], g)
    h = 2.0**-3
    for i in (0, 17, 63):
        e = torch.zeros_like(x)
        e[:, i] = h
        hi, lo = (z.blob_linear((x.detach().double() + s * e.double()).to(HF), blob, activation="gelu").double() for s in (1, -1))
        step = ((x.detach().double() + e.double()).to(HF).double() - (x.detach().double() - e.double()).to(HF).double())[:, i]
        num = ((hi - lo) * g.double()).sum(1) / step
        # rounding: 2u |y| per entry over 2h; truncation: |f'''| <= 1.3, (0.2 h)^2 |w| / 6 at most.
        tol = (2 * u_of(HF) * torch.maximum(hi.abs(), lo.abs()) * g.double().abs()).sum(1) / step
        tol = tol + (1.3 * w.double()[:, i].abs() ** 3 * h * h / 6 * g.double().abs()).sum(1)
        tol = tol + 4 * u_of(HF) * (w.double()[:, i].abs() * g.double().abs()).sum(1) * 1.13 + 1e-3
        assert bool(((dx[:, i].double() - num).abs() <= tol).all())


def test_linear_partial_gradients():
    w, blob = weight(50, 64, BF)
    x, b, r = rnd(4, 64), rnd(50), rnd(4, 50)
    g = rnd(4, 50, seed=9)
    for act in (None, "silu"):
        full = None
        for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
            ls = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, b, r), need)]
            y = z.blob_linear(ls[0], blob, bias=ls[1], activation=act, residual=ls[2])
            got = grads(y, [t for t in ls if t.requires_grad], g)
            if full is None:
                full = got
            else:
                assert torch.equal(got[0], full[need.index(1)])
    x = x.requires_grad_()
    y = z.blob_linear(x, blob)
    gx, = torch.autograd.grad(y.sum(), [x])  # an expanded gradient (stride 0)
    assert_within(gx, torch.ones(4, 50, device=DEV, dtype=torch.double) @ w.double(),
                  u_of(BF) * w.double().abs().sum(0) + 1e-6)
    y = z.blob_linear(x, blob)
    blob.add_(0)  # an in-place change between forward and backward is refused
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---- losses ---------------------------------------------------------------------------------


def reference_loss(h, w, ids, q, counts, temperature, reduction):
    """(loss, d loss / d h for a gradient of 1 (of ones for "none"), p - q) in 64 bits."""
    h = h.detach().double()
    s = h @ w.double().t() / temperature
    lse = torch.logsumexp(s, 1, keepdim=True)
    at = ids.clamp(min=0)
    rows = (torch.special.xlogy(q, q) - q * (s.gather(1, at) - lse)).sum(1) * temperature**2
    rows = torch.where(counts, rows, 0.0)
    d = torch.exp(s - lse).scatter_add(1, at, -q)
    mass = torch.exp(s - lse).scatter_add(1, at, q)  # what the difference is taken of
    d, mass = torch.where(counts[:, None], d, 0.0), torch.where(counts[:, None], mass, 0.0)
    n = max(1, int(counts.sum()))
    scale = temperature / (n if reduction == "mean" else 1)
    loss = {"mean": rows.sum() / n, "sum": rows.sum(), "none": rows}[reduction]
    return loss, (d * scale) @ w.double(), d * scale, mass * scale, lse


def check_loss(call, h, w, ids, q, counts, temperature, reduction, dtype):
    h = h.detach().clone().requires_grad_()
    loss = call(h)
    assert loss.dtype == torch.float32
    want, dh_want, d, mass, lse = reference_loss(h.reshape(-1, h.shape[-1]), w, ids, q, counts, temperature, reduction)
    # A logit is off by its sum's bound over T, lse by as much and 2^-21 of its terms; T^2 scales both.
    smax = (h.detach().double().reshape(-1, h.shape[-1]).abs() @ w.double().abs().t()).amax(1) / temperature
    tol = temperature**2 * (2 * sum_bound(w.shape[1]) * smax + 2.0**-20 * (1 + lse[:, 0].abs() + smax))
    tol = torch.where(counts, tol, 0.0)
    n = max(1, int(counts.sum()))
    tol = {"mean": tol.sum() / n, "sum": tol.sum(), "none": tol}[reduction]
    assert_within(loss.reshape(want.shape), want, tol + 2.0**-23 * want.abs())
    gain = 4096.0 if dtype == HF else 1.0  # a loss scale, so that fp16 gradients are normal numbers
    dh, = grads(loss, [h], torch.full_like(loss, gain))
    u = u_of(dtype)
    dh, dh_want, d, mass = dh.reshape(dh_want.shape).double(), dh_want * gain, d * gain, mass * gain
    # softmax - q in 32 bits before its rounding to 16: softmax is off by its logit's and lse's errors
    # and its own evaluation (2^-19 in all), q by its evaluation (2^-20), and up to 256 entries of one
    # id are subtracted one by one (2^-24 each): relative to softmax + q, not to their difference.
    e32 = (sum_bound(w.shape[1]) * 4 * smax[:, None] + 2.0**-18 + q.shape[1] * 2.0**-24) * mass
    edz = u * d.abs() + (1 + u) * e32 + 2.0**-40 * gain  # 2^-40: fp16's smallest half step over 2^15
    bound = edz @ w.double().abs() + sum_bound(w.shape[0]) * (d.abs() @ w.double().abs()) + u * dh_want.abs() + 2.0**-24
    assert_within(dh, dh_want, bound)
    assert float((dh - dh_want).norm()) <= 2 * 2 * u * float(dh_want.norm()) + float((e32 @ w.double().abs()).norm()) + 2.0**-24 * math.sqrt(dh.numel())
    assert bool((dh[~counts] == 0).all())
    assert z.last_decode_status() == 0
    return loss, dh


LOSS_SIZES = [  # tokens, vocabulary, cols, chunk
    (1, 1, 16, 1024), (1, 300, 128, 1024), (3, 5000, 144, 4096), (8, 2049, 256, 1024), (9, 513, 64, 4096),
    (100, 1001, 75, 4096), (130, 4000, 96, 8192), (257, 777, 512, 32768), (40, 12000, 256, 1024), (333, 7000, 40, 1024),
    (2100, 2503, 2104, 65536),  # every product by pairs of CTAs
    (2100, 8000, 2104, 2048),  # in pieces, with tiles in parts
    (50, 40000, 256, 1024),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", LOSS_SIZES)
def test_cross_entropy(tokens, vocab, cols, chunk, dtype):
    w, blob = weight(vocab, cols, dtype, chunk=chunk)
    h = rnd(tokens, cols, dtype=dtype, scale=2.0)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    t = torch.randint(vocab, (tokens,), generator=g, device=DEV)
    t[::3] = vocab - 1
    t[1::5] = -100
    counts = t >= 0
    for reduction in ("mean", "sum", "none"):
        check_loss(lambda x: z.blob_cross_entropy(x, blob, t, reduction=reduction), h, w, t[:, None],
                   counts[:, None].double(), counts, 1.0, reduction, dtype)


def teacher(tokens, vocab, top, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + tokens)
    ids = torch.randint(vocab, (tokens, top), generator=g, device=DEV)  # the same id twice among them
    logits = torch.randn((tokens, top), generator=g, device=DEV) * 3
    ids[torch.rand((tokens, top), generator=g, device=DEV) < 0.2] = -1
    if top > 1:
        logits[torch.rand((tokens, top), generator=g, device=DEV) < 0.1] = -math.inf
        logits[torch.rand((tokens, top), generator=g, device=DEV) < 0.1] = torch.finfo(torch.float32).min
    return ids, logits


def distribution(ids, logits, temperature):
    held = ids >= 0
    t = logits.double().masked_fill(~held, -math.inf)
    mx = t.amax(1, keepdim=True)
    counts = mx[:, 0] > -math.inf
    e = torch.where(held, torch.exp((t - torch.where(counts[:, None], mx, 0.0)) / temperature), 0.0)
    return e / e.sum(1, keepdim=True).clamp(min=1e-300), counts


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", LOSS_SIZES)
@pytest.mark.parametrize("top,temperature", [(1, 1.0), (5, 2.0), (33, 0.5), (256, 1.0)])
def test_distillation(tokens, vocab, cols, chunk, top, temperature, dtype):
    w, blob = weight(vocab, cols, dtype, chunk=chunk)
    h = rnd(tokens, cols, dtype=dtype, scale=2.0)
    ids, logits = teacher(tokens, vocab, top)
    if tokens > 3:
        ids[1] = -1  # nothing
        logits[2] = -math.inf
        logits[3] = torch.finfo(torch.float32).min  # masked by the type's lowest value: all alike
        ids[3] = vocab - 1
    q, counts = distribution(ids, logits, temperature)
    for reduction in ("mean", "none"):
        check_loss(lambda x: z.blob_distillation(x, blob, logits, ids, temperature=temperature, reduction=reduction), h, w,
                   ids, q, counts, temperature, reduction, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,vocab,cols,chunk", [(20, 900, 64, 4096), (40, 40000, 256, 1024), (300, 6000, 128, 4096)])
@pytest.mark.parametrize("std", [3.0, 30.0, 300.0])
def test_loss_gradient_with_steep_logits(tokens, vocab, cols, chunk, dtype, std):
    """Logits whose maximum is far above the first columns': the references are raised in some pieces,
    in others not, and in some rows only."""
    w, blob = weight(vocab, cols, dtype, chunk=chunk)
    h = rnd(tokens, cols, dtype=dtype, scale=std / (0.05 * math.sqrt(cols)))
    h[::3] *= 0.1
    t = torch.randint(vocab, (tokens,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    t[::2] = (h.double() @ w.double().t()).argmax(1)[::2]  # confident rows: a small difference of p and 1
    t[1] = -100
    counts = t >= 0
    check_loss(lambda x: z.blob_cross_entropy(x, blob, t, reduction="none"), h, w, t[:, None], counts[:, None].double(),
               counts, 1.0, "none", dtype)
    ids, logits = teacher(tokens, vocab, 9)
    ids[::2, 0] = t[::2].clamp(min=0)
    q, counts = distribution(ids, logits, 1.0)
    check_loss(lambda x: z.blob_distillation(x, blob, logits, ids, reduction="none"), h, w, ids, q, counts, 1.0, "none",
               dtype)


def test_loss_no_row_counts():
    w, blob = weight(500, 64, BF)
    for tokens in (2, 20):
        h = rnd(tokens, 64)
        h[0] = math.nan  # what an ignored row holds does not matter
        h[1] = math.inf
        h.requires_grad_()
        none = torch.full((tokens,), -100, device=DEV)
        for reduction in ("mean", "sum", "none"):
            loss = z.blob_cross_entropy(h, blob, none, reduction=reduction)
            assert bool((loss == 0).all())
            dh, = grads(loss, [h], torch.full_like(loss, math.inf))
            assert bool((dh == 0).all())
            loss = z.blob_distillation(h, blob, torch.zeros(tokens, 3, device=DEV), torch.full((tokens, 3), -1, device=DEV),
                                       reduction=reduction)
            assert bool((loss == 0).all())
    assert z.blob_cross_entropy(h[:0], blob, none[:0]).item() == 0
    assert z.blob_cross_entropy(h[:0], blob, none[:0], reduction="none").shape == (0,)


@pytest.mark.parametrize("tokens", [6, 60])
def test_loss_bad_rows_stay_alone(tokens):
    """A target past the vocabulary, or a row of infinities or NaN, is NaN in its own row only."""
    w, blob = weight(700, 128, BF)
    h = rnd(tokens, 128)
    t = torch.randint(700, (tokens,), device=DEV)
    hc = h.clone().requires_grad_()
    clean = z.blob_cross_entropy(hc, blob, t, reduction="none")
    dh_clean, = grads(clean, [hc], torch.ones(tokens, device=DEV))
    clean = clean.detach()
    t2, h2 = t.clone(), h.clone()
    t2[0], t2[1], t2[2] = 700, -1, 1 << 40
    h2[3], h2[4] = math.nan, math.inf
    h2.requires_grad_()
    loss = z.blob_cross_entropy(h2, blob, t2, reduction="none")
    dh, = grads(loss, [h2], torch.ones(tokens, device=DEV))
    assert bool(loss[:5].isnan().all()) and torch.equal(loss[5:], clean[5:])
    assert bool(dh[:5].isnan().all()) and torch.equal(dh[5:], dh_clean[5:])
    ids = t[:, None].repeat(1, 3)
    ids[0, 1] = 700
    loss = z.blob_distillation(h, blob, torch.zeros(tokens, 3, device=DEV), ids, reduction="none")
    assert bool(loss[0].isnan()) and bool(loss[1:].isfinite().all())
    # ignore_index may be any value, an id of the vocabulary among them.
    some = z.blob_cross_entropy(h.requires_grad_(), blob, t, ignore_index=int(t[0]), reduction="none").detach()
    assert some[0] == 0 and torch.equal(some[t != t[0]], clean[t != t[0]])


def test_loss_shapes_types_and_large_logits():
    w, blob = weight(900, 64, BF)
    h = rnd(3, 7, 64)[:, ::2]
    t = torch.randint(900, (3, 4), device=DEV)
    assert z.blob_cross_entropy(h, blob, t, reduction="none").shape == (3, 4)
    ids = torch.randint(900, (3, 4, 6), device=DEV)
    logits = rnd(3, 4, 6, dtype=HF)
    a = z.blob_distillation(h, blob, logits, ids, reduction="none")
    assert a.shape == (3, 4) and torch.equal(a, z.blob_distillation(h, blob, logits.float(), ids, reduction="none"))
    big = rnd(12, 64, scale=2000.0)  # logits of hundreds to thousands
    t = torch.randint(900, (12,), device=DEV)
    check_loss(lambda x: z.blob_cross_entropy(x, blob, t), big, w, t[:, None], torch.ones(12, 1, device=DEV).double(),
               torch.ones(12, dtype=torch.bool, device=DEV), 1.0, "mean", BF)


# ---- as they are used -----------------------------------------------------------------------


def small_model(x, blobs, bias, ids, t, logits):
    y = z.blob_linear(x, blobs[0], bias=bias, activation="silu")
    y = z.blob_linear(y, blobs[1], residual=x)
    return z.blob_cross_entropy(y, blobs[2], t) + 0.5 * z.blob_distillation(y, blobs[2], logits, ids, temperature=2.0)


def model_inputs(tokens=48):
    dims = [(512, 128), (128, 512), (3000, 128)]
    ws, blobs = zip(*(weight(r, c, BF, seed=i, chunk=4096) for i, (r, c) in enumerate(dims)))
    ids, logits = teacher(tokens, 3000, 8)
    t = torch.randint(3000, (tokens,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    t[::4] = -100
    return ws, blobs, rnd(tokens, 128), rnd(512), ids, t, logits


def plain_model(x, ws, bias, ids, t, logits):
    w = [v.double() for v in ws]
    y = F.silu(F.linear(x, w[0], bias))
    y = F.linear(y, w[1]) + x
    s = F.linear(y, w[2])
    q, counts = distribution(ids, logits, 2.0)
    logp = F.log_softmax(s / 2.0, 1)
    kl = (torch.special.xlogy(q, q) - q * logp.gather(1, ids.clamp(min=0))).sum(1) * 4.0
    return F.cross_entropy(s, t) + 0.5 * torch.where(counts, kl, 0.0).sum() / counts.sum()


def test_run_together():
    """A feed-forward layer, its residual, and both losses on one compressed head, with gradients."""
    ws, blobs, x, bias, ids, t, logits = model_inputs()
    x, bias = x.requires_grad_(), bias.requires_grad_()
    loss = small_model(x, blobs, bias, ids, t, logits)
    gx, gb = torch.autograd.grad(loss, [x, bias])
    xd, bd = x.detach().double().requires_grad_(), bias.detach().double().requires_grad_()
    want = plain_model(xd, ws, bd, ids, t, logits)
    wx, wb = torch.autograd.grad(want, [xd, bd])
    u = u_of(BF)
    # Hidden values are rounded twice (u each) on the way to the logits, gradients five times.
    assert abs(loss.item() - want.item()) <= 4 * u * abs(want.item())
    for got, ref in ((gx, wx), (gb, wb)):
        assert float((got.double() - ref).norm()) <= 8 * u * float(ref.norm())


def test_deterministic_and_streams():
    ws, blobs, x, bias, ids, t, logits = model_inputs()
    x = x.requires_grad_()

    def step():
        loss = small_model(x, blobs, bias, ids, t, logits)
        one = z.blob_linear(x.detach()[:1], blobs[0])
        return [loss.detach(), one, *torch.autograd.grad(loss, [x])]

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:  # two at once, each with its own scratch
        with torch.cuda.stream(s):
            outs.append(step())
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(first, o):
            assert torch.equal(a, b)


def test_graph_capture_and_replay():
    ws, blobs, x, bias, ids, t, logits = model_inputs()
    x2, t2 = rnd(48, 128, seed=11), t.roll(1)

    def step(x, t):
        loss = small_model(x, blobs, bias, ids, t, logits)
        return [loss.detach(), z.blob_linear(x.detach()[:2], blobs[0]), *torch.autograd.grad(loss, [x])]

    want = [step(v.clone().requires_grad_(), tt) for v, tt in ((x, t), (x2, t2))]
    xs, ts = x.clone().requires_grad_(), t.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs, ts)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs: each holds its own scratch
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(xs, ts)
        graphs.append((graph, out))
    for (v, tt), ref in zip(((x2, t2), (x, t)), reversed(want)):
        with torch.no_grad():
            xs.copy_(v)
            ts.copy_(tt)
        for graph, out in graphs:
            graph.replay()
            for a, b in zip(out, ref):
                assert torch.equal(a, b)
    assert z.last_decode_status() == 0
    bare = blobs[0].clone()  # no record: its header cannot be read during capture
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="upload_blob"):
        with torch.cuda.graph(graph):
            z.blob_linear(xs.detach(), bare)
    torch.cuda.synchronize()


def test_upload_blob():
    w, blob = weight(200, 144, BF)
    assert z.upload_blob(blob) is blob
    host = blob.cpu()
    for src in (host, host.pin_memory(), blob.clone()):
        up = z.upload_blob(src, compute_device="cuda:0")
        assert up.is_cuda and torch.equal(up, blob)
        check_linear(rnd(2, 144), w, up)
        assert torch.equal(z.decompress_tensor(up), w)
    with pytest.raises(ValueError, match="the blob is on cpu"):
        z.blob_linear(rnd(2, 144), host)


@pytest.mark.parametrize("tokens,rows,cols", [(2, 64, 256), (40, 64, 256), (300, 4100, 256)])
def test_unaligned_operands(tokens, rows, cols):
    """Operands that start 2 bytes past an aligned address, and pitches that no 16-byte access fits."""
    w, blob = weight(rows, cols, BF)
    x = torch.zeros(tokens * cols + 1, dtype=BF, device=DEV)[1:].view(tokens, cols).copy_(rnd(tokens, cols))
    bias = torch.zeros(rows + 1, dtype=BF, device=DEV)[1:].copy_(rnd(rows))
    res = torch.zeros(tokens, rows + 1, dtype=BF, device=DEV)[:, 1:].copy_(rnd(tokens, rows, seed=4))
    check_linear(x, w, blob, bias=bias, act="silu", res=res)
    xg = x.clone().requires_grad_()
    g = torch.zeros(tokens, rows + 3, dtype=BF, device=DEV)[:, 3:].copy_(rnd(tokens, rows, seed=5))
    dx, = grads(z.blob_linear(xg, blob), [xg], g)
    want = g.double() @ w.double()
    assert_within(dx, want, u_of(BF) * want.abs() + sum_bound(rows) * (g.double().abs() @ w.double().abs()))


@pytest.mark.parametrize("tokens", [1, 4, 50, 300])
def test_special_values_stay_in_their_rows(tokens):
    """Infinities and NaN of the weight reach only their own output columns, those of x only their rows."""
    w = rnd(3000, 272, scale=0.05)
    clean_blob = z.compress_tensor(w, chunk_bytes=4096, min_compress_bytes=0, readback_to_cpu=False)
    w2 = w.clone()
    w2[5], w2[7, 100], w2[2048, 271], w2[2999, 0] = math.inf, math.nan, -math.inf, math.nan
    blob = z.compress_tensor(w2, chunk_bytes=4096, min_compress_bytes=0, readback_to_cpu=False)
    x = rnd(tokens, 272).abs() + 0.5
    y, clean = z.blob_linear(x, blob), z.blob_linear(x, clean_blob)
    bad = torch.zeros(3000, dtype=torch.bool, device=DEV)
    bad[[5, 7, 2048, 2999]] = True
    assert torch.equal(y[:, ~bad], clean[:, ~bad])
    assert bool((y[:, 5] == math.inf).all()) and bool((y[:, 2048] == -math.inf).all()) and bool(y[:, [7, 2999]].isnan().all())
    x2 = x.clone()
    x2[-1, 3] = math.nan
    y = z.blob_linear(x2, clean_blob, activation="relu")
    assert torch.equal(y[:-1], z.blob_linear(x, clean_blob, activation="relu")[:-1]) and bool(y[-1].isnan().all())


def test_threads_on_their_own_streams():
    """Calls from several threads at once: each keeps its results and its own decode status."""
    import threading

    ws, blobs, x, bias, ids, t, logits = model_inputs()
    want = small_model(x, blobs, bias, ids, t, logits)
    bad = z.upload_blob(blobs[0].clone())
    bad[40:44] = 255  # a negative unit size
    bad = z.upload_blob(bad.clone())
    torch.cuda.synchronize()
    out, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    out[i] = small_model(x, blobs, bias, ids, t, logits)
                    ok = z.last_decode_status()
                    if i % 2:
                        z.blob_linear(x, bad)
                    status = z.last_decode_status()
                    assert ok == 0 and (status != 0) == bool(i % 2)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors, errors
    assert all(torch.equal(o, want) for o in out.values())


def test_backward_twice_and_captured_afterwards():
    """The same graph twice; then a captured training step of the same leaf, once the eager graph is
    gone (while it lives, PyTorch itself refuses to capture a backward pass of its leaves: their
    gradient nodes belong to the eager stream)."""
    ws, blobs, x, bias, ids, t, logits = model_inputs()
    x = x.requires_grad_()
    loss = small_model(x, blobs, bias, ids, t, logits)
    one, = torch.autograd.grad(loss, [x], retain_graph=True)
    two, = torch.autograd.grad(loss, [x])
    assert torch.equal(one, two)
    del loss
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        inner = small_model(x, blobs, bias, ids, t, logits)
        gi, = torch.autograd.grad(inner, [x])
    graph.replay()
    assert torch.equal(gi, one)


def test_offsets_past_32_bits():
    """A head of 2.15e9 elements (4.3 GB): more than 2^31 elements and 2^32 bytes."""
    rows, cols = 600_064, 3584
    w = torch.empty((rows, cols), dtype=BF, device=DEV).normal_(0.0, 0.02, generator=torch.Generator(device=DEV).manual_seed(0))
    blob = z.compress_tensor(w, readback_to_cpu=False)
    for tokens in (1, 5):
        x = rnd(tokens, cols)
        y = z.blob_linear(x, blob)
        for a, b in ((0, 300), (rows // 2, rows // 2 + 300), (rows - 300, rows)):
            want = x.double() @ w[a:b].double().t()
            s = x.double().abs() @ w[a:b].double().abs().t()
            assert_within(y[:, a:b], want, u_of(BF) * want.abs() + sum_bound(cols) * s + 2.0**-25)
    t = torch.tensor([rows - 1, 0, rows // 2, -100, rows - 7], device=DEV)
    h = rnd(5, cols).requires_grad_()
    loss = z.blob_cross_entropy(h, blob, t, reduction="none")
    dh, = grads(loss, [h], torch.ones(5, device=DEV))
    lse = torch.full((5,), -math.inf, dtype=torch.double, device=DEV)
    ref = torch.zeros(5, cols, dtype=torch.double, device=DEV)
    hd = h.detach().double()
    for a in range(0, rows, 50_000):
        lse = torch.logaddexp(lse, torch.logsumexp(hd @ w[a : a + 50_000].double().t(), 1))
    for a in range(0, rows, 50_000):
        wd = w[a : a + 50_000].double()
        ref += torch.exp(hd @ wd.t() - lse[:, None]) @ wd
    keep = t >= 0
    wt = w[t.clamp(min=0)].double()
    want = torch.where(keep, lse - (hd * wt).sum(1), 0.0)
    ref = torch.where(keep[:, None], ref - wt, 0.0)
    smax = float((hd.abs() @ w[:1000].double().abs().t()).amax()) * 1.1
    assert_within(loss, want, torch.full_like(want, 2 * sum_bound(cols) * smax + 2.0**-20 * (2 + 14 + smax)))
    assert float((dh.double() - ref).norm()) <= 4 * u_of(BF) * float(ref.norm())


@pytest.mark.parametrize("rows", [1, 60, 64, 65, 100, 130, 321])
@pytest.mark.parametrize("tokens,cols", [(1, 128), (2, 64), (20, 75), (130, 144), (600, 200)])
def test_calls_stay_inside_their_buffers(tokens, rows, cols):
    """Every entry point with exactly the scratch, state and output sizes it asks for, each followed by a
    pattern that must stay."""
    import ctypes

    from cuzipnn_b200 import _lib, _ops

    lib, guard, fill = _lib.lib, 1 << 16, 0xA5
    w, blob = weight(rows, cols, BF, chunk=1024)
    x, g = rnd(tokens, cols), rnd(tokens, rows)
    weight_desc = _ops._Weight(blob, x, "x")
    weight_desc.place("x")
    d = ctypes.byref(weight_desc.desc)
    stream = torch.cuda.current_stream().cuda_stream
    buffers = []

    def buf(nbytes):
        b = torch.full((nbytes + guard,), fill, dtype=torch.uint8, device=DEV)
        buffers.append((b, nbytes))
        return b.data_ptr()

    status = buf(4)
    ptr, ldx = x.data_ptr(), cols if tokens > 1 else (cols + 7) // 8 * 8
    ldg = rows if tokens > 1 else (rows + 7) // 8 * 8
    n = lib.zn_linear_temp_bytes(d, ptr, ldx, tokens)
    y, slope = buf(tokens * rows * 2), buf(tokens * rows * 2)
    assert lib.zn_linear(d, ptr, ldx, tokens, None, 4, None, 0, y, slope, status, buf(n), n, stream) == 0
    n = lib.zn_linear_grad_temp_bytes(d, g.data_ptr(), ldg, tokens, 1, 1, 1)
    assert lib.zn_linear_grad(d, g.data_ptr(), ldg, tokens, slope, buf(tokens * cols * 2), buf(rows * 2), status,
                              buf(n), n, stream) == 0
    for top in (1, 3):
        ids = torch.randint(rows, (tokens, top), device=DEV)
        logits = None if top == 1 else torch.zeros(tokens, top, device=DEV)
        grad = torch.ones(tokens, device=DEV)
        for with_grad in (0, 1):
            state = buf(lib.zn_loss_state_bytes(tokens, top))
            n = lib.zn_loss_temp_bytes(d, ptr, ldx, tokens, top, with_grad)
            unit = buf(tokens * cols * 4) if with_grad else None
            for reduction in (0, 2):
                loss = buf(4 * (tokens if reduction == 2 else 1))
                assert lib.zn_loss(d, ptr, ldx, tokens, ids.data_ptr(), None if logits is None else logits.data_ptr(), top,
                                   -100, 1.0, reduction, loss, unit, state, status, buf(n), n, stream) == 0
            if with_grad:
                assert lib.zn_loss_grad(8, tokens, cols, top, 2, state, unit, grad.data_ptr(), buf(tokens * cols * 2),
                                        stream) == 0
            too_small = lib.zn_loss(d, ptr, ldx, tokens, ids.data_ptr(), None if logits is None else logits.data_ptr(), top,
                                    -100, 1.0, 0, loss, unit, state, status, buf(n), n - 1, stream)
            assert too_small == _lib.ZN_ERR_SPACE
    torch.cuda.synchronize()
    for b, nbytes in buffers:
        assert bool((b[nbytes:] == fill).all()), nbytes


@pytest.mark.parametrize("tokens", [1, 30])
def test_malformed_blob_is_reported(tokens):
    """A blob whose payload or tables were damaged sets the status, is read inside its bounds only, and
    leaves the rows of intact chunks exact."""
    w, blob = weight(64, 256, BF, chunk=4096)  # 16 rows per chunk, 4 chunks
    x = rnd(tokens, 256)
    good = z.blob_linear(x, blob)
    nch = 4
    sizes = blob[40 : 40 + 4 * 2 * nch].cpu().view(torch.int32)
    n_comp = int(blob[12:16].cpu().view(torch.int32))
    data = (40 + 4 * (2 * nch + n_comp) + 7) // 8 * 8
    unit = [data + int(sum((int(s) + 7) // 8 * 8 for s in sizes[:i])) for i in range(2 * nch)]
    bad = blob.clone()
    at = unit[nch + 2] + 2  # chunk 2's coded plane: its symbol bitmap
    bad[at : at + 32] = 0
    bad = z.upload_blob(bad)
    y = z.blob_linear(x, bad)
    assert z.last_decode_status() != 0
    keep = torch.ones(64, dtype=torch.bool, device=DEV)
    keep[32:48] = False
    assert torch.equal(y[:, keep], good[:, keep]) and bool((y[:, ~keep] == 0).all())
    for n in (39, 60, data + 8, blob.numel() - 64):  # truncated
        cut = blob.clone()[:n].clone()
        if n >= 40:
            y = z.blob_linear(x, cut)
            assert z.last_decode_status() != 0 and bool(y.isfinite().all())
    assert z.blob_linear(x, blob).equal(good) and z.last_decode_status() == 0


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("chunk", [1024, 4096])
def test_broken_stream_counts_as_zeros(tokens, chunk):
    """A stream that does not end where it should sets the status; its chunk's elements count as zeros,
    both in the decoder's own product and in a decoded piece."""
    w, blob = weight(64, 256, BF, chunk=chunk)
    nch, rows = 64 * 256 // chunk, chunk // 256
    x = rnd(tokens, 256)
    good = z.blob_linear(x, blob)
    sizes = blob[40 : 40 + 4 * 2 * nch].cpu().view(torch.int32).tolist()
    n_comp = int(blob[12:16].cpu().view(torch.int32))
    data = (40 + 4 * (2 * nch + n_comp) + 7) // 8 * 8
    assert sizes[nch + 1] < chunk  # coded
    end = data + sum((s + 7) // 8 * 8 for s in sizes[: nch + 1]) + sizes[nch + 1]
    bad = blob.clone()
    bad[end - 40 : end] ^= 0x5A
    bad = z.upload_blob(bad)
    y = z.blob_linear(x, bad)
    assert z.last_decode_status() != 0
    keep = torch.ones(64, dtype=torch.bool, device=DEV)
    keep[rows : 2 * rows] = False
    assert torch.equal(y[:, keep], good[:, keep]) and bool((y[:, ~keep] == 0).all())


def test_inference_mode():
    """Blobs are made, uploaded and used in inference mode; what upload_blob returns carries its header
    (it can be captured) and stays usable outside, in training too."""
    w, blob = weight(512, 256, BF)
    x, x1 = rnd(30, 256), rnd(1, 256)
    y, y1 = z.blob_linear(x, blob), z.blob_linear(x1, blob)
    t = torch.arange(30, device=DEV)
    loss = z.blob_cross_entropy(x, blob, t)
    with torch.inference_mode():
        host = z.compress_tensor(w)
        made = z.compress_tensor(w, readback_to_cpu=False)
        many = z.compress_tensors([w, w], readback_to_cpu=False)
        for b in (made, *many, z.upload_blob(host, compute_device=DEV), z.upload_blob(made), blob):
            assert torch.equal(z.decompress_tensor(b), w)
            assert torch.equal(z.blob_linear(x, b), y) and torch.equal(z.blob_linear(x1, b), y1)
            assert torch.equal(z.blob_cross_entropy(x, b, t), loss)
        for b in z.decompress_tensors(list(many)):
            assert torch.equal(b, w)
        up = z.upload_blob(host, compute_device=DEV)
        assert z.upload_blob(up) is up
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            yg = z.blob_linear(x, up)
        g.replay()
        assert torch.equal(yg, y)
    xg = x.clone().requires_grad_()
    xe = x.clone().requires_grad_()
    z.blob_linear(xg, up).sum().backward()
    z.blob_linear(xe, blob).sum().backward()
    assert torch.equal(xg.grad, xe.grad)
    z.blob_cross_entropy(xg, made, t).backward()  # the head is not kept for the backward pass
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        z.blob_linear(xg, made)


def test_large_stored_weight():
    """A weight stored uncompressed is copied a bounded piece at a time (here two), never whole."""
    vocab, cols, tokens = 130000, 3592, 30
    w = torch.empty(vocab, cols, dtype=BF, device=DEV).normal_(0, 0.02)
    blob = z.compress_tensor(w, readback_to_cpu=False, min_compress_bytes=1 << 40)
    assert blob.numel() == 40 + w.numel() * 2
    x = rnd(tokens, cols).requires_grad_()
    dy = rnd(tokens, vocab)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = z.blob_linear(x, blob)
    (dx,) = torch.autograd.grad(y, x, dy)
    t = torch.randint(vocab, (tokens,), device=DEV)
    loss = z.blob_cross_entropy(x, blob, t)
    (dh,) = torch.autograd.grad(loss, x)
    plain = z.blob_cross_entropy(x.detach(), blob, t)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held < 0.9e9
    xe = x.detach().double().requires_grad_()
    z64 = torch.cat([xe.detach() @ p.double().T for p in w.split(13000)], 1)
    # The result: one rounding (2^-8) and the 32-bit sum (cols 2^-24 of the sum of magnitudes).
    mag = torch.cat([xe.detach().abs() @ p.double().abs().T for p in w.split(13000)], 1)
    assert bool(((y.double() - z64).abs() <= 2.0**-8 * z64.abs() + cols * 2.0**-24 * mag).all())
    exact = sum(d.double() @ p.double() for d, p in zip(dy.split(13000, 1), w.split(13000)))
    mag = sum(d.double().abs() @ p.double().abs() for d, p in zip(dy.split(13000, 1), w.split(13000)))
    assert bool(((dx.double() - exact).abs() <= 2.0**-8 * exact.abs() + vocab * 2.0**-24 * mag).all())
    zl = z64.requires_grad_()
    le = torch.nn.functional.cross_entropy(zl, t)
    (ds,) = torch.autograd.grad(le, zl)
    # 32-bit logits are off by cols 2^-24 mag at most, the loss by no more than twice that; 1e-5 leaves 80
    # roundings of 2^-24 for the exponentials, their sum and its logarithm on top.
    loss, le = loss.detach(), le.detach()
    assert abs(float(loss.double() - le)) <= 2 * cols * 2.0**-24 * float(
        (xe.detach().abs() * w[:1].double().abs().max()).sum(1).max()) + 1e-5 * float(le)
    assert abs(float(plain.double() - loss.double())) <= 1e-5 * float(le)
    exact = sum(d @ p.double() for d, p in zip(ds.split(13000, 1), w.split(13000)))
    mag = sum(d.abs() @ p.double().abs() for d, p in zip(ds.split(13000, 1), w.split(13000)))
    # dh: one rounding of the result and one of P, relative to what is summed, and the sums' own error.
    assert bool(((dh.double() - exact).abs() <= 2.0**-8 * exact.abs() + (2.0**-8 + 2.0**-10) * mag).all())
