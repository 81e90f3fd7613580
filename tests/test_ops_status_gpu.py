"""last_decode_status() around a backward pass: what the forward pass found is not lost."""

import pytest
import torch

import cuzipnn_b200 as z
from test_ops_gpu import BF, rnd, weight

pytestmark = pytest.mark.gpu


def damaged(blob):
    """The blob with a stored size below zero, which its decoder reports."""
    bad = blob.clone()
    bad[40:44] = 255
    return z.upload_blob(bad)


@pytest.mark.parametrize("tokens", [1, 30])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("need", ["x", "bias", "x and bias"])
def test_status_after_backward(tokens, act, need):
    w, blob = weight(64, 256, BF, chunk=4096)
    bad = damaged(blob)
    x, b = rnd(tokens, 256).requires_grad_("x" in need), rnd(64).requires_grad_("bias" in need)
    leaves = [t for t in (x, b) if t.requires_grad]
    g = rnd(tokens, 64)
    y = z.blob_linear(x, bad, bias=b, activation=act)
    found = z.last_decode_status()
    assert found != 0
    torch.autograd.grad(y, leaves, g)
    assert z.last_decode_status() == found
    # Another operator in between: the backward pass that decodes reports itself and its forward pass.
    y = z.blob_linear(x, bad, bias=b, activation=act)
    z.blob_linear(x.detach(), blob)
    assert z.last_decode_status() == 0
    torch.autograd.grad(y, leaves, g)
    assert z.last_decode_status() == (found if "x" in need else 0)
    # And an intact blob's reports nothing, whatever was before.
    y = z.blob_linear(x, blob, bias=b, activation=act)
    z.blob_linear(x.detach(), bad)
    torch.autograd.grad(y, leaves, g)
    assert z.last_decode_status() == (0 if "x" in need else found)


def test_status_of_the_forward_pass_stays():
    """Damage that only the forward pass met (the blob is mended behind its version counter's back)."""
    w, blob = weight(64, 256, BF, chunk=4096)
    bad = damaged(blob)
    x = rnd(30, 256).requires_grad_()
    y = z.blob_linear(x, bad)
    bad.data.copy_(blob)
    y.sum().backward()
    assert z.last_decode_status() != 0
    assert z.blob_linear(x, blob).shape == (30, 64) and z.last_decode_status() == 0


def test_status_read_on_another_stream():
    """The calls run on a side stream behind 50 ms of other work; the status is read from the default
    stream, which waits for them."""
    w, blob = weight(64, 256, BF, chunk=4096)
    bad, x = damaged(blob), rnd(30, 256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    calls = (lambda b: z.blob_linear(x, b), lambda b: z.blob_linear(x[:1], b), lambda b: z.decompress_tensor(b),
             lambda b: z.decompress_tensors([b, blob]),
             lambda b: z.blob_linear(x.clone().requires_grad_(), b).sum().backward())
    for call in calls:
        with torch.cuda.stream(side):
            call(blob)
            side.synchronize()
            torch.cuda._sleep(100_000_000)
            call(bad)
        assert z.last_decode_status() != 0
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)
            call(blob)
        assert z.last_decode_status() == 0
