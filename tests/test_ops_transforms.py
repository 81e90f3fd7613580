"""Derivatives and transforms that the operators on compressed weights do not have are refused, not dropped."""

import pytest
import torch
from torch.autograd import forward_ad

import cuzipnn_b200 as z

BF = torch.bfloat16


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


def refused(x, bias, residual, blob):
    t = torch.zeros(x.shape[0], dtype=torch.int64, device=x.device)
    ids, logits = t[:, None].repeat(1, 2), torch.zeros(x.shape[0], 2, device=x.device)
    with forward_ad.dual_level():
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                for call in (lambda: z.blob_linear(dual(x), blob), lambda: z.blob_linear(x, blob, bias=dual(bias)),
                             lambda: z.blob_linear(x, blob, residual=dual(residual)),
                             lambda: z.blob_cross_entropy(dual(x), blob, t),
                             lambda: z.blob_distillation(dual(x), blob, logits, ids)):
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call()


def test_dual_tensors():
    blob = z.compress_tensor(torch.zeros(48, 32, dtype=BF), min_compress_bytes=1 << 30)
    refused(torch.zeros(5, 32, dtype=BF), torch.zeros(48, dtype=BF), torch.zeros(5, 48, dtype=BF), blob)


@pytest.mark.gpu
def test_dual_tensors_on_the_gpu():
    blob = z.compress_tensor(torch.randn(48, 32, device="cuda").to(BF), min_compress_bytes=0, readback_to_cpu=False)
    x, bias, res = (torch.randn(s, device="cuda").to(BF) for s in ((5, 32), (48,), (5, 48)))
    refused(x, bias, res, blob)
    with forward_ad.dual_level():  # a level alone does not matter
        y = z.blob_linear(x, blob, bias=bias, residual=res)
    assert torch.equal(y, z.blob_linear(x, blob, bias=bias, residual=res))


@pytest.mark.gpu
def test_function_transforms():
    blob = z.compress_tensor(torch.randn(48, 32, device="cuda").to(BF), min_compress_bytes=0, readback_to_cpu=False)
    x = torch.randn(3, 5, 32, device="cuda").to(BF)
    t = torch.zeros(5, dtype=torch.int64, device="cuda")
    for fn in (lambda v: z.blob_linear(v, blob), lambda v: z.blob_cross_entropy(v, blob, t)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.vmap(fn)(x)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(fn, (x[0],), (x[1],))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.grad(lambda v: fn(v).float().sum())(x[0])
