"""Operators on compressed weights: refusals, which need no GPU (they come before any GPU work)."""

import ctypes

import pytest
import torch

import cuzipnn_b200 as z
from cuzipnn_b200 import _lib

BF = torch.bfloat16


def blob_of(*shape, dtype=BF):
    """A stored blob on the CPU: its header is what the checks read."""
    return z.compress_tensor(torch.zeros(shape, dtype=dtype), min_compress_bytes=1 << 30)


W = blob_of(48, 32)
X = torch.zeros(5, 32, dtype=BF)


@pytest.mark.parametrize("call", [
    lambda b: z.blob_linear(X, b),
    lambda b: z.blob_cross_entropy(X, b, torch.zeros(5, dtype=torch.int64)),
    lambda b: z.blob_distillation(X, b, torch.zeros(5, 2), torch.zeros(5, 2, dtype=torch.int64)),
])
def test_weight_refusals(call):
    with pytest.raises(ValueError, match="1-D uint8"):
        call(W.view(1, -1))
    with pytest.raises(ValueError, match="1-D uint8"):
        call(W.to(torch.int16))
    with pytest.raises(ValueError, match="too short"):
        call(W[:10])
    with pytest.raises(ValueError, match="truncated"):
        call(W[:-1])
    bad = W.clone()
    bad[0] = 0
    with pytest.raises(ValueError, match="not a cuzipnn blob"):
        call(bad)
    bad = W.clone()
    bad[24:32] = 255  # a negative dimension
    with pytest.raises(ValueError, match="not a cuzipnn blob"):
        call(bad)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        call(blob_of(48, 32, dtype=torch.float32))
    with pytest.raises(TypeError, match="has dtype"):
        call(blob_of(48, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="two nonempty"):
        call(blob_of(48, 32, 1))
    with pytest.raises(ValueError, match="two nonempty"):
        call(blob_of(0, 32))
    with pytest.raises(ValueError, match="33 columns"):
        call(blob_of(48, 33))
    with pytest.raises(ValueError, match="must be a CUDA tensor"):
        call(W)


def test_linear_refusals():
    with pytest.raises(ValueError, match="activation"):
        z.blob_linear(X, W, activation="swish")
    with pytest.raises(TypeError, match="bias has dtype"):
        z.blob_linear(X, W, bias=torch.zeros(48))
    with pytest.raises(ValueError, match="bias has shape"):
        z.blob_linear(X, W, bias=torch.zeros(1, dtype=BF))
    with pytest.raises(ValueError, match="residual has shape"):
        z.blob_linear(X, W, residual=torch.zeros(48, dtype=BF))
    with pytest.raises(ValueError, match="columns"):
        z.blob_linear(torch.zeros((), dtype=BF), W)


def test_loss_refusals():
    t = torch.zeros(5, dtype=torch.int64)
    with pytest.raises(ValueError, match="reduction"):
        z.blob_cross_entropy(X, W, t, reduction="max")
    with pytest.raises(TypeError, match="int64"):
        z.blob_cross_entropy(X, W, t.int())
    with pytest.raises(ValueError, match="targets has shape"):
        z.blob_cross_entropy(X, W, t[:4])
    ids, logits = torch.zeros(5, 3, dtype=torch.int64), torch.zeros(5, 3)
    for temperature in (0.0, -1.0, 1e-30, 1e30, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            z.blob_distillation(X, W, logits, ids, temperature=temperature)
    with pytest.raises(ValueError, match="between 1 and 256"):
        z.blob_distillation(X, W, logits[:, :0], ids[:, :0])
    with pytest.raises(ValueError, match="between 1 and 256"):
        z.blob_distillation(X, W, torch.zeros(5, 257), torch.zeros(5, 257, dtype=torch.int64))
    with pytest.raises(ValueError, match="teacher_ids has shape"):
        z.blob_distillation(X, W, logits, ids[:4])
    with pytest.raises(ValueError, match="teacher_logits has shape"):
        z.blob_distillation(X, W, logits[:, :2], ids)
    with pytest.raises(TypeError, match="float type"):
        z.blob_distillation(X, W, ids, ids)


def test_upload_blob_refusals():
    with pytest.raises(ValueError, match="1-D uint8"):
        z.upload_blob(W.view(1, -1))
    with pytest.raises(ValueError, match="CUDA device"):
        z.upload_blob(W, compute_device="cpu")


def test_abi_refusals_without_a_gpu():
    w = _lib.Weight(None, 100, 4, 8, 0, 8)
    r = ctypes.byref(w)
    assert _lib.lib.zn_linear(r, None, 8, 1, None, 0, None, 0, None, None, None, None, 0, None) == _lib.ZN_ERR_INVALID
    assert _lib.lib.zn_linear_temp_bytes(r, None, 7, 1) == 0  # pitch below the row
    assert _lib.lib.zn_linear_grad(r, None, 4, 1, None, None, None, None, None, 0, None) == _lib.ZN_ERR_INVALID
    assert _lib.lib.zn_loss(r, None, 8, 1, None, None, 1, 0, 1.0, 0, None, None, None, None, None, 0, None) == _lib.ZN_ERR_INVALID
    assert _lib.lib.zn_loss_grad(8, 1, 8, 1, 3, None, None, None, None, None) == _lib.ZN_ERR_INVALID
    assert _lib.lib.zn_loss_state_bytes(5, 257) == 0 and _lib.lib.zn_loss_state_bytes(5, 256) > 0
    for field, value in (("rows", 0), ("cols", -1), ("dtype", 9), ("chunk_bytes", 12), ("blob_bytes", 10)):
        bad = _lib.Weight(None, 1000, 4, 8, 0, 8)
        setattr(bad, field, value)
        assert _lib.lib.zn_loss_temp_bytes(ctypes.byref(bad), None, 8, 1, 1, 1) == 0
