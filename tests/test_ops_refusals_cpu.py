"""Refusals of the operators on compressed weights that come before any GPU work."""

import pytest
import torch

import cuzipnn_b200 as z

BF = torch.bfloat16


def test_ignore_index_is_an_int64():
    """ctypes would wrap 2^64 - 100 to -100, and ignore rows that the caller wants."""
    blob = z.compress_tensor(torch.zeros(48, 32, dtype=BF), min_compress_bytes=1 << 30)
    x, t = torch.zeros(5, 32, dtype=BF), torch.zeros(5, dtype=torch.int64)
    for value in (1 << 63, (1 << 64) - 100, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            z.blob_cross_entropy(x, blob, t, ignore_index=value)
    for value in ((1 << 63) - 1, -(1 << 63)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):  # accepted
            z.blob_cross_entropy(x, blob, t, ignore_index=value)
