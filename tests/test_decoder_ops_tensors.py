"""What the Python calls of the decoder operators refuse of a tensor, without a GPU:
fake CUDA tensors have every property but memory."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses import FakeTensorMode

from cruise_b200 import decoder_ops


def cuda(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def attend(view):
    q, cache = cuda(3, 4, 64, dtype=torch.bfloat16), cuda(8, 16, 2, 64, dtype=torch.bfloat16)
    decoder_ops.paged_attention(view(q), cache, cache, cuda(2, 4, dtype=torch.int32), cuda(2, dtype=torch.int32))


def rotate(view):
    cache, table = cuda(8, 16, 2, 64, dtype=torch.bfloat16), cuda(32, 64)
    decoder_ops.rotate_store(view(cuda(3, 512, dtype=torch.bfloat16)), cuda(2, dtype=torch.int64), cuda(2, dtype=torch.int32),
                             table, table, cache, cache, num_heads=4)


def choose(view):
    decoder_ops.choose(view(cuda(3, 100)))


@pytest.mark.parametrize("call", [attend, rotate, choose])
def test_tensors_without_memory_are_refused(call):
    for view in (lambda t: t[:2], lambda t: t[1:]):   # the second has an address, an offset from NULL
        with FakeTensorMode(), pytest.raises(ValueError, match="has no memory"):
            call(view)


@pytest.mark.parametrize("call", [attend, rotate, choose])
def test_forward_mode_tangents_are_refused(call):
    import torch.autograd.forward_ad as forward

    dual = lambda t: forward.make_dual(t[:2], torch.empty_like(t[:2]))  # noqa: E731
    with FakeTensorMode():
        with forward.dual_level(), pytest.raises(ValueError, match="tangent"):
            call(dual)
        with forward.dual_level(), torch.no_grad(), pytest.raises(ValueError, match="tangent"):   # it does not stop forward mode
            call(dual)
        with forward.dual_level(), pytest.raises(ValueError, match="has no memory"):   # the primal alone is fine
            call(lambda t: forward.unpack_dual(dual(t)).primal)
