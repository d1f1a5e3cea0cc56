"""The decoder operators next to autograd and torch.compile: what they write counts
as written, inference tensors pass, compiled functions call them between graphs."""

from __future__ import annotations

import pytest
import torch

from cruise_b200.decoder_ops import choose, paged_attention, rotate_store
from test_gpu_decoder_ops import attend_case, choose_case, rotate_case

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _device(cuda_ok):
    yield
    torch.cuda.synchronize()


def versions(case):
    return {name: t._version for name, t in case.items()}


def moved(case, before):
    return {name for name, t in case.items() if t._version != before[name]}


def test_what_is_written_counts_as_written():
    case = attend_case([20, 3], 4, 2, 64, BF16, seed=70)
    case.update(out=torch.empty_like(case["q"]), lse=torch.empty(2, 4, device="cuda"))
    before = versions(case)
    paged_attention(**case)
    assert moved(case, before) == {"out", "lse"}

    case, keep = rotate_case(4, 4, 2, 64, BF16, norm=True)
    case["out"] = torch.empty(4, 4, 64, dtype=BF16, device="cuda")
    before = versions(case)
    rotate_store(**case, **keep)
    assert moved(case, before) == {"key_cache", "value_cache", "out"}

    case = choose_case(2, 100, FP32)
    case.update(processed=torch.empty(2, 100, device="cuda"), out=torch.empty(2, dtype=torch.int64, device="cuda"))
    before = versions(case)
    choose(**case)
    assert moved(case, before) == {"processed", "out"}
    choose(**case, append=True)
    assert moved(case, before) == {"processed", "out", "history"}


def test_a_kept_value_that_was_overwritten_is_noticed():
    case = choose_case(2, 100, FP32)
    factor = torch.randn(2, 100, device="cuda")
    weight = torch.ones(2, 100, device="cuda", requires_grad=True)
    loss = (weight * factor).sum()
    choose(**case, processed=factor)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_pass():
    with torch.inference_mode():
        case, keep = rotate_case(4, 4, 2, 64, BF16)
        out = rotate_store(*case.values(), **keep)
        pick = choose_case(2, 100, FP32)
        choose(**pick, append=True)
    assert out.is_inference()
    rotate_store(*case.values(), **keep, out=out)


def test_compiled_functions_call_them():
    case = attend_case([20, 300], 4, 2, 64, BF16, seed=71)

    def layer(q, *rest):
        return paged_attention(q * 2, *rest).float() + 1

    want = layer(*case.values())
    got = torch.compile(layer, backend="eager")(*case.values())
    assert torch.equal(got, want)
