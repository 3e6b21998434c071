"""Which paged cache goes with which batch: the others are refused before
anything is allocated or planned (their pools have other sizes and layouts)."""
import pytest
import torch

import tle


def cache(dtype):
    return tle.PagedKVCache(2, 64, tle.Shape(1, 32, 4, 64, 10000.0), device="cpu", dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float16])
def test_decode_over_fp32_pages(dtype):
    with pytest.raises(ValueError, match="float32"):
        tle.PagedDecodeBatch(cache(dtype), [torch.zeros(1, dtype=torch.int32)], [0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8, torch.float16])
def test_decode_over_bf16_pages(dtype):
    with pytest.raises(ValueError, match="bfloat16|bf16"):
        tle.PagedDecodeBatchBf16(cache(dtype), [torch.zeros(1, dtype=torch.int32)], [0])
