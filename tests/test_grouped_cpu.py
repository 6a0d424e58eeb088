"""Refusals of the products grouped by expert and of the 8-bit operands that need no GPU: the C ABI without a context, and the
Python calls' checks of their tensors."""
import pytest
import torch

from sparsewave_b200 import SparseWaveError, _lib


@pytest.mark.parametrize("name,args", [
    ("swb_grouped_mm", (0, 1, 1, 1, 1, None, None, None, 0, None, None)),
    ("swb_grouped_mm_grad", (0, 1, 1, 1, 1, None, None, None, None, 0, None, None, None)),
    ("swb_fp8_quantize_rows", (0, 3, 1, 1, None, None, None, None)),
    ("swb_fp8_quantize_blocks", (0, 3, 1, 1, 1, None, None, None, None)),
    ("swb_fp8_mm", (3, 3, 1, 1, 1, None, None, None, None, 0, None, None)),
    ("swb_fp8_grouped_mm", (3, 3, 1, 1, 1, 1, None, None, None, None, None, 0, None, None)),
])
def test_no_context(name, args):
    lib = _lib.load()
    assert getattr(lib, name)(None, *args) == _lib.SWB_ERR_INVALID_ARGUMENT
    assert lib.swb_last_error(None) == b"context is NULL"


def test_types_have_the_headers_values():
    assert (_lib.SWB_BF16, _lib.SWB_F16, _lib.SWB_F32, _lib.SWB_E4M3, _lib.SWB_E5M2) == (0, 1, 2, 3, 4)


def test_host_tensors_are_refused():
    fast = _lib.binding(SparseWaveError)
    A, B, offsets = torch.zeros((4, 8)), torch.zeros((2, 8, 16)), torch.zeros(3, dtype=torch.int32)
    A8, B8, scales = A.to(torch.float8_e4m3fn), B.to(torch.float8_e4m3fn), torch.zeros((1, 4))
    for call in (lambda: fast.grouped_mm(None, 0, offsets, A, B, None, False),
                 lambda: fast.grouped_mm_grad(None, 0, offsets, A, B, A, None, None, False, True, True),
                 lambda: fast.fp8_quantize(None, 0, True, A, None, None, torch.float8_e4m3fn),
                 lambda: fast.fp8_product(None, 0, offsets, A8, scales, B8, scales, None, False),
                 lambda: fast.fp8_product(None, 0, None, A8, scales, B8, scales, None, False)):
        with pytest.raises(TypeError, match="must be a CUDA tensor"):
            call()
    for call in (fast.grouped_mm, fast.grouped_mm_grad, fast.fp8_quantize, fast.fp8_product):
        with pytest.raises(TypeError, match="arguments"):
            call(None)
