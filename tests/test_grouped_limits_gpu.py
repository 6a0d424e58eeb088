"""Products grouped by expert at the limits of their launches."""
import pytest
import torch

from sparsewave_b200 import Context
from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu


def signs(shape, seed):
    """-1, 0 and 1: every product, and every sum of fewer than 2^24 of them, is exact in f32."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-1, 2, shape, generator=gen, device="cuda", dtype=torch.int8).bfloat16()


@pytest.mark.parametrize("rows", [2 ** 24, 2 ** 24 + 1, 2 ** 25])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_weight_gradient_of_many_rows_off_a_boundary(ctx, rows, transpose_b):
    """Both operands are copied first, in slices of rows that one axis of the copy's grid counts (65,535 at most)."""
    A, dC = signs((rows, 9), 1), signs((rows, 11), 2)
    counts = [rows // 2, 0, rows - rows // 2]
    B = torch.empty((3, 11, 9) if transpose_b else (3, 9, 11), dtype=torch.bfloat16, device="cuda")
    _, dB = ctx.grouped_mm_grad(H.offsets_of(counts), A, B, dC, transpose_b=transpose_b, need_dA=False)
    exact = torch.zeros(B.shape, dtype=torch.float64, device="cuda")
    for g, lo, hi in ((0, 0, rows // 2), (2, rows // 2, rows)):
        left, right = (dC, A) if transpose_b else (A, dC)
        for at in range(lo, hi, 2 ** 22):
            part = slice(at, min(at + 2 ** 22, hi))
            exact[g] += left[part].double().t() @ right[part].double()
    assert float(exact.abs().max()) < 2 ** 24 and torch.equal(dB, exact.bfloat16())
    assert ctx.device_status() == 0


@pytest.mark.parametrize("k,pitch", [(1, 16), (9, 32), (100, 224), (300, 640)])
def test_memory_of_copies(k, pitch):
    """A call whose rows are short takes memory for them and not for whole lines (32 MB at a time, as the driver gives it out)."""
    rows = 2 ** 21
    A, B = signs((rows, k), 1), signs((1, k, 8), 2)
    offsets, C = H.offsets_of([rows]), torch.empty((rows, 8), dtype=torch.bfloat16, device="cuda")
    with Context(0) as fresh:
        fresh.grouped_mm(H.offsets_of([8]), A[:8, :1].repeat(1, 8), B[:, :1].repeat(1, 8, 1))  # loads the kernels
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        fresh.grouped_mm(offsets, A, B, C)
        torch.cuda.synchronize()
        assert before - torch.cuda.mem_get_info()[0] <= rows * pitch + 2 ** 26
    assert torch.equal(C, (A.double() @ B[0].double()).bfloat16())


def test_trim_gives_memory_back():
    rows = 2 ** 22
    A, B = signs((rows, 33), 1), signs((1, 33, 8), 2)
    offsets, C = H.offsets_of([rows]), torch.empty((rows, 8), dtype=torch.bfloat16, device="cuda")
    with Context(0) as fresh:
        fresh.trim()  # nothing kept so far
        fresh.grouped_mm(offsets, A, B, C)
        torch.cuda.synchronize()
        kept = torch.cuda.mem_get_info()[0]
        fresh.trim()
        assert torch.cuda.mem_get_info()[0] - kept >= rows * 96
        want = C.clone()
        assert torch.equal(fresh.grouped_mm(offsets, A, B, C.fill_(7.0)), want)  # memory anew
        fresh.trim()  # with the call perhaps in flight
        assert torch.equal(fresh.grouped_mm(offsets, A, B, C.fill_(7.0)), want)
