"""Products grouped by expert and their gradients against the formulas in 64 bits: group sizes from none to many tiles, sizes that
no tile or copy divides, both layouts of the weights, operands off a 16-byte boundary, rows of no group, NaN next door, captured
calls."""
import pytest
import torch

from sparsewave_b200 import SparseWaveError, _lib
from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu

COUNTS = {
    "one": [1],
    "gaps": [0, 0, 5, 0, 1, 0],
    "ragged": [300, 1, 0, 17, 129, 64],
    "around_tiles": [15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257],
    "long": [1500, 3],
    "many": [(7 * g) % 4 for g in range(200)],
}
SIZES = [(64, 64), (128, 128), (256, 384), (72, 136), (1000, 520), (640, 8), (8, 264), (1, 1), (17, 33), (130, 258), (193, 100)]


def check_forward(ctx, counts, k, n, dtype, transpose_b, first=0, behind=0, seed=0, shift=0):
    offsets = H.offsets_of(counts, first)
    rows = first + sum(counts) + behind
    A = torch.empty(rows * k + shift, dtype=dtype, device="cuda")[shift:].view(rows, k).copy_(H.normal((rows, k), dtype, seed))
    shape = (len(counts), n, k) if transpose_b else (len(counts), k, n)
    B = torch.empty(len(counts) * k * n + shift, dtype=dtype, device="cuda")[shift:].view(shape).copy_(
        H.normal(shape, dtype, seed + 1, k ** -0.5))
    C = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    assert ctx.grouped_mm(offsets, A, B, C, transpose_b=transpose_b) is C
    exact, size = H.grouped_mm(offsets, A, B, transpose_b)
    inside = slice(first, first + sum(counts))
    H.assert_rounded_sum(C[inside], exact[inside], size[inside], k)
    assert bool((C[:first] == 7.0).all()) and bool((C[first + sum(counts):] == 7.0).all())
    assert ctx.device_status() == 0


@pytest.mark.parametrize("k,n", SIZES)
@pytest.mark.parametrize("transpose_b", [False, True])
@pytest.mark.parametrize("counts", COUNTS)
def test_product(ctx, counts, k, n, transpose_b):
    dtype = torch.float16 if (k + n) % 16 == 0 else torch.bfloat16
    check_forward(ctx, COUNTS[counts], k, n, dtype, transpose_b, seed=k + n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("first,behind", [(0, 70), (3, 0), (129, 300)])
@pytest.mark.parametrize("k,n", [(256, 128), (48, 40), (33, 50)])
def test_rows_of_no_group_are_left_alone(ctx, dtype, first, behind, k, n):
    check_forward(ctx, [20, 0, 150, 3], k, n, dtype, True, first, behind, seed=first)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_operands_off_a_boundary(ctx, shift, transpose_b):
    check_forward(ctx, [40, 9, 0, 100], 128, 192, torch.bfloat16, transpose_b, seed=shift, shift=shift)


@pytest.mark.parametrize("counts", [[8], [3, 0, 1], [1] * 8 + [0] * 56, [70] * 8, [513, 511]])
@pytest.mark.parametrize("k,n", [(4096, 1024), (2048, 1536), (8192, 256)])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_long_inner_axis(ctx, counts, k, n, transpose_b):
    check_forward(ctx, counts, k, n, torch.bfloat16, transpose_b, behind=2, seed=len(counts))


def test_large(ctx):
    check_forward(ctx, [4000, 0, 2500, 1692], 2048, 2304, torch.bfloat16, True)
    check_forward(ctx, [4000, 0, 2500, 1692], 2048, 2304, torch.float16, False)


def test_no_rows_no_inner(ctx):
    B = H.normal((3, 16, 32), torch.bfloat16, 1)
    C = ctx.grouped_mm(H.offsets_of([0, 0, 0]), torch.empty((0, 16), dtype=torch.bfloat16, device="cuda"), B)
    assert C.shape == (0, 32)
    C = torch.full((5, 32), 7.0, dtype=torch.float16, device="cuda")
    ctx.grouped_mm(H.offsets_of([2, 1]), torch.empty((5, 0), dtype=torch.float16, device="cuda"),
                   torch.empty((2, 0, 32), dtype=torch.float16, device="cuda"), C)
    assert bool((C[:3] == 0).all()) and bool((C[3:] == 7.0).all())


@pytest.mark.parametrize("k,n", [(256, 256), (41, 30)])
@pytest.mark.parametrize("transpose_b", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_next_door_do_not_leak(ctx, k, n, transpose_b, bad):
    """Rows of A that are NaN or infinite spoil their own rows of C and the gradient of their own group only; weights of a group
    without rows spoil nothing."""
    counts = [30, 7, 0, 90, 200, 11]
    offsets = H.offsets_of(counts, 5)
    rows = sum(counts) + 5 + 9
    A, dC = H.normal((rows, k), torch.bfloat16, 1), H.normal((rows, n), torch.bfloat16, 2)
    B = H.normal((6, n, k) if transpose_b else (6, k, n), torch.bfloat16, 3, k ** -0.5)
    C = ctx.grouped_mm(offsets, A, B, transpose_b=transpose_b)
    dA, dB = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b)
    A2, B2, dC2 = A.clone(), B.clone(), dC.clone()
    spoiled = list(range(5)) + [35 + 5] + list(range(rows - 9, rows))
    for r in spoiled:
        A2[r] = bad
        dC2[r] = bad
    B2[2] = bad
    C2 = ctx.grouped_mm(offsets, A2, B2, transpose_b=transpose_b)
    dA2, dB2 = ctx.grouped_mm_grad(offsets, A2, B2, dC2, transpose_b=transpose_b)
    inside = torch.ones(rows, dtype=torch.bool, device="cuda")
    inside[spoiled] = False
    assert torch.equal(C2[inside], C[inside]) and torch.equal(dA2[inside], dA[inside])
    assert not bool(C2[40].isfinite().any()) and not bool(dA2[40].isfinite().any())
    kept = [0, 2, 3, 4, 5]
    assert torch.equal(dB2[kept], dB[kept]) and bool((dB2[2] == 0).all())
    assert not bool(dB2[1].isfinite().any())


@pytest.mark.parametrize("k,n", [(128, 128), (256, 384), (72, 136), (1000, 520), (8, 264), (1, 1), (17, 33), (130, 258)])
@pytest.mark.parametrize("transpose_b", [False, True])
@pytest.mark.parametrize("counts", ["one", "gaps", "ragged", "around_tiles", "many"])
def test_gradients(ctx, counts, k, n, transpose_b):
    counts = COUNTS[counts]
    dtype = torch.float16 if (k + n) % 16 == 0 else torch.bfloat16
    offsets, rows = H.offsets_of(counts, 2), sum(counts) + 4
    A, dC = H.normal((rows, k), dtype, 1), H.normal((rows, n), dtype, 2)
    B = H.normal((len(counts), n, k) if transpose_b else (len(counts), k, n), dtype, 3, k ** -0.5)
    dA = torch.full_like(A, 7.0)
    dB = torch.full_like(B, 7.0)
    got = ctx.grouped_mm_grad(offsets, A, B, dC, dA, dB, transpose_b=transpose_b)
    assert got[0] is dA and got[1] is dB
    exact, size = H.grouped_mm(offsets, dC, B, not transpose_b)
    H.assert_rounded_sum(dA[2:-2], exact[2:-2], size[2:-2], n)
    assert bool((dA[:2] == 7.0).all()) and bool((dA[-2:] == 7.0).all())
    exact, size = H.weight_gradient(offsets, A, dC, transpose_b, B)
    H.assert_rounded_sum(dB, exact, size, max(counts))
    only_a, none = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b, need_dB=False)
    assert none is None and torch.equal(only_a[2:-2], dA[2:-2])
    none, only_b = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b, need_dA=False)
    assert none is None and torch.equal(only_b, dB)


@pytest.mark.parametrize("transpose_b", [False, True])
@pytest.mark.parametrize("k,n", [(256, 384), (15, 21)])
def test_gradients_are_differences(ctx, transpose_b, k, n):
    """On small integers every product, sum and rounding is exact, and so is the difference of the scalar sum(C * dC), which
    is linear in A and in B: it equals the gradient times the step."""
    counts = [33, 0, 90, 5]
    offsets, rows = H.offsets_of(counts), sum(counts)
    gen = torch.Generator(device="cuda").manual_seed(7)

    def sparse(shape, share):  # -1, 0, 1, few of them: sums below 256, which bf16 holds
        return (torch.randint(-1, 2, shape, generator=gen, device="cuda")
                * (torch.rand(shape, generator=gen, device="cuda") < share)).bfloat16()

    A, dC = sparse((rows, k), 0.3), sparse((rows, n), 0.3)
    shape = (4, n, k) if transpose_b else (4, k, n)
    B, step_A, step_B = sparse(shape, 0.3), sparse((rows, k), 0.3), sparse(shape, 0.3)
    dA, dB = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b)

    def scalar(a, b):
        return (ctx.grouped_mm(offsets, a, b, transpose_b=transpose_b).double() * dC.double()).sum()

    here = scalar(A, B)
    assert scalar(A + step_A, B) - here == (dA.double() * step_A.double()).sum()
    assert scalar(A, B + step_B) - here == (dB.double() * step_B.double()).sum()


def test_wrong_offsets_touch_nothing_outside(ctx):
    """Offsets outside the rows are clipped; the guard rows around C stay."""
    A, B = H.normal((50, 64), torch.bfloat16, 1), H.normal((3, 64, 128), torch.bfloat16, 2)
    offsets = torch.tensor([-20, 30, 10 ** 9, 2 * 10 ** 9], dtype=torch.int32, device="cuda")
    guarded = torch.full((150, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ctx.grouped_mm(offsets, A, B, guarded[50:100])
    exact, size = H.grouped_mm(H.offsets_of([30, 20, 0]), A, B, False)
    H.assert_rounded_sum(guarded[50:100], exact, size, 64)
    assert bool((guarded[:50] == 7.0).all()) and bool((guarded[100:] == 7.0).all())


@pytest.mark.parametrize("rows,groups,k,n", [(3000, 900, 64, 128), (40, 2, 64, 128), (3000, 12, 33, 50)])
def test_offsets_that_decrease_make_no_rows(ctx, rows, groups, k, n):
    A, B = H.normal((rows, k), torch.bfloat16, 1), H.normal((groups, k, n), torch.bfloat16, 2)
    offsets = torch.tensor([0 if g % 2 == 0 else rows for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    C, dA, dC = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full_like(A, 7.0), H.normal((rows, n), torch.bfloat16, 3)
    ctx.grouped_mm(offsets, A, B, C)
    _, dB = ctx.grouped_mm_grad(offsets, A, B, dC, dA)
    assert bool((C == 7.0).all()) and bool((dA == 7.0).all()) and bool((dB == 0).all()) and ctx.device_status() == 0
    one = torch.tensor([5, 3], dtype=torch.int32, device="cuda")
    ctx.grouped_mm(one, A, B[:1], C)
    assert bool((C == 7.0).all())
    ctx.grouped_mm(H.offsets_of([rows]), A, B[:1], C)
    exact, size = H.grouped_mm(H.offsets_of([rows]), A, B[:1], False)
    H.assert_rounded_sum(C, exact, size, k)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("counts", [[5], [70, 0, 30], [400, 90]])
def test_results_off_a_boundary(ctx, shift, counts):
    offsets, rows = H.offsets_of(counts), sum(counts)
    A, B = H.normal((rows, 256), torch.bfloat16, 1), H.normal((len(counts), 136, 256), torch.bfloat16, 2)
    dC = H.normal((rows, 136), torch.bfloat16, 3)

    def room(shape):
        size = 1
        for n in shape:
            size *= n
        flat = torch.full((size + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
        return flat, flat[shift:shift + size].view(shape)

    flats, (C, dA, dB) = zip(*(room(s) for s in ((rows, 136), (rows, 256), tuple(B.shape))))
    ctx.grouped_mm(offsets, A, B, C, transpose_b=True)
    ctx.grouped_mm_grad(offsets, A, B, dC, dA, dB, transpose_b=True)
    assert torch.equal(C, ctx.grouped_mm(offsets, A, B, transpose_b=True))
    want = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=True)
    assert torch.equal(dA, want[0]) and torch.equal(dB, want[1])
    for flat, t in zip(flats, (C, dA, dB)):
        assert bool((flat[:shift] == 7.0).all()) and bool((flat[shift + t.numel():] == 7.0).all())


@pytest.mark.parametrize("k,n,rows", [(512, 256, 400), (512, 256, 24), (31, 45, 70)])
def test_captured_with_other_group_sizes(ctx, k, n, rows):
    """A captured forward and backward pass replayed with other offsets and operands, beside an eager call in between."""
    A, dC, B = H.normal((rows, k), torch.bfloat16, 1), H.normal((rows, n), torch.bfloat16, 2), H.normal((4, k, n), torch.bfloat16, 3)
    offsets = H.offsets_of([rows, 0, 0, 0])
    C, dA, dB = torch.zeros_like(dC), torch.zeros_like(A), torch.zeros_like(B)
    ctx.grouped_mm(offsets, A, B, C)
    ctx.grouped_mm_grad(offsets, A, B, dC, dA, dB)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.grouped_mm(offsets, A, B, C)
        ctx.grouped_mm_grad(offsets, A, B, dC, dA, dB)
    for counts in ([rows // 2, 0, 1, rows - rows // 2 - 1], [0, 0, 0, rows], [5, 6, 7, 2]):
        offsets.copy_(H.offsets_of(counts))
        A.copy_(H.normal((rows, k), torch.bfloat16, sum(counts[:2])))
        for t in (C, dA, dB):
            t.fill_(7.0)
        graph.replay()
        eager = ctx.grouped_mm(offsets, A, B, torch.full_like(C, 7.0))
        eager_a, eager_b = ctx.grouped_mm_grad(offsets, A, B, dC, torch.full_like(A, 7.0))
        assert torch.equal(C, eager) and torch.equal(dA, eager_a) and torch.equal(dB, eager_b)
        exact, size = H.grouped_mm(offsets, A, B, False)
        used = sum(counts)
        H.assert_rounded_sum(C[:used], exact[:used], size[:used], k)


def test_streams_and_repeats_give_the_same_bits(ctx):
    counts = [100, 3, 0, 260]
    offsets, rows = H.offsets_of(counts), sum(counts)
    A, B = H.normal((rows, 640), torch.bfloat16, 1), H.normal((4, 640, 320), torch.bfloat16, 2)
    dC = H.normal((rows, 320), torch.bfloat16, 3)
    want, want_grad = ctx.grouped_mm(offsets, A, B), ctx.grouped_mm_grad(offsets, A, B, dC)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            results.append((ctx.grouped_mm(offsets, A, B), *ctx.grouped_mm_grad(offsets, A, B, dC)))
    torch.cuda.synchronize()
    for C, dA, dB in results:
        assert torch.equal(C, want) and torch.equal(dA, want_grad[0]) and torch.equal(dB, want_grad[1])


def test_refusals(ctx):
    A, B = H.normal((8, 16), torch.bfloat16, 1), H.normal((2, 16, 24), torch.bfloat16, 2)
    dC, offsets = H.normal((8, 24), torch.bfloat16, 3), H.offsets_of([4, 4])

    def refused(status, call):
        with pytest.raises(SparseWaveError) as e:
            call()
        assert e.value.status == status

    shape, capacity = _lib.SWB_ERR_INVALID_SHAPE, _lib.SWB_ERR_CAPACITY
    refused(shape, lambda: ctx.grouped_mm(offsets[:2], A, B))
    refused(shape, lambda: ctx.grouped_mm(offsets, A, B, transpose_b=True))
    refused(shape, lambda: ctx.grouped_mm(offsets, A[0], B))
    refused(shape, lambda: ctx.grouped_mm(offsets, A, B, torch.empty((8, 23), dtype=torch.bfloat16, device="cuda")))
    refused(shape, lambda: ctx.grouped_mm(offsets, A, B[:, :, :0]))
    refused(shape, lambda: ctx.grouped_mm(offsets[:1], A, B[:0]))
    refused(shape, lambda: ctx.grouped_mm_grad(offsets, A, B, dC[:7]))
    refused(shape, lambda: ctx.grouped_mm_grad(offsets, A, B, dC, torch.empty_like(B)))
    refused(shape, lambda: ctx.grouped_mm_grad(offsets, A[:, :0], B[:, :0], dC))
    many = 1025
    refused(capacity, lambda: ctx.grouped_mm(H.offsets_of([0] * many), A, torch.zeros((many, 16, 8), dtype=torch.bfloat16, device="cuda")))
    for call in (lambda: ctx.grouped_mm(offsets.long(), A, B), lambda: ctx.grouped_mm(offsets, A.half(), B),
                 lambda: ctx.grouped_mm(offsets, A.float(), B.float()), lambda: ctx.grouped_mm(offsets, A.cpu(), B),
                 lambda: ctx.grouped_mm(offsets, A.t().contiguous().t(), B), lambda: ctx.grouped_mm(offsets.cpu(), A, B),
                 lambda: ctx.grouped_mm(offsets, A, B.transpose(1, 2).contiguous().transpose(1, 2)),
                 lambda: ctx.grouped_mm(offsets, A, B, torch.empty((8, 24), dtype=torch.float16, device="cuda")),
                 lambda: ctx.grouped_mm_grad(offsets, A, B, dC.half()), lambda: ctx.grouped_mm(None, A, B)):
        with pytest.raises(TypeError):
            call()
    assert torch.equal(ctx.grouped_mm(offsets, A, B), ctx.grouped_mm(offsets, A, B))  # the context still works


def test_the_largest_number_of_groups(ctx):
    counts = [1 if g % 3 == 0 else 0 for g in range(1024)]
    check_forward(ctx, counts, 64, 128, torch.bfloat16, True)
    check_forward(ctx, counts, 24, 12, torch.bfloat16, False)


@pytest.mark.parametrize("groups,most", [(40, 700), (128, 300), (129, 300), (300, 90)])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_many_ragged_groups(ctx, groups, most, transpose_b):
    """More tiles than run at a time, groups from none to many: both orders in which groups are taken."""
    gen = torch.Generator().manual_seed(groups)
    counts = (torch.rand(groups, generator=gen) ** 3 * most).int().tolist()
    counts[3], counts[7] = 0, most * 2
    check_forward(ctx, counts, 192, 520, torch.bfloat16, transpose_b, first=1, behind=3, seed=groups)
    offsets, rows = H.offsets_of(counts, 1), sum(counts) + 2
    A, dC = H.normal((rows, 192), torch.bfloat16, 1), H.normal((rows, 520), torch.bfloat16, 2)
    B = H.normal((groups, 520, 192) if transpose_b else (groups, 192, 520), torch.bfloat16, 3)
    _, dB = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b, need_dA=False)
    exact, size = H.weight_gradient(offsets, A, dC, transpose_b, B)
    H.assert_rounded_sum(dB, exact, size, max(counts))


@pytest.mark.parametrize("rows", [3, 20, 40, 70, 100, 150, 250, 500])
@pytest.mark.parametrize("k", [128, 192, 320, 448, 1024, 1088, 2496])
def test_shared_inner_axes(ctx, rows, k):
    """One group and few columns: the inner axis shared among every number of CTAs, odd ones too, by tiles of 64, 128 and 256 rows."""
    check_forward(ctx, [rows], k, 136, torch.bfloat16, True, behind=1, seed=rows)
    check_forward(ctx, [rows // 2, 0, rows - rows // 2], k, 40, torch.float16, False, seed=k)


def test_subnormal_values(ctx):
    """fp16 subnormals count as what they are, as operands and in the result."""
    A = (torch.arange(64 * 64, device="cuda").view(64, 64) % 37).half() * 2.0 ** -24
    B = torch.full((1, 64, 64), 2.0 ** 3, dtype=torch.float16, device="cuda")
    C = ctx.grouped_mm(H.offsets_of([64]), A, B)
    exact, size = H.grouped_mm(H.offsets_of([64]), A, B, False)
    H.assert_rounded_sum(C, exact, size, 64)
    C = ctx.grouped_mm(H.offsets_of([64]), A, B * 2.0 ** -6)
    exact, size = H.grouped_mm(H.offsets_of([64]), A, B * 2.0 ** -6, False)
    H.assert_rounded_sum(C, exact, size, 64)


def test_a_value_past_the_largest(ctx):
    """Sums above fp16's largest value become infinities, as rounding has it."""
    A, B = torch.full((3, 64), 200.0, dtype=torch.float16, device="cuda"), torch.full((1, 64, 16), 10.0, dtype=torch.float16, device="cuda")
    assert bool((ctx.grouped_mm(H.offsets_of([3]), A, B) == float("inf")).all())
    assert bool((ctx.grouped_mm(H.offsets_of([3]), A.bfloat16(), B.bfloat16()) == 128000.0).all())


def test_past_two_to_the_31_elements(ctx):
    """Weights of 2.4e9 elements of which the last groups are used, and a result of 2.2e9."""
    groups, k, n = 300, 1024, 7808
    B = torch.zeros((groups, n, k), dtype=torch.bfloat16, device="cuda")
    B[298] = H.normal((n, k), torch.bfloat16, 1)
    A = H.normal((70, k), torch.bfloat16, 2)
    offsets = H.offsets_of([0] * 298 + [70, 0])
    C = ctx.grouped_mm(offsets, A, B, transpose_b=True)
    exact, size = H.grouped_mm(H.offsets_of([70]), A, B[298:299], True)
    H.assert_rounded_sum(C, exact, size, k)
    del B
    rows, n = 540000, 4096
    A, B = H.normal((rows, 16), torch.bfloat16, 3), H.normal((2, 16, n), torch.bfloat16, 4)
    C = ctx.grouped_mm(H.offsets_of([rows - 100, 100]), A, B)
    exact, size = H.grouped_mm(H.offsets_of([100]), A[-100:], B[1:], False)
    H.assert_rounded_sum(C[-100:], exact, size, 16)
    dA, dB = ctx.grouped_mm_grad(H.offsets_of([rows - 100, 100]), A, B, C)
    exact, size = H.grouped_mm(H.offsets_of([100]), C[-100:], B[1:], True)
    H.assert_rounded_sum(dA[-100:], exact, size, n)
    exact, size = H.weight_gradient(H.offsets_of([100]), A[-100:], C[-100:], False, B[1:])
    H.assert_rounded_sum(dB[1:], exact, size, 100)


def test_two_graphs_at_a_time(ctx):
    """Two captured layers, whose operands off a boundary are copied in memory of their own, replayed on two streams at once."""
    layers = []
    for seed in range(2):
        A, B = H.normal((300, 511), torch.bfloat16, seed), H.normal((3, 511, 333), torch.bfloat16, seed + 2)
        offsets = H.offsets_of([100 + seed, 150, 50 - seed])
        C = torch.empty((300, 333), dtype=torch.bfloat16, device="cuda")
        ctx.grouped_mm(offsets, A, B, C)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ctx.grouped_mm(offsets, A, B, C)
        layers.append((A, B, offsets, C, graph))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (A, B, offsets, C, graph), stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                C.fill_(7.0)
                graph.replay()
    torch.cuda.synchronize()
    for A, B, offsets, C, _ in layers:
        exact, size = H.grouped_mm(offsets, A, B, False)
        H.assert_rounded_sum(C, exact, size, 511)


def test_other_kernels_in_between(ctx):
    """Calls queued behind one another and behind the block-sparse product, each reading what the one before wrote."""
    from sparsewave_b200 import workloads as W
    m, Bb = W.config_c5(device="cuda", block_grid=160, n_rhs=128)
    bsr = lambda: ctx.bsr_spmm("", m.block_row_ptr, m.block_col_idx, m.block_values, Bb, 16)
    X = bsr()
    rows = X.shape[0]
    offsets = H.offsets_of([rows // 3, 0, rows - rows // 3])
    W1, W2 = H.normal((3, 128, 64), torch.bfloat16, 1, 0.1), H.normal((3, 64, 128), torch.bfloat16, 2, 0.1)
    want = ctx.grouped_mm(offsets, ctx.grouped_mm(offsets, X, W1), W2)
    for _ in range(10):
        got = ctx.grouped_mm(offsets, ctx.grouped_mm(offsets, bsr(), W1), W2)
        assert torch.equal(got, want)


@pytest.mark.parametrize("counts", [[5000], [3001, 0], [64], [1900, 2500, 77], [20011]])
@pytest.mark.parametrize("k,n", [(128, 128), (136, 520), (31, 45), (257, 1000)])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_weight_gradients_of_long_groups(ctx, counts, k, n, transpose_b):
    """Few tiles and many rows: a group's rows shared among several parts, whose sums are added; groups shorter than a part."""
    dtype = torch.float16 if k % 2 else torch.bfloat16
    offsets, rows = H.offsets_of(counts, 3), sum(counts) + 5
    A, dC = H.normal((rows, k), dtype, 1), H.normal((rows, n), dtype, 2)
    A[:3], dC[-2:] = float("nan"), float("inf")
    B = H.normal((len(counts), n, k) if transpose_b else (len(counts), k, n), dtype, 3)
    _, dB = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b, need_dA=False)
    exact, size = H.weight_gradient(offsets, A, dC, transpose_b, B)
    H.assert_rounded_sum(dB, exact, size, max(counts))
    _, again = ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=transpose_b, need_dA=False)
    assert torch.equal(dB, again) and ctx.device_status() == 0
