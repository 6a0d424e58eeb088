"""8-bit operands with block scales: quantisation bit for bit, products against the formulas in 64 bits, and a layer of experts
made of them."""
import pytest
import torch

from sparsewave_b200 import SparseWaveError, _lib
from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu

FP8 = [torch.float8_e4m3fn, torch.float8_e5m2]


def bits(t):
    return t.contiguous().view(torch.uint8)


def spread_values(shape, dtype, seed):
    """Values over some ten binades, a few large ones, whole blocks of zeros."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda") * torch.exp2(torch.randint(-6, 4, shape, generator=gen, device="cuda").float())
    x[..., : min(128, shape[-1] // 3)] = 0.0
    return x.to(dtype)


def assert_quantised(X, Q, scales):
    """Against the definition in 64 bits: the scale to half a step of f32 (2^-24), the value to half a step of the 8-bit type."""
    largest, info = H.LARGEST[Q.dtype], torch.finfo(Q.dtype)
    by_rows = X.dim() == 2 and scales.shape[-1] == X.shape[0] and scales.shape[0] == -(-X.shape[1] // 128)
    spread = H.spread_rows(scales, X.shape[1]) if by_rows else H.spread_blocks(scales, X.shape[-2], X.shape[-1])
    ratio = X.double() / spread.double()
    assert float(ratio.abs().max()) <= largest * (1 + 2.0 ** -23)
    step = info.eps / 2 * ratio.abs().clamp_min(info.smallest_normal) * (1 + 2.0 ** -20)
    assert bool(((Q.double() - ratio).abs() <= step).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (17, 200), (64, 4096), (5, 1004), (130, 136), (257, 640), (33, 7)])
@pytest.mark.parametrize("out", FP8)
def test_quantize_rows(ctx, dtype, rows, cols, out):
    X = spread_values((rows, cols), dtype, rows + cols)
    Q, scales = ctx.fp8_quantize_rows(X, dtype=out)
    q, s = H.quantize_rows(X, out)
    assert Q.dtype == out and torch.equal(scales, s) and torch.equal(bits(Q), bits(q))
    assert_quantised(X, Q, scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (2, 130, 260), (3, 384, 1000), (7, 5, 4), (1, 640, 256)])
@pytest.mark.parametrize("out", FP8)
def test_quantize_blocks(ctx, dtype, shape, out):
    X = spread_values(shape, dtype, sum(shape))
    Q, scales = ctx.fp8_quantize_blocks(X, dtype=out)
    q, s = H.quantize_blocks(X, out)
    assert Q.shape == X.shape and torch.equal(scales, s) and torch.equal(bits(Q), bits(q))


@pytest.mark.parametrize("shift", [1, 2, 3, 4])
def test_quantize_off_a_boundary(ctx, shift):
    X = torch.empty(50 * 256 + shift, dtype=torch.bfloat16, device="cuda")[shift:].view(50, 256).copy_(spread_values((50, 256), torch.bfloat16, 1))
    room = torch.full((50 * 256 + 16,), 9, dtype=torch.uint8, device="cuda")
    Q = room[shift:shift + 50 * 256].view(torch.float8_e4m3fn).view(50, 256)
    for call, plain in ((ctx.fp8_quantize_rows, H.quantize_rows), (ctx.fp8_quantize_blocks, H.quantize_blocks)):
        got, scales = call(X, Q)
        assert got is Q and torch.equal(bits(Q), bits(plain(X)[0])) and torch.equal(scales, plain(X)[1])
        assert bool((room[:shift] == 9).all()) and bool((room[shift + 50 * 256:] == 9).all())


def test_quantize_values_at_the_edges(ctx):
    """Zeros, the tiniest and the largest values; an infinity or a NaN spoils its own block alone."""
    X = torch.zeros((6, 256), dtype=torch.float32, device="cuda")
    X[1, :128] = 1e-45
    X[2, :128] = torch.finfo(torch.float32).max
    X[3, 5], X[3, 200] = float("inf"), 3.0
    X[4, 7], X[4, 201] = float("nan"), -2.0
    X[5, :2] = torch.tensor([-448.0, 17.0])  # 17 lies between 16 and 18: to the even one
    Q, scales = ctx.fp8_quantize_rows(X)
    q, s = H.quantize_rows(X)
    assert torch.equal(scales.nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert torch.equal(Q.double().nan_to_num(-1.0), q.double().nan_to_num(-1.0))
    assert scales[0, 0] == 2.0 ** -126 and bool((Q[0].double() == 0).all())
    assert Q[2, 0].double() == 448 and Q[5, :2].double().tolist() == [-448.0, 16.0]
    assert scales[0, 3] == float("inf") and bool(scales[0, 4].isnan()) and bool(scales[1].isfinite().all())
    assert Q[3, 200].double() == 448 and Q[4, 201].double() == -448
    Qb, sb = ctx.fp8_quantize_blocks(X)
    assert bool(sb[0, 0].isnan()) and sb[0, 1] == H.scale_of(torch.tensor(3.0, device="cuda"), Q.dtype)
    C = ctx.fp8_mm(Q, scales, *ctx.fp8_quantize_blocks(torch.ones((256, 64), device="cuda")))
    assert bool(C[[0, 1, 5]].isfinite().all()) and bool(C[3:5].isnan().all())
    assert bool((C[2] == float("inf")).all())  # 128 times the largest f32 value


def check_product(ctx, counts, k, n, transpose_b, a_type=FP8[0], b_type=FP8[0], first=0, behind=0, seed=0):
    """counts: rows of each group, or a number: one matrix."""
    grouped = isinstance(counts, list)
    rows = first + (sum(counts) if grouped else counts) + behind
    A, As = ctx.fp8_quantize_rows(H.normal((rows, k), torch.bfloat16, seed) * torch.exp(H.normal((rows, 1), torch.float32, seed + 2)), dtype=a_type)
    shape = (n, k) if transpose_b else (k, n)
    W = H.normal(((len(counts),) if grouped else ()) + shape, torch.bfloat16, seed + 1, k ** -0.5)
    B, Bs = ctx.fp8_quantize_blocks(W, dtype=b_type)
    C = torch.full((rows, n), 7.0, dtype=torch.bfloat16, device="cuda")
    if grouped:
        offsets = H.offsets_of(counts, first)
        ctx.fp8_grouped_mm(offsets, A, As, B, Bs, C, transpose_b=transpose_b)
    else:
        offsets = None
        ctx.fp8_mm(A, As, B, Bs, C, transpose_b=transpose_b)
    exact, size = H.fp8_grouped_mm(offsets, A, As, B, Bs, transpose_b)
    inside = slice(first, rows - behind)
    H.assert_rounded_sum(C[inside], exact[inside], size[inside], k)
    assert bool((C[:first] == 7.0).all()) and bool((C[rows - behind:] == 7.0).all())
    assert ctx.device_status() == 0


@pytest.mark.parametrize("rows", [1, 5, 16, 33, 64, 130, 300, 1000])
@pytest.mark.parametrize("k,n", [(128, 128), (512, 384), (4096, 256), (144, 272), (1040, 96), (1, 1), (77, 50), (200, 130)])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_matrix(ctx, rows, k, n, transpose_b):
    check_product(ctx, rows, k, n, transpose_b, seed=rows)


@pytest.mark.parametrize("counts", [[1], [0, 5, 0, 1], [300, 1, 0, 17, 129, 64], [(7 * g) % 4 for g in range(100)],
                                    [15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257]])
@pytest.mark.parametrize("k,n", [(256, 256), (1024, 400), (48, 144), (99, 35)])
@pytest.mark.parametrize("transpose_b", [False, True])
def test_grouped(ctx, counts, k, n, transpose_b):
    check_product(ctx, counts, k, n, transpose_b, first=2, behind=5, seed=k)


@pytest.mark.parametrize("a_type", FP8)
@pytest.mark.parametrize("b_type", FP8)
@pytest.mark.parametrize("counts", [9, 200, [70, 0, 300]])
def test_types(ctx, a_type, b_type, counts):
    for k, n, transpose_b in ((384, 256, True), (384, 256, False), (50, 30, True)):
        check_product(ctx, counts, k, n, transpose_b, a_type, b_type)


def test_large(ctx):
    check_product(ctx, 4096, 4096, 2304, True)
    check_product(ctx, [3000, 0, 1000, 96], 2048, 2560, False)


def test_no_rows_no_inner(ctx):
    e = torch.empty
    f8 = torch.float8_e4m3fn
    C = ctx.fp8_mm(e((0, 64), dtype=f8, device="cuda"), e((1, 0), device="cuda"), *ctx.fp8_quantize_blocks(torch.ones((64, 32), device="cuda")))
    assert C.shape == (0, 32)
    C = ctx.fp8_mm(e((4, 0), dtype=f8, device="cuda"), e((0, 4), device="cuda"), e((0, 32), dtype=f8, device="cuda"), e((0, 1), device="cuda"))
    assert C.shape == (4, 32) and bool((C == 0).all())
    Q, s = ctx.fp8_quantize_rows(e((0, 64), device="cuda"))
    assert Q.shape == (0, 64) and s.shape == (1, 0)
    Q, s = ctx.fp8_quantize_blocks(e((3, 64, 0), device="cuda"))
    assert Q.shape == (3, 64, 0) and s.shape == (3, 1, 0)


def test_rows_next_door_do_not_leak(ctx):
    counts = [40, 7, 100]
    offsets, rows = H.offsets_of(counts), sum(counts)
    A, As = ctx.fp8_quantize_rows(H.normal((rows, 256), torch.bfloat16, 1))
    B, Bs = ctx.fp8_quantize_blocks(H.normal((3, 192, 256), torch.bfloat16, 2))
    C = ctx.fp8_grouped_mm(offsets, A, As, B, Bs, transpose_b=True)
    A2, As2 = A.clone(), As.clone()
    A2[41:43] = torch.full((2, 256), float("nan"), device="cuda").to(A.dtype)
    As2[:, 44] = float("inf")
    C2 = ctx.fp8_grouped_mm(offsets, A2, As2, B, Bs, transpose_b=True)
    rest = [r for r in range(rows) if r not in (41, 42, 44)]
    assert torch.equal(C2[rest], C[rest]) and not bool(C2[[41, 42, 44]].isfinite().any())


@pytest.mark.parametrize("tokens,groups,k,n", [(70, 8, 256, 384), (1, 16, 512, 128), (600, 4, 200, 90)])
def test_layer_of_experts(ctx, tokens, groups, k, n):
    """Tokens routed to two experts each: rows sorted by expert, to 8 bits, through two 8-bit products with a rectifier between
    them, weighted back to the tokens; every step held to the formula on the operands that it got."""
    X = H.normal((tokens, k), torch.bfloat16, 1)
    up, down = H.normal((groups, n, k), torch.bfloat16, 2, k ** -0.5), H.normal((groups, k, n), torch.bfloat16, 3, n ** -0.5)
    up8, up_scales = ctx.fp8_quantize_blocks(up)
    down8, down_scales = ctx.fp8_quantize_blocks(down)
    share, expert = torch.softmax(H.normal((tokens, groups), torch.float32, 4), 1).topk(2)
    order = expert.flatten().argsort(stable=True)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.bincount(expert.flatten(), minlength=groups).cumsum(0)
    rows = X[order // 2]
    A, As = ctx.fp8_quantize_rows(rows)
    hidden = ctx.fp8_grouped_mm(offsets, A, As, up8, up_scales, transpose_b=True)
    exact, size = H.fp8_grouped_mm(offsets, A, As, up8, up_scales, True)
    H.assert_rounded_sum(hidden, exact, size, k)
    active = hidden.relu()
    A2, As2 = ctx.fp8_quantize_rows(active)
    out = ctx.fp8_grouped_mm(offsets, A2, As2, down8, down_scales, transpose_b=True)
    exact, size = H.fp8_grouped_mm(offsets, A2, As2, down8, down_scales, True)
    H.assert_rounded_sum(out, exact, size, n)
    tokens_out = torch.zeros((tokens, k), device="cuda").index_add_(0, order // 2, out.float() * share.flatten()[order, None])
    # Against the layer in 64 bits.  Each 8-bit operand is off by at most 2^-4 of the larger of itself and 2^-6 of its scale's unit,
    # so a product of two by less than 2 * 2^-4 + 2^-8 of the two's size plus the small ones; taken together as a norm over
    # all outputs, where the errors of single products have no sign in common, well below 2^-3 per product: 2^-2 for two.
    hidden_exact, _ = H.grouped_mm(offsets, rows, up, True)
    out_exact, _ = H.grouped_mm(offsets, hidden_exact.relu(), down, True)
    want = torch.zeros((tokens, k), dtype=torch.float64, device="cuda").index_add_(0, order // 2, out_exact * share.flatten()[order, None].double())
    assert float((tokens_out.double() - want).norm() / want.norm()) < 0.25
    # the gradient of the rows: dC to 8 bits, the same weights the other way round
    dC = H.normal(tuple(out.shape), torch.bfloat16, 5)
    G, Gs = ctx.fp8_quantize_rows(dC, dtype=torch.float8_e5m2)
    dA = ctx.fp8_grouped_mm(offsets, G, Gs, down8, down_scales)
    exact, size = H.fp8_grouped_mm(offsets, G, Gs, down8, down_scales, False)
    H.assert_rounded_sum(dA, exact, size, k)
    _, dB = ctx.grouped_mm_grad(offsets, active, down, dC, transpose_b=True, need_dA=False)
    exact, size = H.weight_gradient(offsets, active, dC, True, down)
    H.assert_rounded_sum(dB, exact, size, 2 * tokens)
    assert ctx.device_status() == 0


def test_captured(ctx):
    X = H.normal((48, 512), torch.bfloat16, 1)
    B, Bs = ctx.fp8_quantize_blocks(H.normal((4, 256, 512), torch.bfloat16, 2))
    offsets = H.offsets_of([48, 0, 0, 0])

    def layer():
        return ctx.fp8_grouped_mm(offsets, *ctx.fp8_quantize_rows(X), B, Bs, transpose_b=True)

    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        C = layer()
    for seed, counts in ((3, [10, 0, 30, 8]), (4, [0, 0, 0, 48]), (5, [12, 12, 12, 12])):
        X.copy_(H.normal((48, 512), torch.bfloat16, seed))
        offsets.copy_(H.offsets_of(counts))
        graph.replay()
        assert torch.equal(C, layer())


def test_refusals(ctx):
    A, As = ctx.fp8_quantize_rows(H.normal((8, 256), torch.bfloat16, 1))
    B, Bs = ctx.fp8_quantize_blocks(H.normal((256, 128), torch.bfloat16, 2))
    offsets = H.offsets_of([8])

    def refused(call):
        with pytest.raises(SparseWaveError) as e:
            call()
        assert e.value.status == _lib.SWB_ERR_INVALID_SHAPE

    refused(lambda: ctx.fp8_mm(A, As.t().contiguous(), B, Bs))
    refused(lambda: ctx.fp8_mm(A, As, B, Bs, transpose_b=True))
    refused(lambda: ctx.fp8_mm(A, As, B[None], Bs[None]))
    refused(lambda: ctx.fp8_mm(A, As, B, Bs[:1]))
    refused(lambda: ctx.fp8_grouped_mm(offsets, A, As, B, Bs))
    refused(lambda: ctx.fp8_grouped_mm(H.offsets_of([4, 4]), A, As, B[None], Bs[None]))
    refused(lambda: ctx.fp8_quantize_rows(torch.zeros((2, 3, 4), device="cuda")))
    refused(lambda: ctx.fp8_quantize_blocks(torch.zeros(4, device="cuda")))
    for call in (lambda: ctx.fp8_mm(A.float(), As, B, Bs), lambda: ctx.fp8_mm(A, As.half(), B, Bs),
                 lambda: ctx.fp8_mm(A, As, B.t(), Bs.t().contiguous(), transpose_b=True), lambda: ctx.fp8_mm(A.cpu(), As, B, Bs),
                 lambda: ctx.fp8_mm(A, As, B, Bs, torch.empty((8, 128), device="cuda")),
                 lambda: ctx.fp8_grouped_mm(None, A, As, B[None], Bs[None]), lambda: ctx.fp8_quantize_rows(A),
                 lambda: ctx.fp8_quantize_rows(torch.zeros((4, 4), device="cuda"), dtype=torch.float16),
                 lambda: ctx.fp8_quantize_rows(torch.zeros((4, 4), dtype=torch.float64, device="cuda"))):
        with pytest.raises(TypeError):
            call()
