"""Weight gradients of few long groups, whose rows are shared among parts in memory of the context's pool: captured, on several streams,
off a boundary, with groups shorter than a part and with offsets that decrease."""
import pytest
import torch

from tests import grouped_helpers as H

pytestmark = pytest.mark.gpu


def operands(rows, k, n, groups, transpose_b, dtype=torch.bfloat16, seed=1):
    A, dC = H.normal((rows, k), dtype, seed), H.normal((rows, n), dtype, seed + 1)
    return A, torch.empty((groups, n, k) if transpose_b else (groups, k, n), dtype=dtype, device="cuda"), dC


def check(dB, offsets, A, dC, transpose_b, rows):
    exact, size = H.weight_gradient(offsets, A, dC, transpose_b, dB)
    H.assert_rounded_sum(dB, exact, size, rows)


def launches(ctx, call):
    before = ctx.kernel_launches
    call()
    return ctx.kernel_launches - before


@pytest.mark.parametrize("k,n,transpose_b", [(128, 264, False), (264, 128, True), (41, 30, False)])
@pytest.mark.parametrize("groups", [1, 2])
def test_captured_with_other_group_sizes(ctx, k, n, transpose_b, groups):
    rows = 5000
    A, B, dC = operands(rows, k, n, groups, transpose_b)
    offsets = H.offsets_of([rows] if groups == 1 else [rows // 2, rows - rows // 2])
    dB = torch.full_like(B, 7.0)
    call = lambda out: ctx.grouped_mm_grad(offsets, A, B, dC, None, out, transpose_b=transpose_b, need_dA=False)
    copies = k % 8 != 0 or n % 8 != 0
    assert launches(ctx, lambda: call(dB)) == 2 + copies  # the parts and their sum
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(dB)
    for counts in ([[rows], [0], [1], [77], [4999]] if groups == 1 else [[0, rows], [rows, 0], [3, 4000], [2500, 63], [0, 0], [64, 1]]):
        offsets.copy_(H.offsets_of(counts, 0))
        A.copy_(H.normal((rows, k), torch.bfloat16, 10 + counts[0]))
        dB.fill_(7.0)
        graph.replay()
        eager = torch.full_like(B, 9.0)
        call(eager)
        assert torch.equal(dB, eager)
        check(dB, offsets, A, dC, transpose_b, rows)
    assert ctx.device_status() == 0


def test_streams_at_a_time(ctx):
    shapes = [(5000, 128, 264, 1), (7001, 41, 30, 2), (6000, 136, 72, 2)]
    layers = []
    for i, (rows, k, n, groups) in enumerate(shapes):
        A, B, dC = operands(rows, k, n, groups, False, seed=3 * i)
        offsets = H.offsets_of([rows // groups] * (groups - 1) + [rows - rows // groups * (groups - 1)])
        layers.append((offsets, A, B, dC, ctx.grouped_mm_grad(offsets, A, B, dC, need_dA=False)[1]))
        check(layers[-1][4], offsets, A, dC, False, rows)
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    results = []
    for turn in range(30):
        for i in range(len(layers)):
            offsets, A, B, dC, want = layers[(i + turn) % len(layers)]
            with torch.cuda.stream(streams[i]):
                results.append((ctx.grouped_mm_grad(offsets, A, B, dC, need_dA=False)[1], want))
    torch.cuda.synchronize()
    assert all(torch.equal(got, want) for got, want in results)


def test_two_graphs_at_a_time(ctx):
    layers = []
    for seed in range(2):
        A, B, dC = operands(5000 + seed, 128, 136, 1, False, seed=seed)
        offsets, dB = H.offsets_of([5000 + seed]), torch.empty_like(B)
        call = lambda: ctx.grouped_mm_grad(offsets, A, B, dC, None, dB, need_dA=False)
        call()
        want = dB.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        layers.append((A, dC, offsets, dB, graph, want))
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(20):
        for (*_, dB, graph, _), stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                dB.fill_(7.0)
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(dB, want) for *_, dB, _, want in layers)


@pytest.mark.parametrize("shift", [1, 2, 4, 8])
@pytest.mark.parametrize("k,n", [(128, 136), (33, 50)])
def test_results_off_a_boundary(ctx, shift, k, n):
    rows = 5000
    A, B, dC = operands(rows, k, n, 2, True)
    offsets = H.offsets_of([3000, 2000])
    flat = torch.full((B.numel() + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
    dB = flat[shift:shift + B.numel()].view(B.shape)
    assert launches(ctx, lambda: ctx.grouped_mm_grad(offsets, A, B, dC, None, dB, transpose_b=True, need_dA=False)) >= 2
    check(dB, offsets, A, dC, True, rows)
    assert torch.equal(dB, ctx.grouped_mm_grad(offsets, A, B, dC, transpose_b=True, need_dA=False)[1])
    assert bool((flat[:shift] == 7.0).all()) and bool((flat[shift + B.numel():] == 7.0).all())


@pytest.mark.parametrize("wrong", [[5000, 0], [0, 5000, 10], [4000, 5000, 4999]])
def test_offsets_that_decrease_make_zeros(ctx, wrong):
    A, B, dC = operands(5000, 128, 136, len(wrong) - 1, False)
    offsets, dB = torch.tensor(wrong, dtype=torch.int32, device="cuda"), torch.full_like(B, 7.0)
    assert launches(ctx, lambda: ctx.grouped_mm_grad(offsets, A, B, dC, None, dB, need_dA=False)) == 2
    assert bool((dB == 0).all()) and ctx.device_status() == 0


def test_offsets_outside_the_rows_are_clipped(ctx):
    A, B, dC = operands(5000, 128, 136, 2, False)
    offsets = torch.tensor([-70, 4000, 10 ** 9], dtype=torch.int32, device="cuda")
    _, dB = ctx.grouped_mm_grad(offsets, A, B, dC, need_dA=False)
    check(dB, H.offsets_of([4000, 1000]), A, dC, False, 5000)
