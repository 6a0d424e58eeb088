"""Plain 64-bit forms of the products grouped by expert and of the 8-bit operands, with the error bounds that the tests hold the
kernels to."""
import torch

BLOCK = 128
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}


def offsets_of(counts, first=0):
    ends = torch.cumsum(torch.tensor([first] + list(counts)), 0)
    return ends.to(torch.int32).cuda()


def spans(offsets):
    o = offsets.tolist()
    return [(g, lo, hi) for g, (lo, hi) in enumerate(zip(o, o[1:]))]


def normal(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def assert_rounded_sum(got, exact, size, terms):
    """`got` is an f32 sum of `terms` products rounded once to got.dtype.

    The rounding: half a step, eps / 2 of the value (below the smallest normal of it).  The sum: `size` is the sum of the
    products' absolute values; each of the at most terms / 16 + 16 sums that a product passes through (16 products or more
    at a time, then the blocks of an axis that is split) loses less than 2^-22 of `size`: a step of f32 where the tensor core cuts
    off, and as much for the alignment of its products."""
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal
    bound = eps / 2 * exact.abs().clamp_min(tiny) + (terms / 16 + 16) * 2.0 ** -22 * size * (1 + eps)
    err = (got.double() - exact).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} outside; worst {float((err / bound.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} "
                                 f"times the bound; first at {bad.nonzero()[0].tolist()}: {float(got[tuple(bad.nonzero()[0])])} "
                                 f"for {float(exact[tuple(bad.nonzero()[0])])}")


def grouped_mm(offsets, A, B, transpose_b):
    """(C, sum of |products|) in 64 bits; rows of no group are NaN."""
    n = B.shape[1] if transpose_b else B.shape[2]
    C = torch.full((A.shape[0], n), float("nan"), dtype=torch.float64, device="cuda")
    size = C.clone()
    for g, lo, hi in spans(offsets):
        b = B[g].double().t() if transpose_b else B[g].double()
        C[lo:hi] = A[lo:hi].double() @ b
        size[lo:hi] = A[lo:hi].double().abs() @ b.abs()
    return C, size


def weight_gradient(offsets, A, dC, transpose_b, like):
    exact = torch.zeros(like.shape, dtype=torch.float64, device="cuda")
    size = exact.clone()
    for g, lo, hi in spans(offsets):
        left, right = (dC, A) if transpose_b else (A, dC)
        exact[g] = left[lo:hi].double().t() @ right[lo:hi].double()
        size[g] = left[lo:hi].double().abs().t() @ right[lo:hi].double().abs()
    return exact, size


def spread_rows(scales, inner):
    """(column blocks, rows) -> (rows, inner)"""
    return scales.t().repeat_interleave(BLOCK, 1)[:, :inner]


def spread_blocks(scales, rows, cols):
    return scales.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def scale_of(amax, dtype):
    """amax / largest rounded to f32, at least 2^-126 (torch divides by a number through its rounded reciprocal: a tensor)."""
    return (amax / torch.full_like(amax, LARGEST[dtype])).clamp_min(2.0 ** -126)


def quantize_rows(X, dtype=torch.float8_e4m3fn):
    """The definition in f32 on the GPU, by other steps than the kernels': bit for bit what they give."""
    x = torch.nn.functional.pad(X.float(), (0, -X.shape[1] % BLOCK))
    amax = x.abs().view(X.shape[0], -1, BLOCK).amax(2)
    scales = scale_of(amax, dtype).t().contiguous()
    return (X.float() * spread_rows(1.0 / scales, X.shape[1])).to(dtype), scales


def quantize_blocks(X, dtype=torch.float8_e4m3fn):
    stack = X if X.dim() == 3 else X[None]
    g, r, c = stack.shape
    x = torch.nn.functional.pad(stack.float(), (0, -c % BLOCK, 0, -r % BLOCK))
    amax = x.abs().view(g, x.shape[1] // BLOCK, BLOCK, -1, BLOCK).amax((2, 4))
    scales = scale_of(amax, dtype)
    q = (stack.float() * spread_blocks(1.0 / scales, r, c)).to(dtype)
    return (q, scales) if X.dim() == 3 else (q[0], scales[0])


def fp8_grouped_mm(offsets, A, a_scales, B, b_scales, transpose_b):
    """(C, size) in 64 bits of the 8-bit product; offsets None: one group and B a matrix."""
    if offsets is None:
        offsets, B, b_scales = offsets_of([A.shape[0]]), B[None], b_scales[None]
    a = A.double() * spread_rows(a_scales, A.shape[1]).double()
    b = B.double() * spread_blocks(b_scales, *B.shape[1:]).double()
    return grouped_mm(offsets, a, b, transpose_b)
