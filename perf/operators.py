"""Cases of the operators on matrices grouped by expert and on 8-bit operands with block scales, with their plain forms.

A case is a dict of plain values.  `prepare` makes what a program has in hand before the call, `run` is one pass through
an operator: with `own` false in elementary torch operations in 32 bits, with `own` true through the library's public
Python API.  `work` states the bytes and operations that a pass cannot do without, `exact` is the result in 64 bits.
"""
import functools
import math

import numpy as np
import torch

own = False

BLOCK = 128            # columns (rows) that share a scale
FP8_MAX = 448.0        # largest e4m3 value
SMALLEST_SCALE = 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}
MOST_FLOPS = 2.3e12
MOST_BYTES = 1.5e9


def listed():
    return [
        # One token routed to 8 of 64 experts, weights stored [out, in]: the up projection of a decoding step.
        dict(name="grouped_token", op="grouped", dtype="bf16", rows=8, groups=64, k=2048, n=1536, transpose_b=True, spread="single"),
        # 64 requests decoding together, 8 experts each: few ragged rows per expert, bound by reading the weights.
        dict(name="grouped_decode", op="grouped", dtype="bf16", rows=512, groups=64, k=2048, n=1536, transpose_b=True, spread="zipf"),
        # A prompt chunk over 64 experts, fp16, weights stored [in, out]: 256 rows per expert on average, ragged.
        dict(name="grouped_prefill", op="grouped", dtype="fp16", rows=16384, groups=64, k=2048, n=1536, transpose_b=False, spread="zipf"),
        # Eight large experts on a training batch: the largest product.
        dict(name="grouped_large", op="grouped", dtype="bf16", rows=32768, groups=8, k=4096, n=8192, transpose_b=True, spread="even"),
        # Sizes that no copy of 16 bytes divides, experts without rows.
        dict(name="grouped_odd", op="grouped", dtype="bf16", rows=3001, groups=7, k=1111, n=777, transpose_b=False, spread="gaps"),
        # The backward pass of a training step over 32 experts.
        dict(name="grad_train", op="grad", dtype="bf16", rows=16384, groups=32, k=2048, n=1536, transpose_b=True, spread="zipf"),
        # A small ragged backward pass in fp16, experts without rows (whose weight gradient is zero).
        dict(name="grad_ragged", op="grad", dtype="fp16", rows=1999, groups=12, k=1032, n=520, transpose_b=False, spread="gaps"),
        # Activations of a prompt to 8 bits, a scale per row and 128 columns.
        dict(name="quantize_rows", op="quantize_rows", dtype="bf16", rows=16384, k=4096),
        # Master weights of 8 experts to 8 bits, a scale per 128 x 128 block, odd edges.
        dict(name="quantize_weights", op="quantize_blocks", dtype="f32", groups=8, k=4100, n=1990),
        # A dense 8-bit layer while 16 requests decode.
        dict(name="fp8_decode", op="fp8", rows=16, groups=0, k=4096, n=8192, transpose_b=True, spread="even"),
        # A dense 8-bit layer on a training batch.
        dict(name="fp8_large", op="fp8", rows=8192, groups=0, k=8192, n=8192, transpose_b=True, spread="even"),
        # 8-bit experts on a prompt chunk, weights read as in the gradient of the rows (stored [in, out]).
        dict(name="fp8_grouped", op="fp8", rows=16384, groups=32, k=2048, n=2304, transpose_b=False, spread="zipf"),
    ]


def _log_size(rng, low, high, step=1):
    return max(step, int(round(math.exp(rng.uniform(math.log(low), math.log(high))) / step)) * step)


def draw(rng):
    """Sizes over the range of the listed cases, mostly multiples of 16 as layers have them, odd ones among them."""
    while True:
        op = rng.choice(["grouped", "grouped", "grouped", "grad", "grad", "quantize_rows", "quantize_blocks", "fp8", "fp8", "fp8"])
        step = rng.choice([128, 64, 16, 16, 8, 1])
        case = dict(op=op, k=_log_size(rng, 64, 8192, step), n=_log_size(rng, 64, 8192, step))
        if op == "quantize_blocks":
            case.update(dtype=rng.choice(["bf16", "f32"]), groups=_log_size(rng, 1, 32))
        elif op == "quantize_rows":
            del case["n"]
            case.update(dtype=rng.choice(["bf16", "fp16"]), rows=_log_size(rng, 1, 32768))
        else:
            case.update(rows=_log_size(rng, 1, 32768), groups=_log_size(rng, 1, 128), transpose_b=rng.random() < 0.5,
                        spread=rng.choice(["even", "zipf", "gaps", "single"]))
            if op == "fp8":
                case["groups"] = rng.choice([0, case["groups"]])
            else:
                case["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
        cost = work(case)
        stored = max(1, case.get("groups", 1)) * case["k"] * case.get("n", 1) * 2
        if 2e6 <= cost["bytes"] and cost["flops"] <= MOST_FLOPS and max(cost["bytes"], stored) <= MOST_BYTES:
            return case


def _bounds(case, seed):
    """First row of each group, and the row count: rows dealt to the groups as a router deals them."""
    rows, groups = case["rows"], case["groups"]
    if groups == 0:
        return [0, rows]
    rng = np.random.default_rng([seed, 17])
    if case["spread"] == "even":
        weights = np.ones(groups)
    elif case["spread"] == "zipf":  # some experts are asked far more often
        weights = rng.permutation(1.0 / np.arange(1, groups + 1) ** 0.7)
    elif case["spread"] == "gaps":  # a third of the experts gets nothing
        weights = np.where(rng.permutation(groups) < groups // 3, 0.0, rng.uniform(0.2, 1.0, groups))
    else:  # single: a row for each of `rows` experts, or as many for each
        weights = None
    if weights is None:
        counts = np.full(groups, rows // groups)
        counts[rng.permutation(groups)[:rows % groups]] += 1
    else:
        counts = rng.multinomial(rows, weights / weights.sum())
    return [0] + np.cumsum(counts).tolist()


@functools.lru_cache(maxsize=None)
def _context():
    from sparsewave_b200 import Context
    return Context(0)


def _operand(generator, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _weights(generator, case, dtype):
    """Experts' weights of the size that keeps a layer's outputs near one, one expert at a time."""
    shape = (case["n"], case["k"]) if case["transpose_b"] else (case["k"], case["n"])
    out = torch.empty((max(1, case["groups"]),) + shape, device="cuda", dtype=dtype)
    for g in range(out.shape[0]):
        out[g] = _operand(generator, shape, dtype, case["k"] ** -0.5)
    return out


def _row_scales(x):
    """amax / 448 of 128 columns of a row: (column blocks, rows) in f32."""
    rows, k = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, -k % BLOCK))
    amax = padded.abs().view(rows, -1, BLOCK).amax(2)
    return (amax / FP8_MAX).clamp_min(SMALLEST_SCALE).t().contiguous()


def _quantize_rows(x):
    scales = _row_scales(x)
    spread = scales.t().repeat_interleave(BLOCK, 1)[:, :x.shape[1]]
    return (x.float() / spread).to(torch.float8_e4m3fn), scales


def _spread_blocks(scales, rows, cols):
    return scales.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _quantize_block_matrix(w):
    rows, cols = w.shape
    padded = torch.nn.functional.pad(w.float(), (0, -cols % BLOCK, 0, -rows % BLOCK))
    amax = padded.abs().view(padded.shape[0] // BLOCK, BLOCK, -1, BLOCK).amax((1, 3))
    scales = (amax / FP8_MAX).clamp_min(SMALLEST_SCALE)
    return (w.float() / _spread_blocks(scales, rows, cols)).to(torch.float8_e4m3fn), scales


def _quantize_blocks(w):
    q, scales = torch.empty(w.shape, device=w.device, dtype=torch.float8_e4m3fn), []
    for g in range(w.shape[0]):
        values, s = _quantize_block_matrix(w[g])
        q[g].view(torch.uint8).copy_(values.view(torch.uint8))
        scales.append(s)
    return q, torch.stack(scales)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    op = case["op"]
    if op == "quantize_rows":  # activations: columns of different size, a few rows that stand out
        x = _operand(generator, (case["rows"], case["k"]), torch.float32)
        x *= torch.exp(torch.randn(case["k"], generator=generator, device="cuda"))
        x *= torch.exp(torch.randn((case["rows"], 1), generator=generator, device="cuda"))
        s["x"] = x.to(DTYPES[case["dtype"]])
    elif op == "quantize_blocks":
        s["w"] = _operand(generator, (case["groups"], case["n"], case["k"]), DTYPES[case["dtype"]], case["k"] ** -0.5)
    else:
        bounds = _bounds(case, seed)
        s["bounds"] = bounds
        s["offsets"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        if op == "fp8":
            s["a"], s["a_scales"] = _quantize_rows(_operand(generator, (case["rows"], case["k"]), torch.bfloat16))
            s["b"], s["b_scales"] = _quantize_blocks(_weights(generator, case, torch.bfloat16))
        else:
            dtype = DTYPES[case["dtype"]]
            s["a"] = _operand(generator, (case["rows"], case["k"]), dtype)
            s["b"] = _weights(generator, case, dtype)
            if op == "grad":
                s["dc"] = _operand(generator, (case["rows"], case["n"]), dtype)
    if own:
        s["ctx"] = _context()
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    case, ctx = s["case"], s["ctx"]
    op = case["op"]
    if op == "grouped":
        return ctx.grouped_mm(s["offsets"], s["a"], s["b"], transpose_b=case["transpose_b"])
    if op == "grad":
        return ctx.grouped_mm_grad(s["offsets"], s["a"], s["b"], s["dc"], transpose_b=case["transpose_b"])
    if op == "quantize_rows":
        return ctx.fp8_quantize_rows(s["x"])
    if op == "quantize_blocks":
        return ctx.fp8_quantize_blocks(s["w"])
    if case["groups"] == 0:
        return ctx.fp8_mm(s["a"], s["a_scales"], s["b"][0], s["b_scales"][0], transpose_b=case["transpose_b"])
    return ctx.fp8_grouped_mm(s["offsets"], s["a"], s["a_scales"], s["b"], s["b_scales"], transpose_b=case["transpose_b"])


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "quantize_rows":
        return _quantize_rows(s["x"])
    if op == "quantize_blocks":
        return _quantize_blocks(s["w"])
    a, b, bounds = s["a"], s["b"], s["bounds"]
    spans = [(g, lo, hi) for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])) if hi > lo]
    if op == "fp8":
        c = torch.empty((case["rows"], case["n"]), device=a.device, dtype=torch.bfloat16)
        for g, lo, hi in spans:
            left = a[lo:hi].float() * s["a_scales"][:, lo:hi].t().repeat_interleave(BLOCK, 1)[:, :case["k"]]
            right = b[g].float() * _spread_blocks(s["b_scales"][g], *b[g].shape)
            c[lo:hi] = left @ (right.t() if case["transpose_b"] else right)
        return c
    if op == "grouped":
        c = torch.empty((case["rows"], case["n"]), device=a.device, dtype=a.dtype)
        for g, lo, hi in spans:
            right = b[g].float()
            c[lo:hi] = a[lo:hi].float() @ (right.t() if case["transpose_b"] else right)
        return c
    dc = s["dc"]
    da, db = torch.empty_like(a), torch.zeros_like(b)
    for g, lo, hi in spans:
        left, up, right = a[lo:hi].float(), dc[lo:hi].float(), b[g].float()
        da[lo:hi] = up @ (right if case["transpose_b"] else right.t())
        db[g] = up.t() @ left if case["transpose_b"] else left.t() @ up
    return da, db


def _active(case):
    """Groups that have rows: the expected number of a draw of `rows` rows."""
    rows, groups = case["rows"], case["groups"]
    if groups == 0:
        return 1
    if case["spread"] == "single":
        return min(groups, rows)
    if case["spread"] == "zipf":
        share = 1.0 / np.arange(1, groups + 1) ** 0.7
    else:
        share = np.ones(groups - groups // 3 if case["spread"] == "gaps" else groups)
    return int(round(float((1.0 - (1.0 - share / share.sum()) ** rows).sum())))


def work(case):
    op, k, n = case["op"], case["k"], case.get("n", 0)
    blocks = -(-k // BLOCK)
    if op == "quantize_rows":
        elements = case["rows"] * k
        return {"bytes": elements * (DTYPES[case["dtype"]].itemsize + 1) + 4 * blocks * case["rows"], "flops": 3 * elements}
    if op == "quantize_blocks":
        elements = case["groups"] * k * n
        return {"bytes": elements * (DTYPES[case["dtype"]].itemsize + 1) + 4 * case["groups"] * blocks * -(-n // BLOCK),
                "flops": 3 * elements}
    rows, weights = case["rows"], _active(case) * k * n
    if op == "fp8":
        return {"bytes": rows * k + weights + 2 * rows * n + 4 * rows * blocks + 4 * weights // BLOCK ** 2,
                "flops": 2 * rows * k * n}
    if op == "grouped":
        return {"bytes": 2 * (rows * k + weights + rows * n), "flops": 2 * rows * k * n}
    return {"bytes": 2 * (2 * rows * k + rows * n + weights + case["groups"] * k * n), "flops": 4 * rows * k * n}


def _grid(x):
    """The e4m3 values nearest to f64 values of up to 448, ties to even: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return (torch.round(x / step) * step).clamp(-FP8_MAX, FP8_MAX)


def _exact_blocks(x, high, wide):
    """Scales and 8-bit values of blocks of high x wide elements of one matrix, block by block columns at a time."""
    x = x.double()
    rows, cols = x.shape
    values, scales = torch.empty_like(x), []
    for at in range(0, cols, wide):
        part = x[:, at:at + wide]
        amax = part.abs().amax(1)
        if high > 1:
            amax = torch.stack([piece.max() for piece in amax.split(high)])
        scale = torch.maximum(amax / FP8_MAX, torch.full_like(amax, SMALLEST_SCALE))
        scales.append(scale)
        values[:, at:at + wide] = _grid(part / scale.repeat_interleave(high)[:rows, None])
    return values, torch.stack(scales)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize_rows":
        return _exact_blocks(s["x"], 1, BLOCK)
    if op == "quantize_blocks":
        parts = [_exact_blocks(w, BLOCK, BLOCK) for w in s["w"]]
        return torch.stack([values for values, _ in parts]), torch.stack([scales.t() for _, scales in parts])
    a = s["a"].double()
    layout = "rk,nk->rn" if case["transpose_b"] else "rk,kn->rn"
    if op == "fp8":
        for block in range(s["a_scales"].shape[0]):
            a[:, block * BLOCK:(block + 1) * BLOCK] *= s["a_scales"][block].double()[:, None]
    first = torch.zeros((case["rows"], case["n"]), device="cuda", dtype=torch.float64)
    da = torch.zeros_like(a) if op == "grad" else None
    db = torch.zeros(s["b"].shape, device="cuda", dtype=torch.float64) if op == "grad" else None
    for g in range(len(s["bounds"]) - 1):
        rows = slice(s["bounds"][g], s["bounds"][g + 1])
        b = s["b"][g].double()
        if op == "fp8":
            for i, line in enumerate(s["b_scales"][g].double().tolist()):
                for j, scale in enumerate(line):
                    b[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scale
        if op == "grad":
            dc = s["dc"][rows].double()
            da[rows] = torch.einsum("rn,nk->rk" if case["transpose_b"] else "rn,kn->rk", dc, b)
            db[g] = torch.einsum("rn,rk->nk" if case["transpose_b"] else "rn,rk->kn", dc, a[rows])
        else:
            first[rows] = torch.einsum(layout, a[rows], b)
    return (da, db) if op == "grad" else first
