"""Matrices in microscaled 4-bit floating point on the GPU: quantisation against the definition in 64 bits, products against
64-bit sums of the same values."""
import math

import pytest
import torch

from mini_rsglang_b200 import kernels
from mini_rsglang_b200.errors import InvalidRequest

pytestmark = pytest.mark.gpu
DEV = "cuda"
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def block_exponent(largest):
    """floor(log2) - 2 of 64-bit sizes, from their exponents; blocks of zeros as the smallest."""
    field = (largest.double().view(torch.int64) >> 52) - 1023 - 2
    return field.clamp(-127, 125)


def power_of_two(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def plain_quantise(x):
    """(values float64, scale bytes) of rows by the definition."""
    rows, width = x.shape
    blocks = x.double().view(rows, width // 32, 32)
    finite = blocks.isfinite().all(dim=2, keepdim=True)
    safe = torch.where(finite, blocks, torch.zeros_like(blocks))
    e = block_exponent(safe.abs().amax(dim=2, keepdim=True))
    power = power_of_two(e)
    size = (safe / power).abs()
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    best = torch.zeros_like(size)
    for i in range(1, 8):
        middle = (grid[i - 1] + grid[i]) / 2
        best = torch.where((size > middle) | ((size == middle) & (i % 2 == 0)), grid[i], best)
    value = best * torch.sign(safe) * power
    value = torch.where(finite, value, torch.full_like(value, math.nan))
    byte = torch.where(finite, e + 127, torch.full_like(e, 255))
    return value.view(rows, width), byte.view(rows, width // 32).to(torch.uint8)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(0, 64), (1, 32), (1, 4096), (3, 96), (5, 160), (127, 288), (129, 224), (300, 1056)])
def test_quantise_is_the_definition(dtype, rows, width):
    g = torch.Generator(device=DEV).manual_seed(rows * 5 + width)
    x = torch.randn(rows, width, device=DEV, generator=g) * torch.exp2(torch.randint(-40, 40, (rows, width), device=DEV, generator=g) / 4)
    x = x.to(dtype)
    q = kernels.mxfp4_quantise(x)
    values, bytes_ = plain_quantise(x) if rows else (torch.empty(0, width, dtype=torch.float64, device=DEV), torch.empty(0, width // 32, dtype=torch.uint8, device=DEV))
    assert q.shape == (rows, width)
    assert torch.equal(q.block_scales(), bytes_)
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(kernels.mxfp4_dequantise(q, out).double(), values)


def test_quantise_of_ties_ends_of_the_range_and_what_is_not_finite():
    """Every tie, both signs, in blocks of every power of two; zeros; the smallest and largest floats; infinities and NaN."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 4.0, 0.2490234375, 0.251953125, 0.0, 2.484375, 5.03125])
    block = torch.cat([ties, -ties])
    x = block[None, :].double() * power_of_two(torch.arange(-126, 125))[:, None]
    x = torch.cat([x, torch.zeros(1, 32), torch.full((1, 32), -0.0), torch.full((1, 32), 2.0 ** -149), torch.full((1, 32), 1e-39),
                   torch.full((1, 32), 3.3e38)]).float().to(DEV)
    bad = torch.randn(4, 32, device=DEV)
    bad[0, 3], bad[1, 31], bad[2, 0], bad[3, 7] = math.inf, math.nan, -math.inf, 3.4028234663852886e38
    x = torch.cat([x, bad]).contiguous()
    values, bytes_ = plain_quantise(x)
    q = kernels.mxfp4_quantise(x)
    assert torch.equal(q.block_scales(), bytes_)
    assert same(kernels.mxfp4_dequantise(q, torch.float32).double(), values)
    assert same(kernels.mxfp4_dequantise(q, torch.bfloat16).double(), values)
    # two blocks of a row: what is not finite stays in its own
    wide = torch.cat([bad, bad.flip(1).nan_to_num(1.0, 1.0, 1.0)], dim=1).contiguous()
    values, bytes_ = plain_quantise(wide)
    q = kernels.mxfp4_quantise(wide)
    assert torch.equal(q.block_scales(), bytes_) and same(kernels.mxfp4_dequantise(q, torch.float32).double(), values)


def random_matrix(g, n, k, spread=3):
    """A matrix of every code with scales of different sizes, its 64-bit values, and its plain layout."""
    codes = torch.randint(0, 256, (n, k // 2), device=DEV, generator=g, dtype=torch.uint8)
    scales = torch.randint(127 - spread - 5, 127 + spread - 5, (n, k // 32), device=DEV, generator=g, dtype=torch.uint8)
    return codes, scales, plain_values(codes, scales)


def plain_values(codes, scales):
    n, k = codes.shape[0], codes.shape[1] * 2
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device=codes.device)
    value = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], dim=2).view(n, k // 32, 32)
    power = power_of_two(scales.long() - 127).view(n, k // 32, 1)
    power = torch.where(scales.view(n, k // 32, 1) == 255, torch.full_like(power, math.nan), power)
    return (value * power).view(n, k)


def close_to_sums(out, want, size, k, what):
    """Products of a bfloat16 and a 4-bit value are exact in float32.  The tensor cores add 16 (32 or 64 with 4 bits on both sides) of
    them to a sum at a time; an addition that cuts off instead of rounding loses up to 2^-23 of the sum of sizes so far, and joining
    blocks, ranges and pieces is float32 additions of 2^-24 each: k / 16 + 16 times 2^-23 covers both.  bfloat16 results are rounded
    once more, by 2^-9 of their power of two or less: 2^-8 of themselves."""
    limit = size * (k / 16 + 16) * 2.0 ** -23
    if out.dtype is torch.bfloat16:
        limit = limit + (want.abs() + limit) * 2.0 ** -8
    off = (out.double() - want).abs()
    assert (off <= limit + 1e-45).all(), f"{what}: {(off / (limit + 1e-45)).max().item():.3f} of the limit"


@pytest.mark.parametrize("quantise", [False, True])
@pytest.mark.parametrize("m", [0, 1, 2, 7, 8, 9, 15, 16, 17, 33, 64, 100, 129, 257])
@pytest.mark.parametrize("n,k", [(1, 32), (16, 64), (129, 96), (40, 4096), (300, 1056), (257, 2336), (1000, 512)])
def test_product_over_the_sizes(m, n, k, quantise):
    g = torch.Generator(device=DEV).manual_seed(m * 131 + n + k)
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    values = plain_quantise(x)[0] if quantise and m else x.double()
    want, size = values @ w.T, values.abs() @ w.abs().T
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), float("nan"), device=DEV, dtype=dtype)
        kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
        close_to_sums(out, want, size, k, f"{m} x {n} x {k}")


PLANS = [("few", 1), ("few", 2), ("few", 8), ("many", 16, 5, False), ("many", 16, 7, True), ("many", 32, 1, False), ("many", 64, 3, True), ("many", 128, 148, False),
         ("many", 128, 148, True), ("many", 128, 11, True), ("many", 192, 148, False), ("many", 192, 9, True), ("parts", 16, 5, False), ("parts", 16, 9, True),
         ("parts", 32, 148, False), ("parts", 32, 7, True), ("parts", 64, 3, False), ("parts", 64, 148, True), ("parts", 16, 2, False), ("parts", 32, 1, False),
         ("parts", 64, 2, False)]


def takes(plan, m, k, quantise):
    """Whether a kernel takes these rows."""
    if plan[0] == "parts":
        return m <= plan[1] and k % 128 == 0 and not quantise
    return plan[0] == "few" or plan[1] >= 128 or m <= plan[1]


def fitting(plan, m, n, k):
    """The plan with no more CTAs than have work."""
    if plan[0] == "few":
        return plan
    tiles = -(-n // 128) * -(-m // plan[1])
    return (*plan[:2], min(plan[2], tiles * -(-k // 256) if plan[3] else tiles), plan[3])


SIZES = [(1, 128, 256), (13, 100, 32), (16, 129, 288), (30, 200, 1056), (64, 64, 4096), (100, 300, 544), (260, 513, 768), (257, 130, 2080), (600, 24000, 96),
         (400, 2500, 512), (9, 129, 128), (16, 500, 1152), (31, 1000, 4096), (32, 70, 640), (33, 300, 640), (50, 1000, 1152), (63, 129, 128),
         (24, 700, 1024), (11, 900, 1920), (60, 500, 384)]


@pytest.mark.parametrize("m,n,k,plan,quantise", [(m, n, k, plan, quantise) for m, n, k in SIZES for plan in PLANS for quantise in (False, True)
                                                 if takes(plan, m, k, quantise)])
def test_every_kernel_over_the_sizes(m, n, k, plan, quantise):
    g = torch.Generator(device=DEV).manual_seed(m * 31 + n * 7 + k)
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    values = plain_quantise(x)[0] if quantise else x.double()
    want, size = values @ w.T, values.abs() @ w.abs().T
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n), float("nan"), device=DEV, dtype=dtype)
        kernels.mxfp4_gemm(x, weight, out, quantise=quantise, plan=fitting(plan, m, n, k))
        torch.cuda.synchronize()
        kernels.check_device_errors(certain=True)
        close_to_sums(out, want, size, k, f"{m} x {n} x {k} {plan}")


SOME_PLANS = [("parts", 16, 2, False), ("parts", 64, 2, True), ("few", 1), ("few", 2), ("many", 64, 2, False), ("many", 128, 3, True), ("many", 192, 2, True)]


def check_product(x, weight, w, quantise, plan, what):
    """Against the 64-bit product of the values: not a number where that is none, infinities as they are, the rest within the bound."""
    values = plain_quantise(x)[0] if quantise else x.double()
    want = values @ w.T
    finite = want.isfinite()
    out = torch.full((x.shape[0], w.shape[0]), 7.0, device=DEV)
    kernels.mxfp4_gemm(x, weight, out, quantise=quantise, plan=plan)
    assert torch.equal(out.isnan(), want.isnan()), what
    assert torch.equal(out[want.isinf()], want[want.isinf()].float()), what
    size = values.abs().nan_to_num(0, 0, 0) @ w.abs().nan_to_num(0, 0, 0).T
    close_to_sums(out[finite], want[finite], size[finite], x.shape[1], what)


@pytest.mark.parametrize("plan,quantise", [(plan, q) for plan in SOME_PLANS for q in (False, True) if takes(plan, 11, 128, q)])
@pytest.mark.parametrize("kind", ["wide", "tiny", "huge", "zeros", "infinite", "one_row"])
def test_rows_that_halfs_do_not_hold(kind, plan, quantise):
    """Elements of very different sizes in a row and in neighbouring rows, the ends of bfloat16's range, rows of zeros, infinities
    and NaN beside ordinary rows: exact products whatever the range, and nothing of one row in another."""
    m, n, k = 11, 150, 768 if plan[0] == "parts" else 800
    g = torch.Generator(device=DEV).manual_seed(len(kind))
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g)
    if kind == "wide":
        x = x * torch.exp2(torch.randint(-50, 50, (m, k), device=DEV, generator=g).float())
    elif kind == "tiny":
        x = x * 2.0 ** -118
    elif kind == "huge":
        x = x * 2.0 ** 100
        x[3] *= 2.0 ** -180
    elif kind == "zeros":
        x[::2] = 0.0
        x[1, 5:] = 0.0
    elif kind == "infinite":
        x[2, 7], x[5, 300], x[8, k - 1] = math.inf, math.nan, -math.inf
    elif kind == "one_row":
        x[4, 10] = 1e30
        weight_column = (codes[:, 5] & 0xF0)                # column 10 of every row is 0: what is left of that row is its small elements
        codes = codes.clone()
        codes[:, 5] = weight_column
        weight, w = kernels.mxfp4_matrix(codes, scales), plain_values(codes, scales)
    check_product(x.bfloat16(), weight, w, quantise, plan, kind)


@pytest.mark.parametrize("plan", [("parts", 16, 2, False), ("parts", 32, 4, True), ("parts", 64, 1, False), ("parts", 64, 7, True), ("many", 16, 2, True), ("many", 32, 1, False),
                                  ("many", 64, 2, False), ("many", 128, 3, True), ("many", 192, 2, True), ("many", 192, 1, False)])
@pytest.mark.parametrize("count", [1, 8, 9, 200])
def test_elements_far_below_the_others(plan, count):
    """What stands beside much larger elements and is small enough for no form of x to hold both, `count` in 256: a few are added one
    by one, many make another kernel or another path of it.  The large ones meet codes of zero, so that the result is the small ones'."""
    m, n, k = 13, 150, 896
    g = torch.Generator(device=DEV).manual_seed(count)
    codes, scales, w = random_matrix(g, n, k)
    x = torch.zeros(m, k, device=DEV)
    codes = codes.clone()
    for start in range(0, k, 256):
        width = min(256, k - start)
        order = torch.randperm(width, device=DEV, generator=g)
        small, large = start + order[2:2 + min(count, width - 2)], start + order[:2]
        rows = torch.arange(m, device=DEV) % 3 != 1                      # every third row has none of them
        x[:, small] = rows[:, None] * torch.randn(m, small.numel(), device=DEV, generator=g) * 2.0 ** -40
        x[:, large] = torch.randn(m, 2, device=DEV, generator=g)
        for column in large.tolist():
            codes[:, column // 2] &= 0x0F if column % 2 else 0xF0
    x[:, -2:] = torch.tensor([1.0, 2.0 ** -40], device=DEV) * torch.randn(m, 2, device=DEV, generator=g)             # and the row's last two
    codes[:, -1] = 0x50
    w = plain_values(codes, scales)
    check_product(x.bfloat16(), kernels.mxfp4_matrix(codes, scales), w, False, plan, f"{count}")


@pytest.mark.parametrize("plan", [("parts", 64, 3, False), ("parts", 64, 5, True), ("many", 64, 2, False), ("many", 64, 5, True), ("many", 128, 3, False), ("many", 128, 7, True),
                                  ("many", 192, 5, True), ("many", 192, 4, False)])
@pytest.mark.parametrize("some", [1, 3, 7, 30])
def test_a_few_rows_with_elements_far_below(plan, some):
    """`some` rows among the others have up to eight such elements, which meet the only codes that are not zero."""
    m, n, k = 64 if plan[1] == 64 else 300, 390, 1280
    g = torch.Generator(device=DEV).manual_seed(some + plan[1])
    codes, scales, _ = random_matrix(g, n, k)
    x = torch.randn(m, k, device=DEV, generator=g)
    nonzero = torch.tensor([3, 255, 256, 700, 1024, 1100, 1200, 1279], device=DEV)
    keep = torch.zeros(k, dtype=torch.bool, device=DEV)
    keep[nonzero] = True
    mask = torch.where(keep[0::2], 0x0F, 0) | torch.where(keep[1::2], 0xF0, 0)
    codes = codes & mask.to(torch.uint8)
    rows = torch.randperm(m, device=DEV, generator=g)[:some]
    for i, row in enumerate(rows.tolist()):
        x[row, nonzero[:1 + i % 8]] *= 2.0 ** -50
        x[row, nonzero[1 + i % 8:]] = 0.0
    weight, w = kernels.mxfp4_matrix(codes, scales), plain_values(codes, scales)
    check_product(x.bfloat16(), weight, w, False, plan, f"{some}")


@pytest.mark.parametrize("plan,quantise", [(plan, q) for plan in SOME_PLANS for q in (False, True) if takes(plan, 11, 128, q)])
@pytest.mark.parametrize("kind", ["wide", "nan", "zero_blocks", "small", "large", "unsettled"])
def test_scales_of_every_size(kind, plan, quantise):
    m, n, k = 9, 260, 640 if plan[0] == "parts" else 544
    g = torch.Generator(device=DEV).manual_seed(len(kind) + 50)
    codes, scales, w = random_matrix(g, n, k)
    if kind == "wide":
        scales = torch.randint(60, 190, scales.shape, device=DEV, generator=g, dtype=torch.uint8)
    elif kind == "nan":
        scales[7, 3], scales[200, 16], scales[259, 0] = 255, 255, 255
    elif kind == "zero_blocks":
        codes = codes.view(n, k // 32, 16).clone()
        codes[::3, 1], codes[5], codes[6, 2] = 0, 0x88, 0x80
        scales[::3, 1], scales[5] = 250, 0
        codes = codes.view(n, k // 2)
    elif kind == "small":
        scales = torch.randint(2, 20, scales.shape, device=DEV, generator=g, dtype=torch.uint8)
    elif kind == "large":
        scales = torch.randint(200, 230, scales.shape, device=DEV, generator=g, dtype=torch.uint8)
    w = plain_values(codes, scales)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    if kind == "unsettled":
        weight = kernels.mxfp4_quantise(w.float())
        w = plain_quantise(w.float())[0]
        assert not weight.settled
    check_product(x, weight, w, quantise, plan, kind)
    if kind == "nan":
        assert torch.equal(weight.block_scales(), scales) and kernels.mxfp4_dequantise(weight).isnan().sum().item() == 96


@pytest.mark.parametrize("rows,width,low,high", [(5, 64, 100, 137), (200, 96, 100, 136), (3, 32, 255, 255)])
def test_settle_knows_what_halfs_hold(rows, width, low, high):
    codes = torch.full((rows, width // 2), 0x17, device=DEV, dtype=torch.uint8)
    scales = torch.full((rows, width // 32), low, device=DEV, dtype=torch.uint8)
    scales[-1, -1] = high
    weight = kernels.mxfp4_matrix(codes, scales)
    assert weight.settled and weight.half_exponent == (None if high == 255 or high - low > 36 else high - 140)


ALL_KINDS = [(3, False), (3, True), (12, False), (12, True), (60, False), (60, True), (200, False), (200, True)]


@pytest.mark.parametrize("m,quantise", ALL_KINDS)
def test_nothing_but_the_output_is_written(m, quantise):
    """Odd sizes inside a larger buffer: what stands before and behind the rows stays."""
    n, k = 333, 1152
    g = torch.Generator(device=DEV).manual_seed(m)
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    before = (x.clone(), weight.data.clone())
    for dtype in (torch.bfloat16, torch.float32):
        buffer = torch.full((m * n + 2 * n,), 7.0, device=DEV, dtype=dtype)
        kernels.mxfp4_gemm(x, weight, buffer[n:-n].view(m, n), quantise=quantise)
        assert (buffer[:n] == 7).all() and (buffer[-n:] == 7).all()
        values = plain_quantise(x)[0] if quantise else x.double()
        close_to_sums(buffer[n:-n].view(m, n), values @ w.T, values.abs() @ w.abs().T, k, "inside a buffer")
    assert torch.equal(x, before[0]) and torch.equal(weight.data, before[1])


@pytest.mark.parametrize("m,quantise", ALL_KINDS)
def test_an_output_over_the_input_is_refused(m, quantise):
    weight = kernels.mxfp4_quantise(torch.randn(256, 256, device=DEV)).settle()
    buffer = torch.zeros(3 * m * 256, device=DEV, dtype=torch.bfloat16)
    x = buffer[m * 256:2 * m * 256].view(m, 256)
    for out in (x, buffer[m * 256 - 2:2 * m * 256 - 2].view(m, 256), buffer[:2 * m * 256].view(torch.float32).view(m, 256)):
        with pytest.raises(InvalidRequest):
            kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
    kernels.mxfp4_gemm(x, weight, buffer[:m * 256].view(m, 256), quantise=quantise)
    kernels.mxfp4_gemm(x, weight, buffer[2 * m * 256:].view(m, 256), quantise=quantise)


@pytest.mark.parametrize("m,quantise", ALL_KINDS)
def test_the_same_bits_every_time(m, quantise):
    """Several CTAs add up a tile, in whatever order they end: a result depends on its inputs alone, on every stream."""
    n, k = 1100, 5120
    g = torch.Generator(device=DEV).manual_seed(m)
    weight = kernels.mxfp4_matrix(*random_matrix(g, n, k)[:2])
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    first = torch.empty(m, n, device=DEV)
    kernels.mxfp4_gemm(x, weight, first, quantise=quantise)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.empty_like(first) for _ in range(30)]
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 3]):                 # three at a time, each with its own workspace
            kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
    torch.cuda.synchronize()
    assert all(torch.equal(first, out) for out in outs)
    kernels.check_device_errors(certain=True)


@pytest.mark.parametrize("m,quantise", ALL_KINDS)
def test_recorded_and_replayed(m, quantise):
    """Two recordings with the same weights, replayed in turn and beside eager calls, with new inputs."""
    n, k = 700, 2304
    g = torch.Generator(device=DEV).manual_seed(m + 1)
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    xs = [torch.zeros(m, k, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    outs = [torch.empty(m, n, device=DEV) for _ in range(2)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for x, out in zip(xs, outs):
            kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
    torch.cuda.synchronize()
    graphs = []
    for x, out in zip(xs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
            if quantise:                                         # quantising and reading back in the same recording
                back = kernels.mxfp4_dequantise(kernels.mxfp4_quantise(x), torch.float32)
        graphs.append(graph)
    for _ in range(3):
        for x in xs:
            x.copy_(torch.randn(m, k, device=DEV, generator=g))
        eager = torch.empty(m, n, device=DEV)
        for graph in graphs:
            graph.replay()
        kernels.mxfp4_gemm(xs[0], weight, eager, quantise=quantise)
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            values = plain_quantise(x)[0] if quantise else x.double()
            close_to_sums(out, values @ w.T, values.abs() @ w.abs().T, k, "replayed")
        assert torch.equal(outs[0], eager)
        if quantise:
            assert torch.equal(back.double(), plain_quantise(xs[1])[0])


def test_offsets_beyond_32_bits():
    """Codes of more than 2^31 bytes, results of more than 2^31 elements: the last rows and columns."""
    n, k = 1_100_003, 4096
    g = torch.Generator(device=DEV).manual_seed(5)
    codes = torch.randint(0, 256, (n, k // 2), device=DEV, generator=g, dtype=torch.uint8)
    scales = torch.randint(118, 124, (n, k // 32), device=DEV, generator=g, dtype=torch.uint8)
    weight = kernels.mxfp4_matrix(codes, scales)
    places = torch.tensor([0, 524287, 524288, n - 130, n - 1], device=DEV)
    w = plain_values(codes[places], scales[places])
    del codes, scales
    for m, quantise in ((1, False), (2, True), (9, False), (9, True), (130, False), (140, True)):
        x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
        out = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
        kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
        values = plain_quantise(x)[0] if quantise else x.double()
        close_to_sums(out[:, places], values @ w.T, values.abs() @ w.abs().T, k, f"{m} rows")
    values = kernels.mxfp4_dequantise(weight)
    assert torch.equal(values[places].double(), w)
    again = kernels.mxfp4_quantise(values)
    assert torch.equal(kernels.mxfp4_dequantise(again)[places].double(), w)      # representable values stay
    del values, again, weight, out
    m, n, k = 20011, 120001, 32
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    rows = torch.tensor([0, 17895, 17896, m - 1], device=DEV)
    for quantise in (False, True):
        out = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
        kernels.mxfp4_gemm(x, weight, out, quantise=quantise)
        values = plain_quantise(x[rows])[0] if quantise else x[rows].double()
        close_to_sums(out[rows], values @ w.T, values.abs() @ w.abs().T, k, "many results")
        del out


def test_refusals_on_the_gpu():
    g = torch.Generator(device=DEV).manual_seed(1)
    codes, scales, _ = random_matrix(g, 40, 64)
    weight = kernels.mxfp4_matrix(codes, scales)
    x, out = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16), torch.zeros(4, 40, device=DEV)
    odd = torch.zeros(4 * 64 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(4, 64)
    for bad_x, bad_out in ((x.float(), out), (x.half(), out), (torch.zeros(64, 4, device=DEV, dtype=torch.bfloat16).t(), out), (odd, out), (x[:3], out),
                           (x, out.half()), (x, torch.zeros(4, 41, device=DEV)), (x, torch.zeros(40, 4, device=DEV).t()), (x[:, :32].contiguous(), out)):
        with pytest.raises(InvalidRequest):
            kernels.mxfp4_gemm(bad_x, weight, bad_out)
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_quantise(odd)
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_quantise(x.t())
    with pytest.raises(InvalidRequest, match="float32"):
        kernels.mxfp4_matrix(codes, torch.full_like(scales, 253))
    zeros = kernels.mxfp4_matrix(torch.zeros_like(codes), torch.full_like(scales, 254))         # blocks of zeros may have any scale
    kernels.mxfp4_gemm(x, zeros, out)
    assert (out == 0).all()


@pytest.mark.parametrize("quantise", [False, True])
@pytest.mark.parametrize("m,k", [(8, 11296), (8, 17376), (7, 12832), (7, 14816), (6, 15392), (6, 17376), (5, 18464), (4, 23104), (3, 30752), (1, 131104)])
def test_few_rows_too_long_for_two_ctas(m, k, quantise):
    """Rows that are no multiple of 128 elements and whose x only four CTAs' shared memory holds, as the plan launches them."""
    n = 333
    g = torch.Generator(device=DEV).manual_seed(m * 7 + k)
    codes, scales, w = random_matrix(g, n, k)
    check_product(torch.randn(m, k, device=DEV, generator=g).bfloat16(), kernels.mxfp4_matrix(codes, scales), w, quantise, None, f"{m} x {k}")


def close_to_small_sums(out, want, size, k, what):
    """As `close_to_sums`; beside that, below float32's ordinary numbers each of the k products and each addition of 16 of them, of blocks and
    of pieces is off by up to a step of 2^-149, which is all that float32 has there."""
    limit = (k / 16 + 16) * size * 2.0 ** -23 + (k + k / 16 + 16) * 2.0 ** -149
    off = (out.double() - want).abs()
    assert (off <= limit).all(), f"{what}: {(off / limit).max().item():.3f} of the limit"


def one_sign(x, codes, kind):
    return (x.abs(), codes & 0x77) if kind else (x, codes)


@pytest.mark.parametrize("plan,quantise", [(plan, q) for plan in SOME_PLANS + [("few", 8)] for q in (False, True) if takes(plan, 3, 768, q)])
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("kind,top,low,high", [("all", 127, 97, 113), ("all", 120, 97, 120), ("all", 123, 97, 117), ("one", 127, 100, 122)])
def test_large_rows_and_small_scales(kind, top, low, high, positive, plan, quantise):
    """Elements up to 2^(top + 1) in every column, or in one column of 768 beside ordinary ones, against scales of 2^(low - 127) to 2^(high - 127):
    no sum of sizes leaves float32's range (768 * 6 * 2^(top + 1 + high - 127) < 2^127 for all, 6 * 2^128 * 2^-5 and 768 ordinary products for one), and no
    product may on its way."""
    m, n, k = 3, 150, 768
    g = torch.Generator(device=DEV).manual_seed(top + high)
    codes, _, _ = random_matrix(g, n, k)
    scales = torch.randint(low, high + 1, (n, k // 32), device=DEV, generator=g, dtype=torch.uint8)
    x = torch.randn(m, k, device=DEV, generator=g)
    large = (1 + torch.rand(m, k, device=DEV, generator=g) * 0.984375) * torch.sign(x) * 2.0 ** (top - 60) * 2.0 ** 60       # below 2^(top + 1) as bfloat16 too
    columns = torch.arange(k, device=DEV) if kind == "all" else torch.tensor([517], device=DEV)
    x[:, columns] = large[:, columns]
    x, codes = one_sign(x, codes, positive)
    w = plain_values(codes, scales)
    check_product(x.bfloat16(), kernels.mxfp4_matrix(codes, scales), w, quantise, plan, f"{kind} {top}")


@pytest.mark.parametrize("plan,quantise", [(plan, q) for plan in SOME_PLANS + [("few", 8)] for q in (False, True) if takes(plan, 2, 768, q)])
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("low,high", [(0, 0), (0, 12), (12, 12)])
@pytest.mark.parametrize("beside", [False, True])
def test_small_rows_and_the_smallest_scales(beside, low, high, positive, plan, quantise):
    """Stages of the smallest size that halfs take (2^-20) to 1 against scales of 2^-127 to 2^-115, where a long row's sum may be an ordinary
    float and its products are not; `beside` them a much larger column that meets codes of zero."""
    m, n, k = 2, 150, 12288
    for size in (-20, -19, -12, -8, -7, 0):
        g = torch.Generator(device=DEV).manual_seed(size + high + 100)
        codes, _, _ = random_matrix(g, n, k)
        scales = torch.randint(low, high + 1, (n, k // 32), device=DEV, generator=g, dtype=torch.uint8)
        x = torch.randn(m, k, device=DEV, generator=g).clamp(-1.9, 1.9) * 2.0 ** size
        if beside:
            x[:, ::256] = 2.0 ** (size + 32)
            codes = codes.clone()
            codes[:, ::128] &= 0xF0
        x, codes = one_sign(x, codes, positive)
        w = plain_values(codes, scales)
        x = x.bfloat16()
        values = plain_quantise(x)[0] if quantise else x.double()
        out = torch.full((m, n), 7.0, device=DEV)
        kernels.mxfp4_gemm(x, kernels.mxfp4_matrix(codes, scales), out, quantise=quantise, plan=fitting(plan, m, n, k))
        close_to_small_sums(out, values @ w.T, values.abs() @ w.abs().T, k, f"{size} {low} {high}")


@pytest.mark.parametrize("scale", [253, 254])
def test_scales_beyond_float32_are_refused_beside_blocks_that_are_no_numbers(scale):
    codes = torch.full((5, 64), 0x17, device=DEV, dtype=torch.uint8)
    scales = torch.full((5, 4), 120, device=DEV, dtype=torch.uint8)
    scales[1, 2] = 255
    assert kernels.mxfp4_matrix(codes, scales).half_exponent is None
    scales[4, 3] = scale
    with pytest.raises(InvalidRequest, match="float32"):
        kernels.mxfp4_matrix(codes, scales)
    codes[4, 48:] = 0x80                                       # zeros may have any scale
    weight = kernels.mxfp4_matrix(codes, scales)
    assert torch.equal(weight.block_scales(), scales)
    check_product(torch.ones(3, 128, device=DEV).bfloat16(), weight, plain_values(codes, scales), False, None, "beside no numbers")


@pytest.mark.parametrize("m,quantise", ALL_KINDS)
def test_an_output_over_the_weights_is_refused(m, quantise):
    """Over the first codes, the last scales, or all of them; right before and behind them is no overlap."""
    n, k = 256, 512
    x = torch.randn(m, k, device=DEV).bfloat16()
    held = kernels.mxfp4_quantise(torch.randn(n, k, device=DEV))
    size, bytes_ = 2 * m * n, held.bytes()
    buffer = torch.zeros(2 * size + bytes_, device=DEV, dtype=torch.uint8)
    buffer[size:size + bytes_] = held.data
    weight = kernels.Mxfp4(buffer[size:size + bytes_], n, k).settle()

    def out(begin):
        return buffer[begin:begin + size].view(torch.bfloat16).view(m, n)

    for begin in {2, size, size + bytes_ - 2, min(size + 4096, size + bytes_ - 2)}:
        with pytest.raises(InvalidRequest, match="overlaps the weights"):
            kernels.mxfp4_gemm(x, weight, out(begin), quantise=quantise)
    before = weight.data.clone()
    want = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
    kernels.mxfp4_gemm(x, weight, want, quantise=quantise)
    for begin in (0, size + bytes_):
        kernels.mxfp4_gemm(x, weight, out(begin), quantise=quantise)
        assert torch.equal(out(begin), want) and torch.equal(weight.data, before)


WIDE_PLANS = [("parts", 16, 5, False), ("parts", 16, 9, True), ("parts", 32, 4, False), ("parts", 32, 7, True), ("parts", 64, 3, False), ("parts", 64, 6, True)]


@pytest.mark.parametrize("plan", WIDE_PLANS)
@pytest.mark.parametrize("kind", ["far", "infinite", "nan"])
@pytest.mark.parametrize("n,k", [(390, 1280), (133, 128), (17, 640)])
def test_rows_that_parts_do_not_hold_beside_others(n, k, kind, plan):
    """One row, the last, a few, more than sixteen or all of a batch have elements that three parts do not hold, nine and more in 256, or two
    each that are too many together: what belongs to each row is right, and the other rows' results have the bits that they have without."""
    m = plan[1] - 1
    g = torch.Generator(device=DEV).manual_seed(n + k + plan[1])
    codes, scales, w = random_matrix(g, n, k)
    weight = kernels.mxfp4_matrix(codes, scales)
    plan = fitting(plan, m, n, k)
    plain = torch.randn(m, k, device=DEV, generator=g).bfloat16()
    without = torch.full((m, n), 7.0, device=DEV)
    kernels.mxfp4_gemm(plain, weight, without, plan=plan)
    order = torch.randperm(m, device=DEV, generator=g).tolist()
    for rows in ([m - 1], order[:1], order[:3], order[:17], order):
        for each in (2, 9, k):
            x = plain.float()
            columns = torch.randperm(k, device=DEV, generator=g)[:each]
            for row in rows:
                if kind == "far":
                    x[row, columns] *= 2.0 ** -45
                else:
                    x[row, columns[::2]] = math.inf if kind == "infinite" else math.nan
                    x[row, columns[1::2]] *= 2.0 ** 60
            check_product(x.bfloat16(), weight, w, False, plan, f"{len(rows)} rows {each}")
            out = torch.full((m, n), 7.0, device=DEV)
            kernels.mxfp4_gemm(x.bfloat16(), weight, out, plan=plan)
            others = sorted(set(range(m)) - set(rows))
            assert torch.equal(out[others], without[others]), f"{len(rows)} rows {each}"


@pytest.mark.parametrize("m,n,k,rows,each", [(300, 390, 4096, 1, 40), (300, 390, 4096, 7, 3), (300, 390, 4096, 300, 1), (2048, 24576, 4096, 8, 12), (2048, 24576, 4096, 110, 1),
                                             (2048, 24576, 4096, 111, 1), (2048, 24576, 4096, 8, 128), (100, 24576, 4096, 1, 5), (100, 24576, 4096, 3, 2), (11, 4096, 4128, 1, 1)])
def test_either_operand_for_rows_with_elements_far_below(m, n, k, rows, each):
    """Few elements in many rows and many in few (more in a row than a number of four bits counts), on both sides of what changes the whole
    product's operands.  They alone meet codes that are not zero."""
    g = torch.Generator(device=DEV).manual_seed(m + k + rows)
    codes, scales, _ = random_matrix(g, n, k)
    order = torch.randperm(k // 256, device=DEV, generator=g)                # no more than eight in 256 elements of a row
    nonzero = (order[:, None] * 256 + torch.arange(3, 256, 32, device=DEV)[None, :]).T.reshape(-1)[:each]
    keep = torch.zeros(k, dtype=torch.bool, device=DEV)
    keep[nonzero] = True
    codes = codes & (torch.where(keep[0::2], 0x0F, 0) | torch.where(keep[1::2], 0xF0, 0)).to(torch.uint8)
    x = torch.randn(m, k, device=DEV, generator=g)
    x[:, nonzero] = 0.0
    for row in torch.randperm(m, device=DEV, generator=g)[:rows].tolist():
        x[row, nonzero] = torch.randn(each, device=DEV, generator=g) * 2.0 ** -50
    x = x.bfloat16()
    weight, w = kernels.mxfp4_matrix(codes, scales), plain_values(codes, scales)[:, nonzero]
    out = torch.full((m, n), 7.0, device=DEV)
    kernels.mxfp4_gemm(x, weight, out)
    close_to_sums(out, x[:, nonzero].double() @ w.T, x[:, nonzero].double().abs() @ w.abs().T, k, f"{rows} rows {each}")


@pytest.mark.parametrize("plan,quantise", [(plan, q) for plan in SOME_PLANS + [("few", 8), ("parts", 32, 3, True), ("many", 16, 4, True)] for q in (False, True) if takes(plan, 8, 640, q)])
@pytest.mark.parametrize("kind", ["infinity", "infinities", "nan", "all nan", "both", "all infinite", "beside far"])
def test_rows_that_are_not_finite_beside_others(kind, plan, quantise):
    """An infinity or NaN decides its own row, whatever else is in it and whether it meets weights of zero, and leaves the others what they are."""
    m, n, k = 8, 150, 1408
    g = torch.Generator(device=DEV).manual_seed(len(kind))
    codes, scales, _ = random_matrix(g, n, k)
    codes[::2, 100:140] = 0                                    # weights of zero: infinity times these is none
    codes[1::4, 100:140] &= 0x70
    scales[5, 7] = 255
    w = plain_values(codes, scales)
    weight = kernels.mxfp4_matrix(codes, scales)
    x = torch.randn(m, k, device=DEV, generator=g)
    x[:, 64:96] = 0.0
    plain = torch.full((m, n), 7.0, device=DEV)
    kernels.mxfp4_gemm(x.bfloat16(), weight, plain, quantise=quantise, plan=plan)
    for row in (6, 2):                                         # first one such row, then two
        if kind == "infinity":
            x[row, 3] = -math.inf
        elif kind == "infinities":
            x[row, [5, 6, 900]] = math.inf
            x[row, 1200] = -math.inf if row == 2 else math.inf
        elif kind == "nan":
            x[row, k - 1] = math.nan
        elif kind == "all nan":
            x[row] = -math.nan
        elif kind == "both":
            x[row, 200], x[row, 210], x[row, 700] = math.inf, -math.inf, math.nan
        elif kind == "all infinite":
            x[row] = math.inf
        else:
            x[row] *= torch.exp2(torch.randint(-60, 60, (k,), device=DEV, generator=g).float())
            x[row, 77] = math.inf
        check_product(x.bfloat16(), weight, w, quantise, plan, kind)
        out = torch.full((m, n), 7.0, device=DEV)
        kernels.mxfp4_gemm(x.bfloat16(), weight, out, quantise=quantise, plan=plan)
        others = [i for i in range(m) if i != row and (i != 6 or row != 2)]
        columns = [i for i in range(n) if i != 5]              # a row of w that is not a number is none for every row of x
        assert out[:, 5].isnan().all()
        if plan[0] != "few":                                   # there such a row brings the others' stages to bfloat16: another order of their sums
            assert torch.equal(out[others][:, columns], plain[others][:, columns])
