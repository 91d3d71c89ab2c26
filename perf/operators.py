"""The operators of 4-bit weights: what they are timed and checked on.

A matrix in microscaled 4-bit floating point (MXFP4) holds for every element a sign, two bits of exponent and one of
mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), and for every 32 neighbours of a row one power of two.

Kinds of cases:
  quantise   rows of bfloat16 or float32 to 4 bits, and the values that these stand for
  weights    x . W^T with W in 4 bits and x in bfloat16: a decoded token's or a prompt's projection
  both       the same with x's rows brought to 4 bits first
Sizes are those of `bench.py`'s dense shapes ("0.6b", "8b", "14b") and odd ones beside them; the weights are seeded normal numbers
brought to 4 bits, the activations have a few columns that are much larger than the others, as activations have."""
import math

import torch

own = False

BLOCK = 32
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LARGEST = 4096 * 24576 * 4096        # multiply-adds of the largest product
LARGEST_ROWS = 2048 * 17408          # elements of the largest quantised matrix


def listed():
    return [
        # the input of a decode step's projection
        {"name": "quantise_decode", "kind": "quantise", "rows": 8, "width": 4096, "dtype": "bfloat16"},
        # a prompt's input of the last product of a feed-forward
        {"name": "quantise_prompt", "kind": "quantise", "rows": 2048, "width": 17408, "dtype": "bfloat16"},
        # weights from a float32 checkpoint, an odd number of rows
        {"name": "quantise_float32", "kind": "quantise", "rows": 5003, "width": 5120, "dtype": "float32"},
        # one user's token through the projection to queries, keys and values
        {"name": "weights_one_token", "kind": "weights", "rows": 1, "n": 6144, "k": 4096, "out": "bfloat16"},
        # eight users' tokens through gate and up
        {"name": "weights_decode_8", "kind": "weights", "rows": 8, "n": 24576, "k": 4096, "out": "bfloat16"},
        # eleven users' tokens through a long product back to the stream
        {"name": "weights_decode_11", "kind": "weights", "rows": 11, "n": 5120, "k": 17408, "out": "bfloat16"},
        # a batch's logits over the whole vocabulary, in float32
        {"name": "weights_head", "kind": "weights", "rows": 24, "n": 151936, "k": 1024, "out": "float32"},
        # a portion of a prompt, of odd length, and an odd number of outputs
        {"name": "weights_portion", "kind": "weights", "rows": 485, "n": 6145, "k": 4096, "out": "bfloat16"},
        # a long prompt through gate and up
        {"name": "weights_prompt", "kind": "weights", "rows": 2048, "n": 24576, "k": 4096, "out": "bfloat16"},
        # decoded tokens, activations in 4 bits too
        {"name": "both_decode_4", "kind": "both", "rows": 4, "n": 4096, "k": 12288, "out": "bfloat16"},
        # a portion of a prompt, activations in 4 bits too
        {"name": "both_portion", "kind": "both", "rows": 333, "n": 4096, "k": 12288, "out": "bfloat16"},
        # long prompts through gate and up, activations in 4 bits too
        {"name": "both_prompts", "kind": "both", "rows": 4096, "n": 24576, "k": 4096, "out": "bfloat16"},
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantise", "weights", "weights", "both", "both"])
    if kind == "quantise":
        rows = _between(rng, 1, 8192)
        width = BLOCK * _between(rng, 1, max(1, min(544, LARGEST_ROWS // (BLOCK * rows))))
        return {"kind": kind, "rows": rows, "width": width, "dtype": rng.choice(["bfloat16", "float32"])}
    rows = _between(rng, 1, 4096)
    n = _between(rng, 40, 24576)
    k = BLOCK * _between(rng, 2, max(2, min(544, LARGEST // (BLOCK * rows * n))))
    return {"kind": kind, "rows": rows, "n": n, "k": k, "out": rng.choice(["bfloat16", "bfloat16", "float32"])}


def _codes_and_scales(x):
    """Codes (0 to 15, one a byte) and scale bytes of rows of finite float32: the exponent of a block is that of its largest
    element less two; ties go to the even code; what lies above 6 becomes 6."""
    rows, width = x.shape
    blocks = x.view(rows, width // BLOCK, BLOCK)
    largest = blocks.abs().amax(dim=2, keepdim=True)
    exponent = (torch.frexp(largest)[1] - 3).clamp(-127, 125)
    exponent = torch.where(largest == 0, torch.full_like(exponent, -127), exponent).to(torch.int32)
    y = blocks * ((127 - exponent) << 23).view(torch.float32)            # 2^-exponent, an ordinary number
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = code + 8 * (y < 0).to(torch.uint8)
    return code.view(rows, width), (exponent + 127).to(torch.uint8).view(rows, width // BLOCK)


def _values(code, scale):
    """What codes (one a byte) and scale bytes stand for."""
    rows, width = code.shape
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float32, device=code.device)
    value = table[code.to(torch.int32)].view(rows, width // BLOCK, BLOCK)
    power = (scale.to(torch.int32) << 23).clamp(min=1 << 22).view(torch.float32)        # byte 0: 2^-127, under the ordinary numbers
    return (value * power.view(rows, width // BLOCK, 1)).view(rows, width)


def _unpack(packed):
    return torch.stack([packed & 15, packed >> 4], dim=2).view(packed.shape[0], -1)


def _activations(generator, rows, width, dtype):
    x = torch.randn(rows, width, device="cuda", generator=generator)
    strong = torch.rand(width, device="cuda", generator=generator) < 0.01
    x = torch.where(strong, x * 25.0, x)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    if case["kind"] == "quantise":
        dtype = TYPES[case["dtype"]]
        return {"case": case, "x": _activations(g, case["rows"], case["width"], dtype)}
    x = _activations(g, case["rows"], case["k"], torch.bfloat16)
    weight = torch.randn(case["n"], case["k"], device="cuda", generator=g) * 0.02
    code, scale = _codes_and_scales(weight)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    state = {"case": case, "x": x, "codes": packed.contiguous(), "scales": scale}
    if own:
        from mini_rsglang_b200 import kernels

        state["weight"] = kernels.mxfp4_matrix(state["codes"], state["scales"])
    return state


def run(state):
    case, x = state["case"], state["x"]
    if own:
        from mini_rsglang_b200 import kernels

        if case["kind"] == "quantise":
            return kernels.mxfp4_dequantise(kernels.mxfp4_quantise(x), x.dtype)
        out = torch.empty(case["rows"], case["n"], dtype=TYPES[case["out"]], device=x.device)
        kernels.mxfp4_gemm(x, state["weight"], out, quantise=case["kind"] == "both")
        return out
    if case["kind"] == "quantise":
        return _values(*_codes_and_scales(x.float())).to(x.dtype)
    x = x.float()
    if case["kind"] == "both":
        x = _values(*_codes_and_scales(x))
    weight = _values(_unpack(state["codes"]), state["scales"])
    return torch.matmul(x, weight.t()).to(TYPES[case["out"]])


def exact(case, seed):
    """In 64 bits, from the definition: a block's power of two is 2^(floor(log2 of its largest) - 2), an element the nearest of the
    fifteen values times it (of two equally near the one whose last mantissa bit is 0)."""
    state = prepare(case, seed)
    grid = torch.tensor(VALUES, dtype=torch.float64, device="cuda")

    def power_of_two(exponent):                   # from its bits: exp2 need not be exact
        return ((exponent.long() + 1023) << 52).view(torch.float64)

    def rounded(x):
        blocks = x.double().view(x.shape[0], -1, BLOCK)
        largest = blocks.abs().amax(dim=2, keepdim=True)
        power = power_of_two(((largest.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 125))
        size = (blocks / power).abs()
        best = torch.zeros_like(size)
        for i in range(1, len(VALUES)):
            middle = (grid[i - 1] + grid[i]) / 2
            best = torch.where((size > middle) | ((size == middle) & (i % 2 == 0)), grid[i], best)
        return (best * torch.sign(blocks) * power).view(x.shape)

    if case["kind"] == "quantise":
        return rounded(state["x"])
    x = rounded(state["x"]) if case["kind"] == "both" else state["x"].double()
    low, high = (state["codes"] & 15).long(), (state["codes"] >> 4).long()
    signed = torch.cat([grid, -grid])
    weight = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
    weight[:, 0::2], weight[:, 1::2] = signed[low], signed[high]
    weight *= power_of_two(state["scales"].long() - 127).repeat_interleave(BLOCK, dim=1)
    return x @ weight.t()


def work(case):
    if case["kind"] == "quantise":
        elements, size = case["rows"] * case["width"], 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": elements * size * 2, "flops": 0}
    m, n, k = case["rows"], case["n"], case["k"]
    weight = n * k // 2 + n * k // BLOCK
    return {"bytes": m * k * 2 + weight + m * n * (2 if case["out"] == "bfloat16" else 4), "flops": 2 * m * n * k}
