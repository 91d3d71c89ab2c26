"""What the 4-bit entry points refuse before anything is launched; host arithmetic of their launches.  No GPU."""
import pytest
import torch

from mini_rsglang_b200 import RuntimeConfig, kernels
from mini_rsglang_b200.csrc.build import mxfp4_kernel_library
from mini_rsglang_b200.errors import BackendError, InvalidRequest


def matrix(rows, width):
    return kernels._mxfp4_empty(rows, width, "cpu")


@pytest.mark.parametrize("shape", [(4, 33), (4, 16), (4, 0), (32,), (2, 2, 32)])
def test_quantise_refuses_rows_that_are_no_whole_blocks(shape):
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_quantise(torch.zeros(shape))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64, torch.int32])
def test_quantise_refuses_other_types(dtype):
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_quantise(torch.zeros(4, 32, dtype=dtype))


def test_nothing_runs_without_a_gpu():
    with pytest.raises(BackendError):
        kernels.mxfp4_quantise(torch.zeros(4, 32))
    with pytest.raises(BackendError):
        kernels.mxfp4_dequantise(matrix(4, 32))
    with pytest.raises(BackendError):
        kernels.mxfp4_matrix(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    with pytest.raises(BackendError):
        kernels.mxfp4_gemm(torch.zeros(2, 64, dtype=torch.bfloat16), matrix(8, 64), torch.zeros(2, 8))


def test_dequantise_refuses_other_types():
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_dequantise(matrix(4, 32), torch.float16)


@pytest.mark.parametrize("codes,scales", [((4, 16), (4, 2)), ((4, 16), (3, 1)), ((4, 17), (4, 1)), ((4, 16), (4,)), ((64,), (4, 1)), ((4, 0), (4, 0))])
def test_matrix_refuses_sizes_that_do_not_match(codes, scales):
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_matrix(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8))


@pytest.mark.parametrize("x,out,dtype", [((2, 96), (2, 8), torch.float32), ((2, 64, 1), (2, 8), torch.float32),
                                         ((2, 64), (16,), torch.float32), ((2, 64), (2, 8), torch.float16)])
def test_product_refuses_sizes_and_types(x, out, dtype):
    with pytest.raises(InvalidRequest):
        kernels.mxfp4_gemm(torch.zeros(x, dtype=torch.bfloat16), matrix(8, 64), torch.zeros(out, dtype=dtype))


@pytest.mark.parametrize("data,rows,width", [(torch.zeros(10, dtype=torch.uint8), 128, 256), (torch.zeros(1152 - 1, dtype=torch.uint8), 1, 256),
                                             (torch.zeros(1152, dtype=torch.int8), 1, 256), (torch.zeros(1152 * 2, dtype=torch.uint8)[::2], 1, 256),
                                             (torch.zeros(2, 576, dtype=torch.uint8), 1, 256), (torch.zeros(1152, dtype=torch.uint8), -1, 256),
                                             (torch.zeros(1152, dtype=torch.uint8), 1, 250), (torch.zeros(1152 + 16, dtype=torch.uint8)[16:], 1, 256)])
def test_a_matrix_has_the_bytes_of_its_sizes(data, rows, width):
    with pytest.raises(InvalidRequest):
        kernels.Mxfp4(data, rows, width)


def test_a_matrix_of_given_bytes():
    data = matrix(3, 320).data
    held = kernels.Mxfp4(data, 3, 320)
    assert held.data is data and held.shape == (3, 320) and not held.settled and held.codes.shape == (3, 160)


def test_block_scales_reads_the_tiles():
    """A scale lies at byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 of tile (r / 128, b / 4)."""
    for rows, width in ((1, 32), (129, 288), (300, 1056)):
        m = matrix(rows, width)
        want = torch.randint(0, 256, (rows, width // 32), dtype=torch.uint8)
        tiles = -(-width // 256) * 2
        for r in range(rows):
            for b in range(width // 32):
                m.scales[(r // 128 * tiles + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4] = want[r, b]
        assert torch.equal(m.block_scales(), want)
    assert matrix(0, 64).block_scales().shape == (0, 2)


@pytest.mark.parametrize("kwargs", [dict(weight_format="int4"), dict(activation_format="mxfp4"), dict(weight_format="mxfp4", activation_format="fp8")])
def test_runtime_config_refuses_other_formats(kwargs):
    with pytest.raises(InvalidRequest):
        RuntimeConfig(**kwargs).validate()


def test_runtime_config_takes_both_formats():
    RuntimeConfig().validate()
    RuntimeConfig(weight_format="mxfp4").validate()
    RuntimeConfig(weight_format="mxfp4", activation_format="mxfp4").validate()


@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 33, 128, 129, 485, 4096])
@pytest.mark.parametrize("n,k", [(1, 32), (128, 4096), (6145, 4096), (24576, 4096), (5120, 17408), (151936, 1024), (40, 65536)])
@pytest.mark.parametrize("tokens,shared", [(16, None), (32, True), (192, None), (128, False)])
def test_tiles_have_work_for_every_cta(m, n, k, tokens, shared):
    """No more CTAs than SMs, and none without a stage (shared tiles) or a tile of its own."""
    got, ctas, is_shared = kernels.mxfp4_tiles(m, n, k, tokens, 148, 11, shared)
    tiles, depth = -(-n // 128) * -(-m // tokens), -(-k // 256)
    assert got == tokens and 1 <= ctas <= 148 and ctas <= (tiles * depth if is_shared else tiles)
    assert shared is None or is_shared is shared


@pytest.mark.parametrize("quantise", [False, True])
@pytest.mark.parametrize("m", range(1, 9))
def test_few_rows_get_clusters_that_hold_them(m, quantise, monkeypatch):
    """Whatever the plan weighs, the CTAs of a cluster of the kernel for few rows have shared memory for their ranges of x."""
    lib = mxfp4_kernel_library()
    monkeypatch.setattr(kernels, "mxfp4_library", lambda: lib)
    for n in (1, 100, 3394, 5120, 8193, 18944, 18945, 30000):
        for k in (*range(32, 1024, 32), *range(1024, 36000, 416), 11296, 12832, 14816, 15392, 17376, 18464, 23104, 30752, 65536, 131072, 131104, 1 << 20):
            plan = kernels.mxfp4_plan(m, n, k, quantise, 148)
            if plan[0] == "few":
                assert 0 < lib.mrs_mxfp4_few_rows_cluster(m, k) <= plan[1], (m, n, k, plan)


def test_product_refuses_an_output_over_what_it_reads(monkeypatch):
    """Over the input and over the weights, from either side, before the GPU is asked for anything."""
    def gpu():
        raise BackendError("asked for")

    monkeypatch.setattr(kernels, "_need", lambda *_: None)
    monkeypatch.setattr(kernels, "_current_device", gpu)
    memory = torch.zeros(1 << 14, dtype=torch.uint8)
    memory = memory[-memory.data_ptr() % 32:]
    size = matrix(128, 64).bytes()
    weight = kernels.Mxfp4(memory[4096:4096 + size], 128, 64)
    x = memory[12288:12288 + 256].view(torch.bfloat16).view(2, 64)
    for begin, end, over in ((4096, 4096 + size, "weights"), (12288, 12288 + 256, "input")):
        for at in (begin - 510, begin - 2, begin, end - 2):
            with pytest.raises(InvalidRequest, match=f"overlaps the {over}"):
                kernels.mxfp4_gemm(x, weight, memory[at:at + 512].view(torch.bfloat16).view(2, 128))
        for at in (begin - 512, end):
            with pytest.raises(BackendError, match="asked for"):
                kernels.mxfp4_gemm(x, weight, memory[at:at + 512].view(torch.bfloat16).view(2, 128))
