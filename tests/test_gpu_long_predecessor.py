"""A GEMM of a declared weight behind a kernel that runs longer than the limit of the GEMM's own waits: it becomes resident
and requests its weight while that kernel runs, and must then wait for it without a limit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LIMIT = 1.53  # seconds that a wait in the kernels lasts, at the highest clock


@pytest.fixture(scope="module")
def long_kernel(hom):
    """A mask of one row, whose sum one warp walks through."""
    import torch

    hom.use_torch_stream()
    cu = torch.empty(2, dtype=torch.int32, device="cuda")

    def seconds(mask):
        start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        hom.thrustCuSeqLenI64(mask, cu)
        stop.record()
        stop.synchronize()
        return start.elapsed_time(stop) * 1e-3

    probe = torch.zeros((1, 1 << 24), dtype=torch.int64, device="cuda")
    seconds(probe)
    n = min(int(1.4 * LIMIT / seconds(probe) * (1 << 24)), (1 << 31) - 64)
    mask = torch.zeros((1, n), dtype=torch.int64, device="cuda")
    mask[0, -1] = 7
    assert seconds(mask) > 1.2 * LIMIT
    yield lambda: hom.thrustCuSeqLenI64(mask, cu)
    hom.synchronize()
    assert cu.tolist() == [0, 7]


@pytest.mark.parametrize("form", ["one_cta", "pair", "cluster"])
def test_fp16_gemm(hom, cuda, long_kernel, form):
    import torch

    m, n, k = 512, 512, 2048
    row, split = {"one_cta": (1, 1), "pair": (6, 1), "cluster": (1, 2)}[form]
    torch.manual_seed(1)
    a, b = torch.randn((1, m, k), device=cuda).half(), torch.randn((1, k, n), device=cuda).half()
    want, got = (torch.zeros((1, m, n), dtype=torch.float16, device=cuda) for _ in range(2))
    torch.cuda.synchronize()
    hom.declare_weights(b)
    try:
        hom.cutlassGemmF16(a, b, want, want, gemmNum=row, splitKFactor=split)
        hom.synchronize()
        long_kernel()
        hom.cutlassGemmF16(a, b, got, got, gemmNum=row, splitKFactor=split)
        hom.synchronize()
    finally:
        hom.forget_weights(b)
    assert torch.equal(got, want) and bool(want.any())


@pytest.mark.parametrize("m,n", [(200, 512), (2048, 1024)])
def test_4_bit_product(hom, pkg, cuda, long_kernel, m, n):
    """One wave of small tiles, and pairs."""
    import torch

    k = 4096
    torch.manual_seed(2)
    a, b = ([torch.empty(s, dtype=torch.uint8, device=cuda) for s in pkg.mxf4_shapes(rows, k)] for rows in (m, n))
    for operand, rows in ((a, m), (b, n)):
        hom.homQuantizeMxF4F32(torch.randn((rows, k), device=cuda), *operand)
    want, got = (torch.zeros((m, n), dtype=torch.float16, device=cuda) for _ in range(2))
    hom.synchronize()
    for t in b:
        hom.declare_weights(t)
    try:
        hom.homGemmMxF4F16(*a, *b, None, want)
        hom.synchronize()
        long_kernel()
        hom.homGemmMxF4F16(*a, *b, None, got)
        hom.synchronize()
    finally:
        for t in b:
            hom.forget_weights(t)
    assert torch.equal(got, want) and bool(np.isfinite(want.float().cpu().numpy()).all()) and bool(want.any())
