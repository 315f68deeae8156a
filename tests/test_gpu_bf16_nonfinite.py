"""bf16_gemm, which has no error flag, over operands that hold NaN and
infinities: the rows and columns that they reach come out as the formula says,
the others as without them."""
import pytest

from pih_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import torch

    from pih_amd.device import engine_stream

    with engine_stream() as s:
        yield s
        torch.cuda.synchronize()


# one row, a batch of few, tiles chosen per shape, walked tiles, 128 x 256 tiles
@pytest.mark.parametrize("m,n,k", [(1, 512, 512), (3, 256, 1024), (8, 1024, 512), (40, 512, 2048), (70, 256, 512),
                                   (200, 1024, 1024), (300, 512, 256), (1024, 2048, 1024), (100, 49152, 256)])
@pytest.mark.parametrize("output", [abi.OUTPUT_BF16, abi.OUTPUT_F32])
def test_nonfinite_operands(eng, m, n, k, output):
    import torch

    from pih_amd.linear import bf16_gemm

    g = torch.Generator(device="cuda").manual_seed(m + n)
    a = torch.randn(m, k, generator=g, device="cuda").abs().add_(0.1).to(torch.bfloat16)
    w = torch.randn(n, k, generator=g, device="cuda").abs().add_(0.1).to(torch.bfloat16)
    clean = bf16_gemm(a, w, output)
    w[n // 3, 5], w[n - 1, k - 1] = float("inf"), float("nan")
    if m > 2:
        a[m // 2, 7] = float("inf")
        a[m - 1, 0] = float("nan")
    got = bf16_gemm(a, w, output)
    torch.cuda.synchronize()
    want = clean.clone()
    want[:, n // 3] = float("inf")  # (all factors are positive)
    if m > 2:
        want[m // 2] = float("inf")
        want[m - 1] = float("nan")
    want[:, n - 1] = float("nan")
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))
