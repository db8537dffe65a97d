"""Linear layers in e4m3 that quantise their input themselves: the product is launched while the kernel that writes the
quantised rows still runs, and those rows lie in memory that the call gives back when it returns."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from xdit_b200 import ops  # noqa: E402
from xdit_b200.fp8_linear import fp8_linear, quantize_weight  # noqa: E402

# the kernel for few rows, alone and with the inner axis shared by a cluster; tiles of single CTAs; tiles of pairs
SIZES = [(64, 20000, 8192), (200, 384, 8192), (600, 2048, 1920), (8000, 4096, 1024)]


def _case(M, N, K, seed, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, device="cuda", generator=g).to(dtype)
    w = quantize_weight(torch.randn(N, K, device="cuda", generator=g) * K ** -0.5)
    return x, w, torch.randn(N, device="cuda", generator=g)


@pytest.mark.parametrize("M,N,K", SIZES)
def test_a_skipped_product_ends_behind_the_kernel_that_quantises_its_rows(M, N, K):
    """A failure is pending on the device, so every CTA skips its work.  The memory of the quantised rows goes to the next
    tensor of the stream, and what is written there stays."""
    x, w, b = _case(M, N, K, 1)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    status = ops._status(x.device).dev  # (allocated on its first use: before the address is looked up)
    size = (M * K + 15) // 16 * 16 + 4 * M * -(-K // 128)
    first = torch.empty(size, dtype=torch.uint8, device="cuda")
    address = first.data_ptr()
    del first
    try:
        status.fill_(777)
        for _ in range(5):
            ops.fp8_linear(x.unsqueeze(0), None, w.data, w.scale, b, out=out)
            after = torch.full((size,), 0x5a, dtype=torch.uint8, device="cuda")
            assert after.data_ptr() == address  # the memory that the call worked in
            torch.cuda.synchronize()
            assert (after == 0x5a).all()
            del after
        assert torch.isnan(out).all()
    finally:
        ops.clear_status(x.device)
    assert torch.equal(fp8_linear(x, w, b), fp8_linear(x, w, b))
