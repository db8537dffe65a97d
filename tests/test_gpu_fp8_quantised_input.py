"""Linear layers in e4m3 that quantise their input themselves: the product is launched while the kernel that writes the
quantised rows still runs, and those rows lie in memory that the call gives back when it returns."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from xdit_b200 import ops  # noqa: E402
from xdit_b200.fp8_linear import fp8_linear, quantize_rows, quantize_weight  # noqa: E402

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


def _same(a, b):
    return torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8)) and torch.equal(a.scale, b.scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,s,N,K", [(1, 1, 2304, 5120), (2, 1, 4608, 1040), (3, 21, 1152, 2064), (5, 40, 384, 8192), (2, 300, 2048, 1920),
                                     (2, 1021, 4096, 272), (3, 2700, 4096, 400), (1, 30000, 528, 144)])
def test_the_bits_of_rows_quantised_before(B, s, N, K, dtype):
    """Every kernel and every split behind the quantising one, from samples of a larger tensor: rows apart, a batch stride of its
    own.  What the call makes is what it makes of the rows that quantize_rows made before, in 16 or 32 bits and in e4m3."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(B, s + 3, K + 32, device="cuda", generator=g).to(dtype)[:, 2:2 + s, 16:16 + K]
    w = quantize_weight(torch.randn(N, K, device="cuda", generator=g) * K ** -0.5)
    b = torch.randn(N, device="cuda", generator=g)
    rows = quantize_rows(x.contiguous())
    assert _same(quantize_rows(x), rows)
    torch.cuda.synchronize()
    for _ in range(3):
        got = fp8_linear(x, w, b, activation="gelu_tanh")
        assert got.shape == (B, s, N) and got.dtype == dtype
        assert torch.equal(got, fp8_linear(rows, w, b, activation="gelu_tanh", out_dtype=dtype))
    assert _same(fp8_linear(x, w, b, quantize_out=True), fp8_linear(rows, w, b, quantize_out=True))


@pytest.mark.parametrize("M,N,K", [(2, 9216, 5120), *SIZES])
def test_two_streams_at_once(M, N, K):
    """Each call quantises into memory of its own, on both streams while the other one's products run."""
    cases = [_case(M, N, K, seed) for seed in (3, 4)]
    want = [fp8_linear(quantize_rows(x), w, b) for x, w, b in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = []
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(fp8_linear(*cases[i % 2]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(outs))
    ops.check_status()


@pytest.mark.parametrize("M,N,K", SIZES)
def test_a_chain_of_calls_captured_and_replayed(M, N, K):
    """Several calls in one graph, each behind the last, whose workspaces the graph may give to one another."""
    x, w, b = _case(M, N, K, 5)
    back = quantize_weight(torch.randn(K, N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)) * N ** -0.5)

    def chain():
        y = x
        for _ in range(3):
            y = fp8_linear(fp8_linear(y, w, b, activation="gelu_tanh"), back)
        return y

    chain()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for seed in (7, 8):
        x.copy_(_case(M, N, K, seed)[0])
        want = chain()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    ops.check_status()
