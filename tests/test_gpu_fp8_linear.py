"""Linear layers in e4m3 with block scales against their definition in 64 bits.

Tolerance.  A product of two e4m3 values is exact in fp32; a block's sum takes 128 additions in the tensor core, which may
cut where fp32 would round (2^-23 each), then one scaled sum per block in fp32, one product of the scales and one
addition of the bias.  So (128 + blocks + 4) 2^-23 of the sum of the magnitudes bounds the fp32 value, and half a spacing of
the result's type is added where it is rounded.  GELU's slope is below 1.13 and its exponential is good to 2^-16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from xdit_b200 import ops  # noqa: E402
from xdit_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear, quantize_rows, quantize_weight  # noqa: E402


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(M, K, seed, columns=False):
    g = _gen(seed)
    x = (torch.randn(M, K, device="cuda", generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    kb = -(-K // 128)
    s = torch.rand(M, kb, device="cuda", generator=g) * 0.02 + 1e-3
    return Fp8Rows(x, s.t().contiguous().t() if columns else s)


def _weight(N, K, seed):
    g = _gen(seed)
    w = (torch.randn(N, K, device="cuda", generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    return Fp8Weight(w, torch.rand(-(-N // 128), -(-K // 128), device="cuda", generator=g) * 1e-3 + 1e-5)


def _values(x, w):
    K, N = x.data.shape[1], w.data.shape[0]
    k = torch.arange(K, device="cuda") // 128
    return x.data.double() * x.scale.double()[:, k], w.data.double() * w.scale.double()[torch.arange(N, device="cuda") // 128][:, k]


def _want(x, w, bias, act):
    """(result, bound on the fp32 value's error) in 64 bits."""
    a, b = _values(x, w)
    y, mag = a @ b.T, a.abs() @ b.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    tol = (128 + x.scale.shape[1] + 4) * 2.0 ** -23 * mag
    if act:
        z = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return z, 1.13 * tol + 2.0 ** -16 * z.abs()
    return y, tol


def _check(x, w, bias=None, act=None, dtype=torch.bfloat16):
    y = fp8_linear(x, w, bias, activation=act, out_dtype=dtype)
    want, tol = _want(x, w, bias, act)
    f = torch.finfo(dtype)
    assert y.shape == want.shape and y.dtype == dtype
    tol = tol + (want.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)
    err = (y.double() - want).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.3g} of the bound"
    return y


@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 33, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("N,K", [(128, 128), (256, 640), (1, 16), (100, 144), (257, 1040), (520, 2064)])
def test_sizes(M, N, K):
    g = _gen(1)
    bias = torch.randn(N, device="cuda", generator=g)
    _check(_rows(M, K, 2), _weight(N, K, 3), bias if (M + N) % 2 else None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(3, 384, 512), (200, 384, 512), (77, 1000, 272)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_types_bias_and_gelu(M, N, K, act, dtype):
    for bias_dtype in {dtype, torch.float32}:
        bias = (torch.randn(N, device="cuda", generator=_gen(4)) * 2).to(bias_dtype)
        _check(_rows(M, K, 5, columns=True), _weight(N, K, 6), bias, act, dtype)


@pytest.mark.parametrize("M,N,K", [(2, 5120, 5120), (1, 30720, 1024), (4, 384, 13824), (509, 1152, 4096), (2100, 2304, 1152),
                                   (9450, 640, 768)])
def test_model_sizes(M, N, K):
    _check(_rows(M, K, 7, columns=True), _weight(N, K, 8), torch.randn(N, device="cuda", generator=_gen(9)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(65, 352, 6528), (129, 1000, 2064), (273, 352, 6528), (509, 130, 4096), (1000, 16, 2048)])
def test_few_tiles_of_a_long_inner_axis(M, N, K, dtype):
    """More rows than one tile of the kernel for few rows, the inner axis shared by a cluster: the last tile is a part."""
    x, w = _rows(M, K, 50, columns=True), _weight(N, K, 51)
    _check(x, w, torch.randn(N, device="cuda", generator=_gen(52)), "gelu_tanh" if M % 2 else None, dtype)


@pytest.mark.parametrize("M,N,K", [(2, 4608, 1040), (16, 2304, 2064), (64, 9216, 1024), (3, 1536, 4096), (2, 20000, 528)])
def test_every_way_that_few_rows_are_split(M, N, K):
    _check(_rows(M, K, 53, columns=True), _weight(N, K, 54), torch.randn(N, device="cuda", generator=_gen(55)))
    if N % 16 == 0:
        x, w = _rows(M, K, 53), _weight(N, K, 54)
        r = fp8_linear(x, w, quantize_out=True)
        want, tol = _want(x, w, None, None)
        s = r.scale.double().repeat_interleave(128, 1)[:, :N]
        half = torch.maximum((want.abs() + tol) * 2.0 ** -4, s * 2.0 ** -10)
        assert ((r.data.double() * s - want).abs() <= half + tol).all()


def test_one_block_at_a_time_takes_its_own_scale():
    """Every block of 128 holds ones in one place; the result is the product of the two scales of that block."""
    K, N, M = 128 * 5, 128 * 3, 160
    w = _weight(N, K, 10)
    x = _rows(M, K, 11)
    for c in range(5):
        x.data.copy_(torch.zeros(M, K))
        w.data.copy_(torch.zeros(N, K))
        x.data[:, 128 * c + 17 * c] = 1.0
        w.data[:, 128 * c + 17 * c] = 1.0
        y = fp8_linear(x, w, out_dtype=torch.float32)
        want = x.scale[:, c, None] * w.scale[torch.arange(N, device="cuda") // 128, c][None]
        assert torch.equal(y, want)


def quantised(x, K):
    """(values, scales) of the quantisation rule, in exact arithmetic on rows x [M, K] (64 bits)."""
    M = x.shape[0]
    p = torch.nn.functional.pad(x, (0, -K % 128)).view(M, -1, 128)
    m, e = torch.frexp(p.abs().amax(-1, keepdim=True))
    s = torch.exp2((e - 9 + (m > 0.875).int()).clamp_min(-126).double())
    s = torch.where(m == 0, torch.ones_like(s), s)
    y = p / s
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp_min(-6) - 3)
    return (torch.round(y / step) * step).view(M, -1)[:, :K], s[..., 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 16), (5, 128), (2, 9, 144), (3, 1000, 1152), (700, 5120)])
def test_quantize_rows_to_the_bit(shape, dtype):
    g = _gen(12)
    x = torch.randn(*shape, device="cuda", generator=g) * torch.exp2(torch.randint(-12, 8, shape[:-1] + (1,), device="cuda", generator=g).float())
    x = x.to(dtype)
    r = quantize_rows(x)
    assert r.shape == shape
    want, s = quantised(x.double().reshape(-1, shape[-1]), shape[-1])
    assert torch.equal(r.scale.double(), s)
    assert torch.equal(r.data.double(), want)


def test_quantize_rows_at_the_edges():
    x = torch.zeros(9, 256, device="cuda")
    x[1, 3] = 448.0            # fits as it is
    x[2, 3] = 448.0001         # needs the next power of two
    x[3, 130] = 1e-40          # below the smallest normal value
    x[4, 5] = 3.0e38
    x[5, 7] = float("inf")
    x[6, 200] = float("nan")
    x[7, :128] = torch.arange(128, device="cuda") / 16 + 17 / 32  # ties
    x[8, 0] = -0.4375
    r = quantize_rows(x)
    assert torch.equal(r.scale[:5, 0].cpu(), torch.tensor([1.0, 1.0, 2.0, 1.0, 2.0 ** 120]))
    assert float(r.scale[3, 1]) == 2.0 ** -126
    assert torch.isnan(r.scale[5, 0]) and float(r.scale[5, 1]) == 1.0
    assert torch.isnan(r.scale[6, 1]) and float(r.scale[6, 0]) == 1.0
    want, s = quantised(x[7:].double(), 256)
    assert torch.equal(r.data[7:].double(), want) and torch.equal(r.scale[7:].double(), s)
    w = _weight(200, 256, 13)
    y = fp8_linear(r, w)
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all() and torch.isfinite(y[[0, 1, 2, 3, 7, 8]]).all()


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 272), (5120, 1152)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_weight_to_the_bit(N, K, dtype):
    w = (torch.randn(N, K, device="cuda", generator=_gen(14)) * 0.02).to(dtype)
    r = quantize_weight(w)
    p = torch.nn.functional.pad(w.double(), (0, -K % 128, 0, -N % 128))
    blocks = p.view(-(-N // 128), 128, -(-K // 128), 128).transpose(1, 2).flatten(2)
    m, e = torch.frexp(blocks.abs().amax(-1))
    s = torch.exp2((e - 9 + (m > 0.875).int()).double())
    assert torch.equal(r.scale.double(), s)
    sx = s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = w.double() / sx
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp_min(-6) - 3)
    assert torch.equal(r.data.double(), torch.round(y / step) * step)


@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (5, 256, 640), (33, 144, 512), (200, 400, 512), (700, 1152, 256)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_result_as_e4m3_rows(M, N, K, act):
    x, w, bias = _rows(M, K, 15), _weight(N, K, 16), torch.randn(N, device="cuda", generator=_gen(17))
    r = fp8_linear(x, w, bias, activation=act, quantize_out=True)
    want, tol = _want(x, w, bias, act)
    assert isinstance(r, Fp8Rows) and r.shape == (M, N) and r.scale.shape == (M, -(-N // 128))
    s = r.scale.double()
    assert torch.equal(torch.exp2(torch.log2(s).round()), s)
    top = torch.nn.functional.pad(want, (0, -N % 128)).view(M, -1, 128).abs().amax(-1)
    slack = torch.nn.functional.pad(tol, (0, -N % 128)).view(M, -1, 128).amax(-1)
    assert (top <= 448 * s + slack).all() and (2 * (top + slack) > 448 * s).all()
    sx = s.repeat_interleave(128, 1)[:, :N]
    half = torch.maximum((want.abs() + tol) * 2.0 ** -4, sx * 2.0 ** -10)
    assert ((r.data.double() * sx - want).abs() <= half + tol).all()


@pytest.mark.parametrize("M", [3, 40, 150])
def test_strides_of_rows_scales_and_result(M):
    """Rows, weight and scales inside larger tensors, a result with rows apart; nothing beside it is written."""
    N, K = 200, 256
    big = _rows(M, K + 64, 18)
    x = Fp8Rows(big.data[:, 16:16 + K], big.scale[:, :2])
    bw = _weight(N, K + 128, 19)
    w = Fp8Weight(bw.data[:, :K], bw.scale[:, 1:3])
    buf = torch.full((M + 2, N + 9), float("nan"), dtype=torch.bfloat16, device="cuda")
    out = buf[1:-1, 4:4 + N]
    ops.fp8_linear(x.data, x.scale, w.data, w.scale, out=out)
    want, tol = _want(x, w, None, None)
    assert ((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -8 + 1e-30).all()
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[1:-1, 4:4 + N] = False
    assert torch.isnan(buf[mask]).all()


@pytest.mark.parametrize("M,N,K,dtype,act,bias", [
    (4000, 4161, 272, torch.float32, None, True), (4097, 4096, 1040, torch.float16, "gelu_tanh", True),
    (3841, 4328, 144, torch.bfloat16, None, False), (60000, 257, 16, torch.bfloat16, "gelu_tanh", False)])
def test_many_tiles(M, N, K, dtype, act, bias):
    """Sizes that go to pairs of CTAs: last tiles of one row or column, an odd number of blocks, several tiles a CTA."""
    b = torch.randn(N, device="cuda", generator=_gen(32)).to(dtype) if bias else None
    _check(_rows(M, K, 33, columns=M % 2 == 0), _weight(N, K, 34), b, act, dtype)


@pytest.mark.parametrize("M,N,K", [(4100, 4112, 400), (30000, 528, 128)])
def test_many_tiles_as_e4m3_rows(M, N, K):
    """The e4m3 result is the fp32 result quantised by the rule: the same sums, so the same bits."""
    x, w, b = _rows(M, K, 35), _weight(N, K, 36), torch.randn(N, device="cuda", generator=_gen(37))
    r = fp8_linear(x, w, b, activation="gelu_tanh", quantize_out=True)
    want = quantize_rows(fp8_linear(x, w, b, activation="gelu_tanh", out_dtype=torch.float32))
    assert torch.equal(r.scale, want.scale) and torch.equal(r.data.view(torch.uint8), want.data.view(torch.uint8))


@pytest.mark.parametrize("M,N", [(150, 200), (20, 200), (9000, 2008)])
def test_aligned_result_inside_a_larger_buffer(M, N):
    """Rows on 16-byte boundaries leave in boxes of 64 columns: nothing beside the result is written."""
    K = 256
    x, w = _rows(M, K, 38), _weight(N, K, 39)
    buf = torch.full((M + 2, N + 16), float("nan"), dtype=torch.bfloat16, device="cuda")
    out = buf[1:-1, 8:8 + N]
    ops.fp8_linear(x.data, x.scale, w.data, w.scale, out=out)
    want, tol = _want(x, w, None, None)
    assert ((out.double() - want).abs() <= tol + want.abs() * 2.0 ** -8 + 1e-30).all()
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[1:-1, 8:8 + N] = False
    assert torch.isnan(buf[mask]).all()


def test_no_rows_and_leading_axes():
    w = _weight(144, 256, 20)
    assert fp8_linear(torch.empty(2, 0, 256, device="cuda"), w).shape == (2, 0, 144)
    x = torch.randn(2, 3, 5, 256, device="cuda", generator=_gen(21)).to(torch.float16)
    y = fp8_linear(x, w)
    assert y.shape == (2, 3, 5, 144) and y.dtype == torch.float16
    assert torch.equal(y.view(30, 144), fp8_linear(x.view(30, 256), w))
    assert fp8_linear(x, w, quantize_out=True).shape == (2, 3, 5, 144)


@pytest.mark.parametrize("M", [2, 30, 500])
def test_same_result_every_time_and_on_two_streams(M):
    x, w = _rows(M, 2048, 22), _weight(640, 2048, 23)
    first = fp8_linear(x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(fp8_linear(x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("M", [2, 300])
def test_captured_and_replayed(M):
    x = torch.randn(M, 1024, device="cuda", generator=_gen(24)).to(torch.bfloat16)
    w, b = _weight(384, 1024, 25), torch.randn(384, device="cuda", generator=_gen(26))
    fp8_linear(x, w, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = fp8_linear(x, w, b, activation="gelu_tanh")
    x.copy_(torch.randn(M, 1024, device="cuda", generator=_gen(27)))
    g.replay()
    want, tol = _want(quantize_rows(x), w, b, "gelu_tanh")
    assert ((y.double() - want).abs() <= tol + want.abs() * 2.0 ** -8 + 1e-30).all()
    torch.cuda.synchronize()
    ops.check_status()


def test_a_pending_failure_is_reported_and_cleared():
    from xdit_b200._capi import XditError

    x, w = _rows(4, 128, 28), _weight(128, 128, 29)
    fp8_linear(x, w)
    torch.cuda.synchronize()
    ops._status(x.data.device).host.fill_(777)  # as an earlier launch that gave up a wait leaves it
    with pytest.raises(XditError) as e:
        fp8_linear(x, w)
    assert e.value.code == -6
    _check(x, w)


@pytest.mark.parametrize("M,N,K", [(3, 384, 1024), (40, 5120, 5120), (200, 512, 384), (8000, 4096, 256)])
def test_a_wait_that_runs_out_is_reported_by_the_next_call(M, N, K):
    """Nothing is loaded, so the kernel's waits run out after a millisecond; it drains, sets the status words and ends, the next
    call raises and launches nothing, and the one after it runs again.  Few rows (with and without a split of K), tiles of
    single CTAs and of pairs."""
    from xdit_b200._capi import XditError

    x, w = _rows(M, K, 30), _weight(N, K, 31)
    out = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    ops.fp8_linear(x.data, x.scale, w.data, w.scale, out=out, _wait_limit_ns=1_000_000, _selftest_stall=True)
    torch.cuda.synchronize()
    assert torch.isnan(out).all()
    with pytest.raises(XditError) as e:
        ops.fp8_linear(x.data, x.scale, w.data, w.scale, out=out)
    assert e.value.code == -6
    _check(x, w)
