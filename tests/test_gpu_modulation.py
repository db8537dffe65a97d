"""The gated residual and the modulated norm against their definition in 64 bits.

Tolerance, with u = 2^-24 (half a spacing of fp32 at 1).  A row's sums run over at most 40 values in a thread and
then over the threads in a tree, so a sum is off by less than 60 u of the sum of magnitudes; the mean is off by that,
the reciprocal root by half of it and two units of rsqrt.  Each element then takes at most ten more roundings.  So
128 u of the magnitudes that enter (|h| and the row's mean |h|, scaled like h) bounds both results in fp32, and half
a spacing of the result's type is added where it is rounded."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from xdit_b200.fp8_linear import Fp8Rows  # noqa: E402
from xdit_b200.modulation import gated_residual_norm  # noqa: E402

U = 2.0 ** -24


def _rand(shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)


def _norm64(x, mag, how, w, b, eps):
    """(norm(x), magnitudes that its rounding is measured by)."""
    if how is None:
        return x, mag
    mean = x.mean(-1, keepdim=True) if how == "layer" else torch.zeros_like(x[..., :1])
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y, m = (x - mean) * r, (mag + mag.mean(-1, keepdim=True)) * r
    # an error of the row's own sums moves every element in proportion to it
    m = m + y.abs() * (mag * mag).mean(-1, keepdim=True) * r * r
    if w is not None:
        y, m = y * w, m * w.abs()
    if b is not None:
        y, m = y + b, m + b.abs()
    return y, m


def _rows(t, x):
    if t is None:
        return None
    t = t.double()
    return t[:, None] if t.dim() == 2 else t


def _want(x, branch, o):
    h = x.double()
    mag = h.abs()
    if branch is not None:
        y = branch.double()
        y, m = _norm64(y, y.abs(), o.get("post_norm"), _rows(o.get("post_weight"), x), _rows(o.get("post_bias"), x), o["eps"])
        if o.get("gate") is not None:
            y, m = y * _rows(o["gate"], x), m * _rows(o["gate"], x).abs()
        rs = o.get("residual_scale", 1.0)
        h, mag = rs * h + y, abs(rs) * mag + m
    z, zm = _norm64(h, mag, o.get("norm", "layer"), _rows(o.get("weight"), x), _rows(o.get("bias"), x), o["eps"])
    if o.get("scale") is not None:
        z, zm = z * (1 + _rows(o["scale"], x)), zm * (1 + _rows(o["scale"], x).abs())
    if o.get("shift") is not None:
        z, zm = z + _rows(o["shift"], x), zm + _rows(o["shift"], x).abs()
    return h, mag, z, zm


def _within(got, want, mag, what):
    f = torch.finfo(got.dtype)
    tol = 128 * U * mag + (want.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f"{what}: worst {float((err / tol).max()):.3g} of the bound"


def _check(x, branch, **o):
    o.setdefault("eps", 1e-6)
    h, z = gated_residual_norm(x, branch, **o)
    wh, hm, wz, zm = _want(x, branch, o)
    if branch is not None:
        _within(h, wh, hm, "hidden")
    else:
        assert h is x
    if o.get("norm", "layer") is not None:
        _within(z, wz, zm, "normed")
    else:
        assert z is None
    return h, z


def _options(B, s, C, vec, how, norm, post):
    shape = {"shared": (C,), "batch2": (B, C), "batch": (B, 1, C), "token": (B, s, C)}[how]
    r = lambda n, shape=shape, **k: _rand(shape, vec, n, **k)  # noqa: E731
    return dict(gate=r(1, scale=0.5), scale=r(2, scale=0.3), shift=r(3), norm=norm, post_norm=post,
                post_weight=r(4, (C,), scale=0.1, shift=1.0) if post else None, post_bias=r(5, (C,)) if post else None,
                weight=r(6, (C,), scale=0.1, shift=1.0), bias=r(7, (C,)), residual_scale=0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C", [1, 7, 64, 72, 1152, 1155, 1288, 2056, 5120, 5128, 6001, 16384])
def test_widths_and_types(C, dtype):
    x, y = _rand((2, 5, C), dtype, 10, 2.0, 0.5), _rand((2, 5, C), dtype, 11)
    for vec in {dtype, torch.float32}:
        _check(x, y, **_options(2, 5, C, vec, "batch", "layer", None))
        _check(x, y, **_options(2, 5, C, vec, "token", "rms", "rms"))


@pytest.mark.parametrize("how", ["shared", "batch2", "batch", "token"])
@pytest.mark.parametrize("norm", ["layer", "rms", None])
@pytest.mark.parametrize("post", ["layer", "rms", None])
@pytest.mark.parametrize("B,s,C", [(1, 1, 256), (3, 67, 640)])
def test_every_combination(B, s, C, how, norm, post):
    o = _options(B, s, C, torch.float32, how, norm, post)
    if norm is None:
        for n in ("weight", "bias", "scale", "shift"):
            o[n] = None
    _check(_rand((B, s, C), torch.bfloat16, 12), _rand((B, s, C), torch.bfloat16, 13), **o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("C", [2, 130, 234, 235, 386, 387, 766, 769, 770, 1537, 2562, 10002])
def test_widths_by_pairs_and_by_values(C, dtype):
    """Widths that 16-byte words do not fit, at both ends of every way that they are split over threads."""
    x, y = _rand((3, 7, C), dtype, 30, 2.0, 0.5), _rand((3, 7, C), dtype, 31)
    for vec in {dtype, torch.float32}:
        _check(x, y, **_options(3, 7, C, vec, "batch", "layer", "rms"))
        _check(x, y, **_options(3, 7, C, vec, "token", "rms", None))


@pytest.mark.parametrize("C", [234, 1152])
@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("which", ["x", "branch", "scale"])
def test_one_operand_off_its_words(which, offset, C):
    """One operand starts between words: all of them go by pairs, or by values where the start is odd."""
    def at(shape, dtype, seed, off):
        return _rand((*shape[:-1], shape[-1] + 8), dtype, seed)[..., off:off + shape[-1]]
    x = at((2, 5, C), torch.bfloat16, 32, offset if which == "x" else 0)
    y = at((2, 5, C), torch.bfloat16, 33, offset if which == "branch" else 0)
    scale = at((2, 1, C), torch.float32, 34, offset if which == "scale" else 0)
    _check(x, y, scale=scale, shift=_rand((2, 1, C), torch.float32, 35), norm="layer")


@pytest.mark.parametrize("C", [64, 1152, 5120])
@pytest.mark.parametrize("offset", [0, 4, 8, 12])
def test_modulation_in_fp32_at_16_and_32_byte_boundaries(offset, C):
    """Rows of modulation that start on 16-byte words, and those on 32-byte ones, for all, for samples and for tokens."""
    x, y = _rand((2, 7, C), torch.bfloat16, 36), _rand((2, 7, C), torch.bfloat16, 37)
    for shape, step in (((C,), 0), ((2, 1, C), 4), ((2, 7, C), 8)):
        def at(seed):
            return _rand((*shape[:-1], C + 16 + step), torch.float32, seed)[..., offset:offset + C]
        _check(x, y, gate=at(38), scale=at(39), shift=at(40), post_norm="rms", post_weight=_rand((C,), torch.float32, 41), norm="layer")


@pytest.mark.parametrize("s", [1, 2, 149, 5000])
def test_modulated_norm_alone(s):
    C = 1152
    x = _rand((2, s, C), torch.bfloat16, 14)
    _check(x, None, scale=_rand((2, 1, C), torch.float32, 15), shift=_rand((2, 1, C), torch.float32, 16))
    _check(x, None, norm="rms", weight=_rand((C,), torch.bfloat16, 17))
    _check(x, None, shift=_rand((2, 1, C), torch.float32, 16))


def test_rows_with_a_large_mean_constant_rows_and_zeros():
    x = _rand((1, 6, 1024), torch.float32, 18)
    x[0, 1] += 1000.0
    x[0, 2] = 3.0
    x[0, 3] = 0.0
    x[0, 4] *= 1e-12
    for norm in ("layer", "rms"):
        _, z = _check(x, None, norm=norm)
        assert torch.isfinite(z).all()


def test_non_finite_values_stay_in_their_row():
    x = _rand((1, 4, 512), torch.bfloat16, 19)
    x[0, 1, 3], x[0, 2, 100] = float("inf"), float("nan")
    _, z = gated_residual_norm(x)
    assert torch.isfinite(z[0, 0]).all() and torch.isfinite(z[0, 3]).all()
    assert not torch.isfinite(z[0, 1]).any() and torch.isnan(z[0, 2]).all()


@pytest.mark.parametrize("C,offset", [(1024, 0), (1024, 8), (1024, 4), (1024, 1), (333, 0)])
def test_strides_alignment_and_neighbours(C, offset):
    """Column slices at any alignment, rows that are apart, a result in place; nothing beside it is written."""
    wide = _rand((2, 9, C + 24), torch.bfloat16, 20)
    keep = wide.clone()
    x = wide[:, 1:8, offset:offset + C]
    y = _rand((2, 7, C + 3), torch.bfloat16, 21)[..., :C]
    o = _options(2, 7, C, torch.bfloat16, "batch", "layer", None)
    o["eps"] = 1e-5
    wh, hm, wz, zm = _want(x, y, o)
    h, z = gated_residual_norm(x, y, out_residual=x, **o)
    assert h is x
    _within(h, wh, hm, "hidden")
    _within(z, wz, zm, "normed")
    mask = torch.ones_like(wide, dtype=torch.bool)
    mask[:, 1:8, offset:offset + C] = False
    assert torch.equal(wide[mask], keep[mask])


def test_no_rows():
    x = torch.empty(2, 0, 64, device="cuda")
    h, z = gated_residual_norm(x, x.clone())
    assert h.shape == z.shape == (2, 0, 64)


def rounded_e4m3(z, s):
    """z / s rounded to e4m3 by the type's definition, times s (64 bits)."""
    y = z / s
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp_min(-6) - 3)
    return torch.round(y / step) * step * s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,s,C", [(1, 1, 16), (2, 37, 1152), (1, 300, 5120), (2, 5, 1296), (1, 3, 6400)])
def test_quantised_rows(B, s, C, dtype):
    """The e4m3 rows stand for the normed values: half a step of the value's power of two, or of the smallest normal's
    where it is below, and what fp32 is off."""
    x, y = _rand((B, s, C), dtype, 22), _rand((B, s, C), dtype, 23)
    o = _options(B, s, C, torch.float32, "batch", "layer", None)
    o["eps"] = 1e-6
    h, rows = gated_residual_norm(x, y, quantize=True, **o)
    wh, hm, wz, zm = _want(x, y, o)
    _within(h, wh, hm, "hidden")
    assert isinstance(rows, Fp8Rows) and rows.shape == (B, s, C) and rows.scale.shape == (B * s, -(-C // 128))
    wz, zm = wz.reshape(B * s, C), zm.reshape(B * s, C)
    sc = rows.scale.double()
    assert torch.equal(torch.exp2(torch.log2(sc).round()), sc)  # powers of two
    pad = torch.nn.functional.pad(wz, (0, -C % 128)).view(B * s, -1, 128).abs().amax(-1)
    slack = 1 + 1e-5
    assert (pad <= 448 * sc * slack).all() and (pad * 2 * slack > 448 * sc).all()
    sx = sc.repeat_interleave(128, 1)[:, :C]
    got = rows.data.double() * sx
    half = torch.maximum(wz.abs() * 2.0 ** -4, sx * 2.0 ** -10)
    assert ((got - wz).abs() <= half * slack + 128 * U * zm).all()
    exact = got == rounded_e4m3(wz, sx)
    assert exact.double().mean() > 0.999  # all but those next to a tie


def test_captured_and_replayed():
    x, y = _rand((1, 64, 512), torch.bfloat16, 24), _rand((1, 64, 512), torch.bfloat16, 25)
    gate = _rand((1, 1, 512), torch.float32, 26)
    out = torch.empty_like(x)
    gated_residual_norm(x, y, gate=gate, out_residual=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, z = gated_residual_norm(x, y, gate=gate, out_residual=out)
    gate.mul_(2)
    y.copy_(_rand(y.shape, y.dtype, 27))
    g.replay()
    wh, hm, wz, zm = _want(x, y, dict(gate=gate, eps=1e-6))
    _within(h, wh, hm, "hidden")
    _within(z, wz, zm, "normed")
