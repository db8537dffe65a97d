"""Rotary positions with several axes against their definition in 64 bits.

Tolerance.  The kernel takes a pair's angle in 64 bits as turns and rounds the fraction to 32: half a spacing of a
value below 1 is 2^-25 half-turns, pi 2^-25 = 9.4e-8 radians; sincospi adds at most two units of 2^-24 (1.2e-7).  Two
products and a sum in fp32 add at most three roundings of 2^-24 of |a| + |b|.  Together below 4e-7 (|a| + |b|), and
half a spacing of the result's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from xdit_b200.rotary import RotaryEmbedding, rotary_embed  # noqa: E402


def _turned(x, e):
    """(rotated x in 64 bits, |a| + |b| of every element's pair) for x [B, H, s, D]."""
    B, _, s, D = x.shape
    axes = list(e.axes_dim)
    if e.grid is not None:
        n = torch.arange(s, device=x.device, dtype=torch.int64) + e.start
        pos, below, volume = [], 1, math.prod(e.grid)
        for side in reversed(e.grid):
            pos.insert(0, n // below % side)
            below *= side
        pos = (torch.stack(pos, -1) * (n < volume)[:, None])[None]
    else:
        pos = e.positions if e.positions.dim() == 3 else e.positions[None]
    n = sum(axes) // 2
    axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    if e.frequencies is not None:
        f = list(e.frequencies)
    elif e.ladder == "shared":
        f = [e.theta ** (-i / n) for i in range(n)]
    else:
        f = [e.theta ** (-2 * i / d) for d in axes for i in range(d // 2)]
    ang = (pos[..., axis].double() * torch.tensor(f, dtype=torch.float64, device=x.device))[:, None]
    x = x.double()
    a_at, b_at = (slice(0, n), slice(n, 2 * n)) if e.pairing == "halves" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    a, b = x[..., a_at], x[..., b_at]
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., a_at], y[..., b_at] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    mag[..., a_at] = mag[..., b_at] = a.abs() + b.abs()
    return y, mag


def _check(got, x, e):
    want, mag = _turned(x, e)
    f = torch.finfo(x.dtype)
    tol = 4e-7 * mag + (want.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)
    tol = torch.where(mag > 0, tol, torch.zeros_like(tol))  # elements behind the rotated part are copied
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol.clamp_min(1e-300)).max()):.3g} of the bound"


def _rand(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("axes,D,s,H,Hk", [((44, 42, 42), 128, 301, 5, 5), ((16, 56, 56), 128, 1, 40, 40),
                                           ((24, 24, 24), 72, 77, 3, 1), ((32, 40, 40), 128, 513, 8, 2),
                                           ((2,), 2, 9, 1, 1), ((6, 4), 13, 40, 3, 2), ((64,), 80, 33, 2, 0)])
def test_ids(axes, D, s, H, Hk, dtype, pairing):
    B = 2
    q = _rand((B, s, H, D), dtype, 1).transpose(1, 2)
    k = _rand((B, Hk, s, D), dtype, 2) if Hk else None
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-50, 2000, (B, s, len(axes)), device="cuda", generator=g)
    e = RotaryEmbedding(axes, positions=ids, pairing=pairing)
    before = q.clone()
    oq, ok = rotary_embed(q, k, e)
    assert oq.stride() == q.stride() and torch.equal(q, before)
    _check(oq, q, e)
    if Hk:
        _check(ok, k, e)
    else:
        assert ok is None


@pytest.mark.parametrize("grid,start,s", [((21, 45, 80), 0, 4001), ((21, 45, 80), 75600 - 100, 333), ((7,), 3, 11),
                                          ((3, 5), 0, 15), ((2, 3, 4, 5), 17, 200), ((1, 1, 1), 0, 5)])
def test_grid_walk_and_padding(grid, start, s):
    axes = {1: (32,), 2: (16, 16), 3: (12, 10, 10), 4: (8, 8, 8, 8)}[len(grid)]
    q, k = _rand((1, 3, s, 32), torch.bfloat16, 4), _rand((1, 3, s, 32), torch.bfloat16, 5)
    e = RotaryEmbedding(axes, grid=grid, start=start)
    oq, ok = rotary_embed(q, k, e)
    _check(oq, q, e)
    _check(ok, k, e)
    past = max(0, math.prod(grid) - start)
    assert torch.equal(oq[:, :, past:], q[:, :, past:])  # tokens behind the grid are not rotated


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("ladder", ["axis", "shared"])
def test_far_positions_and_fractions(kind, ladder):
    q = _rand((1, 2, 64, 64), torch.float32, 6)
    g = torch.Generator(device="cuda").manual_seed(7)
    ids = torch.randint(0, 1 << 24, (64, 2), device="cuda", generator=g)
    ids = (ids.float() / 8 if kind == torch.float32 else ids.to(kind))
    e = RotaryEmbedding((32, 32), positions=ids, theta=1e6, ladder=ladder)
    _check(rotary_embed(q, None, e)[0], q, e)


def test_frequencies_of_the_caller_and_zero_positions():
    q = _rand((2, 2, 5, 16), torch.float32, 8)
    e = RotaryEmbedding((8, 8), positions=torch.randint(0, 9, (1, 5, 2), device="cuda"),
                        frequencies=[0.0, 1.0, 3.5, -2.0, 1e-9, 0.3, 7.0, 0.001])
    _check(rotary_embed(q, None, e)[0], q, e)
    e = RotaryEmbedding((8, 8), positions=torch.zeros(5, 2, dtype=torch.int32, device="cuda"))
    assert torch.equal(rotary_embed(q, None, e)[0], q)


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 3), (4, 4), (8, 8), (2, 6)])
def test_strides_alignment_and_neighbours(offset, pad):
    """Column slices of a fused projection at any alignment; nothing beside the outputs is written."""
    B, s, H, D = 2, 21, 3, 24
    wide = _rand((B, s, H * D + offset + pad), torch.bfloat16, 9)
    q = wide[..., offset:offset + H * D].unflatten(2, (H, D)).transpose(1, 2)
    buf = torch.full((B, s + 2, H, D + offset + pad), float("nan"), dtype=q.dtype, device="cuda")
    out = buf[:, 1:-1, :, offset:offset + D].transpose(1, 2)
    e = RotaryEmbedding((8, 8, 8), grid=(3, 3, 3), pairing="halves" if offset == 2 else "interleaved")
    rotary_embed(q, None, e, out_query=out)
    _check(out, q, e)
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[:, 1:-1, :, offset:offset + D] = False
    assert torch.isnan(buf[mask]).all()


def test_in_place_empty_and_nan():
    q, k = _rand((1, 4, 50, 64), torch.float16, 10), _rand((1, 4, 50, 64), torch.float16, 11)
    e = RotaryEmbedding((32, 32), grid=(5, 10))
    want = rotary_embed(q, k, e)
    a, b = q.clone(), k.clone()
    assert rotary_embed(a, b, e, out_query=a, out_key=b) == (a, b)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    none = rotary_embed(q[:, :, :0], k[:, :, :0], e)
    assert none[0].shape == (1, 4, 0, 64)
    q[0, 1, 7, 5] = float("nan")  # only its pair takes it
    got = rotary_embed(q, None, e)[0]
    assert torch.isnan(got).nonzero().tolist() == [[0, 1, 7, 4], [0, 1, 7, 5]]


def test_offsets_past_32_bits():
    """Rows of a tensor whose elements reach beyond 2^31."""
    s, row = 3, 1 << 30
    base = torch.empty(s * row + 64, dtype=torch.bfloat16, device="cuda")
    q = base.as_strided((1, 1, s, 64), (0, 0, row, 1))
    q.copy_(_rand((1, 1, s, 64), torch.bfloat16, 12))
    e = RotaryEmbedding((32, 32), positions=torch.tensor([[5, 6], [700, 8], [9, 1000]], device="cuda"))
    got = rotary_embed(q, None, e, out_query=q.clone(memory_format=torch.contiguous_format))[0]
    _check(got, q, e)


def test_tables_are_what_the_prologue_takes():
    """The tables through the fused prologue give what rotary_embed gives on the same values."""
    from xdit_b200.prologue import qk_norm_rope_heads

    B, s, H, D = 2, 130, 4, 128
    x = [_rand((B, s, H * D), torch.bfloat16, 20 + i) for i in range(3)]
    e = RotaryEmbedding((44, 42, 42), grid=(2, 8, 8))
    q, k, v = qk_norm_rope_heads(*x, H, rotary_emb=e)
    heads = [t.view(B, s, H, D).transpose(1, 2) for t in x]
    _check(q, heads[0], e)
    _check(k, heads[1], e)
    assert torch.equal(v, heads[2])


def test_captured_and_replayed_on_another_stream():
    q, k = _rand((1, 4, 200, 64), torch.bfloat16, 30), _rand((1, 2, 200, 64), torch.bfloat16, 31)
    ids = torch.randint(0, 300, (200, 2), device="cuda")
    e = RotaryEmbedding((32, 32), positions=ids)
    oq, ok = torch.empty_like(q), torch.empty_like(k)
    rotary_embed(q, k, e, out_query=oq, out_key=ok)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rotary_embed(q, k, e, out_query=oq, out_key=ok)
    q.copy_(_rand(q.shape, q.dtype, 32))
    ids.add_(11)  # read at replay
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g.replay()
    torch.cuda.current_stream().wait_stream(s)
    _check(oq, q, e)
    _check(ok, k, e)
