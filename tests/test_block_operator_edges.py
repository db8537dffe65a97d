"""Calls at the edges of the operators around a DiT block's attention: no tokens, outputs that lie on inputs, parameters that
nothing would read."""
import ctypes

import pytest
import torch

from xdit_b200 import _capi


@pytest.fixture(scope="module")
def lib():
    from xdit_b200 import build

    build.build()
    return _capi.load()


F, AXIS = (ctypes.c_double * 8)(), (ctypes.c_uint8 * 8)()
PAIR = ctypes.c_int64 * 2


def _rotary(lib, **kw):
    """``xdit_rotary_axes`` on made-up addresses: what gets past the refusals ends at the missing device."""
    pos = dict(kind=0, axes=1, pairs=8, frequencies=F, axis=AXIS)
    pos.update({k[4:]: kw.pop(k) for k in list(kw) if k.startswith("pos_")})
    p = _capi.RotaryParams(dtype=0, B=1, H=2, Hk=0, s=4, D=16, q=1 << 20, out_q=2 << 20, stride_h=PAIR(64, 64), stride_row=PAIR(16, 16),
                           out_stride_h=PAIR(64, 64), out_stride_row=PAIR(16, 16), pos=_capi.RotaryPositions(**pos))
    p.pos.grid[0] = 4
    for k, v in kw.items():
        setattr(p, k, v)
    return lib.xdit_rotary_axes(ctypes.byref(p), None)


def _norm(lib, **kw):
    p = _capi.NormParams(dtype=0, B=1, s=2, C=32, norm=1, residual=1 << 20, out=2 << 20, residual_stride_row=32, out_stride_row=32)
    for k, v in kw.items():
        setattr(p, k, v)
    return lib.xdit_gated_residual_norm(ctypes.byref(p), None)


def test_no_tokens_at_the_c_entries(lib):
    """An empty tensor's address is NULL: a call without tokens has nothing to read there."""
    empty = dict(q=None, out_q=None)
    for kind in (0, 1, 2, 3):
        assert _rotary(lib, pos_kind=kind, s=0, **empty) == 0 and _rotary(lib, pos_kind=kind, B=0, **empty) == 0
        pos = _capi.RotaryPositions(kind=kind, axes=1, pairs=8, frequencies=F, axis=AXIS)
        pos.grid[0] = 4
        assert lib.xdit_rotary_tables(ctypes.byref(pos), None, None, 0, 16, None) == 0
    for n in (dict(s=0), dict(B=0)):
        assert _norm(lib, norm=0, residual=None, branch=None, out_residual=None, out=None, **n) == 0
        assert _norm(lib, norm=1, residual=None, branch=None, out_residual=None, out=None, **n) == 0
    # with tokens the same addresses are refused
    assert _rotary(lib, pos_kind=2) == -1 and _norm(lib, norm=0, branch=None, out=None) == -2


@pytest.mark.gpu
def test_no_tokens():
    from xdit_b200.modulation import gated_residual_norm
    from xdit_b200.rotary import RotaryEmbedding, rotary_embed

    for B, s in ((2, 0), (0, 3)):
        q, k = (torch.empty(B, h, s, 32, device="cuda") for h in (4, 2))
        for positions in (torch.empty(s, 2, dtype=torch.int64, device="cuda"), torch.empty(B, s, 2, device="cuda")):
            a, b = rotary_embed(q, k, RotaryEmbedding((16, 16), positions=positions))
            assert a.shape == q.shape and b.shape == k.shape
        x = torch.empty(B, s, 64, device="cuda")
        h, z = gated_residual_norm(x, x.clone(), norm=None)
        assert h.shape == x.shape and z is None
        gate = torch.ones(64, device="cuda")
        h, z = gated_residual_norm(x, x.clone(), gate=gate, norm="rms", quantize=True)
        assert h.shape == x.shape and z.shape == x.shape
    cos, sin = RotaryEmbedding((16, 16), positions=torch.empty(0, 2, dtype=torch.int32, device="cuda")).tables(0, 32, "cuda")
    assert cos.shape == sin.shape == (0, 32)
