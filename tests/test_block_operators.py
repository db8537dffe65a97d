"""Refusals of the operators around a DiT block's attention (rotary axes, gated residual norm, fp8 linear), which
need no GPU: shapes, types, strides and combinations are looked at before anything is launched."""
import ctypes
import os
import subprocess

import pytest
import torch

from xdit_b200 import _capi, ops
from xdit_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear, quantize_rows, quantize_weight
from xdit_b200.modulation import gated_residual_norm
from xdit_b200.rotary import RotaryEmbedding, rotary_embed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from xdit_b200 import build

    build.build()
    return _capi.load()


def test_structs_have_the_header_s_layout(tmp_path):
    names = ["xdit_rotary_positions", "xdit_rotary_params", "xdit_row_vec", "xdit_norm_params", "xdit_fp8_linear_params"]
    mirrors = [_capi.RotaryPositions, _capi.RotaryParams, _capi.RowVec, _capi.NormParams, _capi.Fp8LinearParams]
    lines, want = [], []
    for n, m in zip(names, mirrors):
        lines.append(f'printf("%zu\\n", sizeof(struct {n}));')
        want.append(ctypes.sizeof(m))
        for field, _ in m._fields_:
            lines.append(f'printf("%zu\\n", offsetof(struct {n}, {field}));')
            want.append(getattr(m, field).offset)
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "xdit_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n"
    (tmp_path / "probe.c").write_text(src)
    exe = str(tmp_path / "probe")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "probe.c"), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


# ---- rotary ---------------------------------------------------------------------------------------
Q = torch.zeros(2, 3, 5, 16)


@pytest.mark.parametrize("kw,error", [
    (dict(axes_dim=(8, 7), grid=(1, 5)), ValueError), (dict(axes_dim=(), grid=()), ValueError),
    (dict(axes_dim=(2,) * 5, grid=(1,) * 5), ValueError), (dict(axes_dim=(8, 8)), ValueError),
    (dict(axes_dim=(8, 8), grid=(1, 5), positions=torch.zeros(5, 2, dtype=torch.int32)), ValueError),
    (dict(axes_dim=(8, 8), grid=(5,)), ValueError), (dict(axes_dim=(8, 8), grid=(1, 5), pairing="thirds"), ValueError),
    (dict(axes_dim=(8, 8), grid=(1, 5), ladder="rope"), ValueError), (dict(axes_dim=(0, 0), grid=(1, 5)), ValueError),
    (dict(axes_dim=(8, 8), grid=(1, 5), frequencies=[1.0] * 7), ValueError),
    (dict(axes_dim=(8, 8), positions=torch.zeros(5, 3, dtype=torch.int32)), ValueError),
    (dict(axes_dim=(8, 8), positions=torch.zeros(4, 2, dtype=torch.int32)), ValueError),
    (dict(axes_dim=(8, 8), positions=torch.zeros(3, 5, 2, dtype=torch.int32)), ValueError),
    (dict(axes_dim=(8, 8), positions=torch.zeros(5, 2, dtype=torch.float64)), TypeError),
    (dict(axes_dim=(8, 10), grid=(1, 5)), ValueError)])
def test_rotary_refuses(kw, error):
    with pytest.raises(error):
        rotary_embed(Q, None, RotaryEmbedding(**kw))


def test_rotary_refuses_tensors():
    e = RotaryEmbedding((8, 8), grid=(1, 5))
    for q, k in ((Q[0], None), (Q, torch.zeros(2, 3, 6, 16)), (Q, torch.zeros(1, 3, 5, 16)), (Q, torch.zeros(2, 3, 5, 18)),
                 (Q.transpose(2, 3).contiguous().transpose(2, 3), None)):
        with pytest.raises(ValueError):
            rotary_embed(q, k, e)
    with pytest.raises(TypeError):
        rotary_embed(Q, Q.half(), e)
    with pytest.raises(TypeError):
        rotary_embed(Q.double(), None, e)
    with pytest.raises(ValueError):
        rotary_embed(Q, None, e, out_query=torch.zeros(2, 3, 5, 8))
    with pytest.raises(ValueError):
        rotary_embed(Q, None, e, out_key=Q)
    with pytest.raises(NotImplementedError, match="backward"):
        rotary_embed(Q.clone().requires_grad_(), None, e)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary_embed(Q, Q, e)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        e.tables(5, 16, "cpu")
    with pytest.raises(ValueError):
        RotaryEmbedding((8, 8), grid=(1, 5), pairing="halves").tables(5, 16, "cuda")
    with pytest.raises(ValueError):
        e.tables(5, 8, "cuda")


def test_rotary_c_entry_refuses(lib):
    f, a = (ctypes.c_double * 8)(), (ctypes.c_uint8 * 8)()

    def call(**kw):
        pos = dict(kind=0, axes=1, pairs=8, frequencies=f, axis=a)
        pos.update({k[4:]: kw.pop(k) for k in list(kw) if k.startswith("pos_")})
        grid = pos.pop("grid", 4)
        p = _capi.RotaryParams(dtype=0, B=1, H=1, Hk=0, s=4, D=16, q=16, out_q=16, pos=_capi.RotaryPositions(**pos))
        p.pos.grid[0] = grid
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_rotary_axes(ctypes.byref(p), None)

    assert lib.xdit_rotary_axes(None, None) == -1
    assert call(dtype=9) == -4 and call(pos_kind=7) == -4
    assert call(q=None) == -1 and call(Hk=1) == -1 and call(pos_kind=2) == -1
    assert call(D=14) == -2 and call(H=0) == -2 and call(s=-1) == -2 and call(pos_pairs=0) == -2 and call(pos_axes=5) == -2
    assert call(pos_grid=0) == -2 and call(pos_start=-1) == -2
    a[3] = 1
    assert call() == -2  # a pair on an axis that is not there
    a[3] = 0
    assert call(s=0) == 0 and call(B=0) == 0
    assert lib.xdit_rotary_tables(None, None, None, 4, 16, None) == -1


# ---- gated residual norm ----------------------------------------------------------------------------
X = torch.zeros(2, 3, 32)


@pytest.mark.parametrize("kw,error", [
    (dict(norm="batch"), ValueError), (dict(post_norm="rms"), ValueError), (dict(gate=torch.zeros(32)), ValueError),
    (dict(norm=None), ValueError), (dict(branch=X, norm=None, scale=torch.zeros(32)), ValueError),
    (dict(branch=X, post_weight=torch.ones(32)), ValueError), (dict(branch=X[:, :2]), ValueError),
    (dict(branch=X.half()), TypeError), (dict(branch=X, gate=torch.zeros(31)), ValueError),
    (dict(branch=X, gate=torch.zeros(3, 32)), ValueError), (dict(branch=X, gate=torch.zeros(2, 2, 32)), ValueError),
    (dict(branch=X, gate=torch.zeros(1, 1, 1, 32)), ValueError), (dict(scale=torch.zeros(32).half()), TypeError),
    (dict(scale=torch.zeros(32, 2)[:, 0]), ValueError), (dict(weight=torch.zeros(2, 1, 32)), ValueError),
    (dict(out_residual=X), ValueError), (dict(branch=X, norm=None, quantize=True), ValueError)])
def test_norm_refuses(kw, error):
    with pytest.raises(error):
        gated_residual_norm(X, **kw)


def test_norm_refuses_tensors():
    with pytest.raises(ValueError):
        gated_residual_norm(X[0])
    with pytest.raises(ValueError):
        gated_residual_norm(X.transpose(1, 2))
    with pytest.raises(ValueError, match="multiple of 16"):
        gated_residual_norm(torch.zeros(1, 2, 24), quantize=True)
    with pytest.raises(TypeError):
        gated_residual_norm(X.double())
    with pytest.raises(NotImplementedError, match="backward"):
        gated_residual_norm(X, weight=torch.ones(32, requires_grad=True))
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
        gated_residual_norm(X, weight=torch.ones(32, requires_grad=True))


def test_norm_c_entry_refuses(lib):
    def call(**kw):
        p = _capi.NormParams(dtype=0, B=1, s=2, C=32, norm=1, residual=16, out=16)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_gated_residual_norm(ctypes.byref(p), None)

    assert lib.xdit_gated_residual_norm(None, None) == -1
    assert call(dtype=3) == -4 and call(norm=3) == -4 and call(post_norm=-1) == -4
    assert call(C=0) == -2 and call(C=16385) == -2 and call(B=-1) == -2 and call(norm=0) == -2
    assert call(B=65536, s=65536) == -2
    assert call(residual=None) == -1 and call(out=None) == -1 and call(branch=16) == -1 and call(out_q=16) == -1
    assert call(scale=_capi.RowVec(ptr=16, dtype=1)) == -4
    q = dict(out=None, out_q=16, out_scale=16, out_scale_ld=2)
    assert call(**q, C=24) == -3 and call(**q, residual=18) == -3 and call(**{**q, "out_scale_ld": 1}) == -3
    assert call(s=0) == 0


# ---- fp8 linear ---------------------------------------------------------------------------------------
def _rows(M=3, K=256, data=E4, scale=torch.float32):
    return Fp8Rows(torch.zeros(M, K).to(data), torch.ones(M, -(-K // 128), dtype=scale))


def _weight(N=48, K=256):
    return Fp8Weight(torch.zeros(N, K).to(E4), torch.ones(-(-N // 128), -(-K // 128)))


@pytest.mark.parametrize("x,w,kw,error", [
    (_rows(data=torch.bfloat16), _weight(), {}, TypeError), (_rows(scale=torch.float16), _weight(), {}, TypeError),
    (_rows(K=272), _weight(), {}, ValueError), (_rows(K=24), _weight(K=24), {}, ValueError),
    (Fp8Rows(torch.zeros(3, 256).to(E4), torch.ones(3, 1)), _weight(), {}, ValueError),
    (_rows(), Fp8Weight(torch.zeros(300, 256).to(E4), torch.ones(2, 2)), {}, ValueError),
    (_rows(), _weight(), dict(activation="relu"), ValueError), (_rows(), _weight(), dict(bias=torch.zeros(47)), ValueError),
    (_rows(), _weight(), dict(bias=torch.zeros(48, 2)[:, 0]), ValueError),
    (_rows(), _weight(), dict(bias=torch.zeros(48, dtype=torch.float64)), TypeError),
    (_rows(), _weight(N=40), dict(quantize_out=True), ValueError), (_rows(), _weight(), dict(out_dtype=torch.float64), TypeError),
    (Fp8Rows(torch.zeros(256, 3).to(E4).t(), torch.ones(3, 2)), _weight(), {}, ValueError)])
def test_linear_refuses(x, w, kw, error):
    with pytest.raises(error):
        fp8_linear(x, w, **kw)


def test_linear_refuses_tensors():
    with pytest.raises(NotImplementedError, match="backward"):
        fp8_linear(_rows(), _weight(), torch.zeros(48, requires_grad=True))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fp8_linear(_rows(), _weight())
    for x, error in ((torch.zeros(2, 24), ValueError), (torch.zeros(2, 32, dtype=torch.float64), TypeError),
                     (torch.zeros(32, 2).t(), ValueError), (torch.zeros(2, 32), RuntimeError),
                     (torch.zeros(2, 32, requires_grad=True), NotImplementedError)):
        with pytest.raises(error):
            quantize_rows(x)
    for w, error in ((torch.zeros(2, 3, 32), ValueError), (torch.zeros(2, 24), ValueError), (torch.zeros(0, 32), ValueError),
                     (torch.zeros(2, 32, dtype=torch.int8), TypeError), (torch.zeros(2, 32), RuntimeError)):
        with pytest.raises(error):
            quantize_weight(w)


def test_linear_c_entry_refuses(lib):
    def call(**kw):
        p = _capi.Fp8LinearParams(M=2, N=16, K=128, x=16, w=16, x_stride_row=128, w_stride_row=128, x_scale=16, w_scale=16,
                                  out=16, out_stride_row=16)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_fp8_linear(ctypes.byref(p), None)

    assert lib.xdit_fp8_linear(None, None) == -1
    assert call(K=0) == -2 and call(K=120) == -2 and call(N=0) == -2 and call(M=-1) == -2
    assert call(activation=2) == -4 and call(out_dtype=3) == -4 and call(bias=16, bias_dtype=7) == -4
    assert call(x=None) == -1 and call(out=None) == -1 and call(w_scale=None) == -1 and call(out_q=16) == -1
    assert call(x=8) == -3 and call(x_stride_row=136) == -3 and call(w_stride_row=112) == -3 and call(out=17) == -3
    assert call(out_stride_row=15) == -3 and call(out_q=16, out_scale=16, out_scale_ld=1) == -3
    word = ctypes.c_int32(5)
    assert call(status_host=ctypes.addressof(word)) == -6
    assert call(M=0) == 0
    assert lib.xdit_quantize_rows(16, 0, 0, 0, 1, 1, 24, 16, 16, 1, None) == -2
    assert lib.xdit_quantize_rows(24, 0, 0, 0, 1, 1, 32, 16, 16, 1, None) == -3
    assert lib.xdit_quantize_rows(None, 0, 0, 0, 1, 1, 32, 16, 16, 1, None) == -1
    assert lib.xdit_quantize_weight(16, 32, 0, 0, 32, 16, 16, None) == -2
    assert lib.xdit_quantize_weight(16, 36, 0, 2, 32, 16, 16, None) == -3


# ---- outputs that could not take the result, sizes that 32 bits would take for others --------------------------------
def test_e4m3_outputs_are_looked_at():
    x, w = _rows(), _weight()
    good_q, good_s = ops.empty_fp8_rows(3, 48, "cpu")
    bad = [(torch.zeros(3, 48, dtype=torch.uint8), good_s, TypeError), (good_q, None, TypeError), (good_q, good_s.half(), TypeError),
           (good_q[:2], good_s, ValueError), (good_q, good_s[:2], ValueError), (good_q, torch.ones(3, 2), ValueError),
           (torch.zeros(3, 64).to(E4)[:, :48], good_s, ValueError)]
    for q, s, error in bad:
        with pytest.raises(error):
            ops.fp8_linear(x.data, x.scale, w.data, w.scale, out_q=q, out_scale=s)
        with pytest.raises(error):
            ops.gated_residual_norm(torch.zeros(1, 3, 48), None, out_q=q, out_scale=s, norm="rms")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.fp8_linear(x.data, x.scale, w.data, w.scale, out_q=good_q, out_scale=good_s)


def test_sizes_beyond_32_bits_are_refused():
    """Each of these would be a call of five rows if its size were cut to 32 bits."""
    many = 2 ** 32 + 5
    row = torch.zeros(16)
    q = row.expand(1, 1, many, 16)
    e = RotaryEmbedding((8, 8), grid=(1, 5))
    with pytest.raises(ValueError, match="above"):
        ops.rotary_axes(q, None, e._params(1, many), False, q, None)
    with pytest.raises(ValueError, match="above"):
        ops.rotary_axes(q.transpose(1, 2), None, e._params(1, 1), False, q.transpose(1, 2), None)
    with pytest.raises(ValueError, match="above"):
        ops.rotary_tables(e._params(1, many), many, 16, "cuda")
    for x in (row.expand(1, many, 16), row.expand(2 ** 16, 2 ** 16 + 1, 16)):
        with pytest.raises(ValueError, match="above"):
            ops.gated_residual_norm(x, None, out=x, norm="rms")
        with pytest.raises(ValueError, match="above"):
            ops.fp8_linear(x, None, _weight(K=16).data, _weight(K=16).scale, out=row.expand(x.shape[0] * x.shape[1], 16))
    with pytest.raises(ValueError, match="above"):
        ops.quantize_rows(row.expand(1, many, 16))
    with pytest.raises(ValueError, match="above"):
        ops.quantize_weight(row.expand(many, 16))


def test_c_entries_refuse_outputs_in_one_place_and_pointers_between_elements(lib):
    f, a = (ctypes.c_double * 8)(), (ctypes.c_uint8 * 8)()
    pair = ctypes.c_int64 * 2

    def rotary(**kw):
        p = _capi.RotaryParams(dtype=0, B=1, H=2, Hk=0, s=4, D=16, q=16, out_q=16, stride_h=pair(64, 64), stride_row=pair(16, 16),
                               out_stride_h=pair(64, 64), out_stride_row=pair(16, 16),
                               pos=_capi.RotaryPositions(kind=0, axes=1, pairs=8, frequencies=f, axis=a))
        p.pos.grid[0] = 4
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_rotary_axes(ctypes.byref(p), None)

    assert rotary(out_stride_h=pair(0, 0)) == -2 and rotary(out_stride_row=pair(0, 0)) == -2 and rotary(B=2) == -2
    assert rotary(Hk=2, k=32, out_k=16) == -2 and rotary(Hk=2, k=32, out_k=48, out_stride_row=pair(16, 0)) == -2
    assert rotary(out_q=17) == -3

    def norm(**kw):
        p = _capi.NormParams(dtype=0, B=1, s=2, C=32, norm=1, residual=16, out=16, residual_stride_row=32, out_stride_row=32)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_gated_residual_norm(ctypes.byref(p), None)

    both = dict(branch=16, branch_stride_row=32, out_residual=64, out_residual_stride_row=32)
    assert norm(out_stride_row=0) == -2 and norm(B=2) == -2 and norm(**{**both, "out_residual_stride_row": 0}) == -2
    assert norm(**{**both, "out_residual": 16}) == -2
    assert norm(residual=17) == -3 and norm(out=17) == -3 and norm(scale=_capi.RowVec(ptr=18, dtype=2)) == -3

    def linear(**kw):
        p = _capi.Fp8LinearParams(M=2, N=16, K=128, x=16, w=16, x_stride_row=128, w_stride_row=128, x_scale=16, w_scale=16,
                                  out=16, out_stride_row=16)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.xdit_fp8_linear(ctypes.byref(p), None)

    assert linear(x_scale=18) == -3 and linear(w_scale=17) == -3 and linear(bias=17, bias_dtype=0) == -3


def test_packed_parameters_are_the_structures_bytes():
    f, a = (ctypes.c_double * 8)(), (ctypes.c_uint8 * 8)()
    pos = _capi.RotaryPositions(2, 3, 8, f, a, 123456, 7, 8, 9, (5, 6, 7, 8), 11)
    pair = ctypes.c_int64 * 2
    want = _capi.RotaryParams(2, 3, 4, 5, 6, 7, True, pos, 2 ** 63 + 1, 12, 13, 0, *(pair(i, -i) for i in range(6)))
    got = _capi.pack_rotary(2, 3, 4, 5, 6, 7, True, bytes(pos), 2 ** 63 + 1, 12, 13, 0, *(j for i in range(6) for j in (i, -i)))
    assert got == bytes(want)
    rows = [(1000 + i, i, 2 * i, i % 3) for i in range(7)]
    head = (1, 2, 3, 4, 2, 1, 0.75, 1e-6, *range(20, 35))
    assert _capi.pack_norm(*head, *(v for r in rows for v in r)) == bytes(_capi.NormParams(*head, *rows))
    n = len(_capi.Fp8LinearParams._fields_)
    assert _capi.pack_fp8_linear(*range(n)) == bytes(_capi.Fp8LinearParams(*range(n)))
    with pytest.raises(Exception):
        _capi.pack_fp8_linear(2 ** 32 + 5, *range(1, n))
