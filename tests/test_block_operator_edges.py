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
    """``xdit_rotary_axes`` on made-up addresses, one of them between two elements: no call gets past that refusal (-3)."""
    pos = dict(kind=0, axes=1, pairs=8, frequencies=F, axis=AXIS)
    pos.update({k[4:]: kw.pop(k) for k in list(kw) if k.startswith("pos_")})
    p = _capi.RotaryParams(dtype=0, B=1, H=2, Hk=0, s=4, D=16, q=(1 << 20) + 1, out_q=2 << 20, stride_h=PAIR(64, 64), stride_row=PAIR(16, 16),
                           out_stride_h=PAIR(64, 64), out_stride_row=PAIR(16, 16), pos=_capi.RotaryPositions(**pos))
    p.pos.grid[0] = 4
    for k, v in kw.items():
        setattr(p, k, v)
    return lib.xdit_rotary_axes(ctypes.byref(p), None)


def _norm(lib, **kw):
    """``xdit_gated_residual_norm`` in the same way."""
    p = _capi.NormParams(dtype=0, B=1, s=2, C=32, norm=1, residual=(1 << 20) + 1, out=2 << 20, residual_stride_row=32, out_stride_row=32)
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


# ---- parameters that nothing would read, results that nothing would write ---------------------------------------------
BRANCH = dict(branch=3 << 20, branch_stride_row=32, out_residual=4 << 20, out_residual_stride_row=32)
ROW = _capi.RowVec(ptr=5 << 20, dtype=0)


def test_norm_c_entry_refuses_what_it_would_not_use(lib):
    """Without a norm there is no second result to write, and no row that only the norm takes is read; the same holds for the
    post norm and for the branch."""
    past = -3  # the answer of a call that is refused for its address alone
    assert _norm(lib, **BRANCH) == past
    alone = {**BRANCH, "norm": 0, "out": None}
    assert _norm(lib, **alone) == past
    assert _norm(lib, **{**alone, "out": 2 << 20, "out_stride_row": 32}) == -2
    assert _norm(lib, **alone, out_q=6 << 20, out_scale=7 << 20, out_scale_ld=2) == -2
    for row in ("weight", "bias", "scale", "shift"):
        assert _norm(lib, **alone, **{row: ROW}) == -2
        assert _norm(lib, **BRANCH, **{row: ROW}) == past
    for row in ("post_weight", "post_bias"):
        assert _norm(lib, **BRANCH, **{row: ROW}) == -2
        assert _norm(lib, **BRANCH, post_norm=2, **{row: ROW}) == past
        assert _norm(lib, post_norm=2, **{row: ROW}) == -2
    assert _norm(lib, gate=ROW) == -2 and _norm(lib, post_norm=1) == -2
    assert _norm(lib, **BRANCH, gate=ROW) == past


def test_ops_norm_refuses_a_second_result_without_a_norm():
    from xdit_b200 import ops

    x = torch.zeros(1, 3, 32)
    q, s = ops.empty_fp8_rows(3, 32, "cpu")
    for kw in (dict(out=torch.empty_like(x)), dict(out_q=q, out_scale=s)):
        with pytest.raises(ValueError, match="norm"):
            ops.gated_residual_norm(x, x.clone(), out_residual=torch.empty_like(x), **kw)


# ---- outputs that lie on inputs ------------------------------------------------------------------------------------------
def test_rotary_refuses_outputs_on_the_other_input_or_with_other_strides(lib):
    """In place means each output in its own input, element by element: CTAs of q and of k run at the same time, and so do the
    tokens of one."""
    q, k, past = (1 << 20) + 1, 3 << 20, -3
    both = dict(Hk=2, k=k, out_k=4 << 20)
    assert _rotary(lib, **both) == past
    assert _rotary(lib, **{**both, "out_k": k}) == past and _rotary(lib, out_q=q) == past  # in place
    assert _rotary(lib, **{**both, "out_q": k}) == -2 and _rotary(lib, **{**both, "out_k": q}) == -2
    assert _rotary(lib, **{**both, "out_q": k, "out_k": q}) == -2
    for strides in (dict(out_stride_row=PAIR(32, 16)), dict(out_stride_h=PAIR(128, 64)), dict(B=2, out_stride_b=PAIR(256, 256), stride_b=PAIR(128, 128))):
        assert _rotary(lib, out_q=q, **strides) == -2 and _rotary(lib, **strides) == past
    for strides in (dict(out_stride_row=PAIR(16, 32)), dict(out_stride_h=PAIR(64, 128))):
        assert _rotary(lib, **{**both, "out_k": k}, **strides) == -2 and _rotary(lib, **both, **strides) == past
    # a stride that no step takes may be any
    assert _rotary(lib, out_q=q, s=1, out_stride_row=PAIR(32, 16)) == past and _rotary(lib, out_q=q, H=1, out_stride_h=PAIR(1, 1)) == past


@pytest.mark.gpu
def test_rotary_in_place_and_in_refused_places():
    from xdit_b200._capi import XditError
    from xdit_b200.rotary import RotaryEmbedding, rotary_embed

    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(2, 3, 40, 32, device="cuda", generator=g) for _ in range(2))
    e = RotaryEmbedding((16, 16), grid=(5, 8))
    a, b = rotary_embed(q, k, e)
    kept = q.clone(), k.clone()
    with pytest.raises(XditError):
        rotary_embed(q, k, e, out_query=k, out_key=q)
    with pytest.raises(XditError):
        rotary_embed(q, q, e, out_query=q, out_key=k)
    assert torch.equal(q, kept[0]) and torch.equal(k, kept[1])
    rotary_embed(q, k, e, out_query=q, out_key=k)
    assert torch.equal(q, a) and torch.equal(k, b)


def test_norm_refuses_outputs_on_the_modulation_or_with_other_strides(lib):
    past, x = -3, (1 << 20) + 1
    h = dict(BRANCH)
    assert _norm(lib, **{**h, "out_residual": x}) == past and _norm(lib, **{**h, "out_residual": h["branch"]}) == past  # in place
    assert _norm(lib, out=x) == past
    for at in (x, h["branch"]):
        assert _norm(lib, **{**h, "out_residual": at, "out_residual_stride_row": 64}) == -2
        assert _norm(lib, **{**h, "out": at, "out_stride_row": 64}) == -2
        far = dict(B=2, residual_stride_b=64, branch_stride_b=64, out_residual_stride_b=128, out_stride_b=128)
        assert _norm(lib, **{**h, **far, "out_residual": at}) == -2 and _norm(lib, **{**h, **far, "out": at}) == -2
        assert _norm(lib, **{**h, "s": 1, "out_residual": at, "out_residual_stride_row": 64}) == past
    for row in ("gate", "weight", "bias", "scale", "shift", "post_weight", "post_bias"):
        rows = {**h, "post_norm": 1, row: ROW}
        assert _norm(lib, **rows) == past
        assert _norm(lib, **{**rows, "out_residual": ROW.ptr}) == -2 and _norm(lib, **rows, out=ROW.ptr) == -2


@pytest.mark.gpu
def test_norm_in_place_and_in_refused_places():
    from xdit_b200._capi import XditError
    from xdit_b200.modulation import gated_residual_norm

    g = torch.Generator(device="cuda").manual_seed(2)
    x, y, gate = (torch.randn(2, 5, 64, device="cuda", generator=g) for _ in range(3))
    h, z = gated_residual_norm(x, y, gate=gate)
    with pytest.raises(XditError):
        gated_residual_norm(x, y, gate=gate, out_residual=gate)
    for which in (0, 1):
        both = [x.clone(), y.clone()]
        h1, z1 = gated_residual_norm(*both, gate=gate, out_residual=both[which])
        assert h1 is both[which] and torch.equal(h1, h) and torch.equal(z1, z)


# ---- positions of the tables that the attention prologue takes ------------------------------------------------------------
def test_tables_look_at_their_positions(monkeypatch):
    """The kernel that rotates runs on the query's device and reads the tables there."""
    from xdit_b200 import ops
    from xdit_b200.rotary import RotaryEmbedding

    e = RotaryEmbedding((8, 8), positions=torch.zeros(5, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        e.tables(5, 16, "cuda")
    with pytest.raises(NotImplementedError, match="backward"):
        RotaryEmbedding((8, 8), positions=torch.zeros(5, 2, requires_grad=True)).tables(5, 16, "cuda")
    made = []
    monkeypatch.setattr(ops, "_check_tensors", lambda *t: None)  # (as if the positions were on a GPU)
    monkeypatch.setattr(ops, "rotary_tables", lambda p, s, D, device: made.append(device) or (None, None))
    with pytest.raises(ValueError, match="cuda:1"):
        e.tables(5, 16, "cuda:1")
    with pytest.raises(ValueError):
        e.tables(5, 16, torch.device("cuda", 0))
    e.tables(5, 16, "cpu")
    assert made == [torch.device("cpu")]


# ---- an embedding that does not fit, beside a stale-KV buffer ------------------------------------------------------------
@pytest.mark.parametrize("pairing", ["interleaved", "halves"])
@pytest.mark.parametrize("wrong", ["tokens", "head", "type", "pairing", "gradient"])
def test_a_refused_embedding_leaves_the_stale_buffers_alone(monkeypatch, pairing, wrong):
    """Keys that have been written but not rotated would be what the next steps attend to.  Interleaved pairs are rotated by
    tables in the prologue, halves behind it."""
    import xdit_b200
    from tests import fake_ops
    from xdit_b200 import cache_manager, ops
    from xdit_b200.prologue import attention_from_projections
    from xdit_b200.rotary import RotaryEmbedding

    def check(*tensors):  # (as on a GPU)
        if any(t.requires_grad for t in tensors):
            raise NotImplementedError

    fake_ops.install(monkeypatch)
    monkeypatch.setattr(ops, "_check_tensors", check)
    xdit_b200.init_sequence_parallel(1, 1)
    manager = cache_manager.CacheManager()
    manager.register_cache_entry("layer", "attn")
    monkeypatch.setattr(cache_manager, "get_cache_manager", lambda: manager)
    monkeypatch.setattr(cache_manager, "runtime_state_is_initialized", lambda: False)
    B, n, H, D = 2, 6, 2, 16
    entry = manager.cache["attn", "layer"]
    entry.k, entry.v = torch.ones(B, H, n + 2, D), torch.ones(B, H, n + 2, D)
    k, v = entry.k, entry.v
    ids = torch.zeros(n, 2) if pairing == "interleaved" else torch.zeros(B, n, 2)
    kw = dict(axes_dim=(8, 8), positions=ids, pairing=pairing)
    kw.update({"tokens": dict(positions=ids[..., 1:, :]), "head": dict(axes_dim=(12, 12)), "type": dict(positions=ids.double()),
               "pairing": dict(pairing="thirds"), "gradient": dict(positions=ids.clone().requires_grad_())}[wrong])
    x = torch.randn(B, n, H * D)
    error = {"type": TypeError, "gradient": NotImplementedError}.get(wrong, ValueError)
    with pytest.raises(error):
        attention_from_projections(x, x, x, H, rotary_emb=RotaryEmbedding(**kw), attn_layer="layer")
    assert entry.k is k and entry.v is v and (k == 1).all() and (v == 1).all()


# ---- gradients ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["hidden_states", "qkv_weight", "qkv_bias", "out_proj_weight", "out_proj_bias", "norm_q_weight"])
def test_attention_from_hidden_states_refuses_a_gradient(monkeypatch, which):
    """With 16- and 32-bit weights too: the projections would record it, and the attention between them would cut it."""
    import xdit_b200
    from tests import fake_ops
    from xdit_b200.prologue import attention_from_hidden_states

    fake_ops.install(monkeypatch)
    xdit_b200.init_sequence_parallel(1, 1)
    H, C = 2, 32
    kw = dict(hidden_states=torch.randn(1, 5, C), qkv_weight=torch.randn(3 * C, C), qkv_bias=torch.randn(3 * C),
              out_proj_weight=torch.randn(C, C), out_proj_bias=torch.randn(C), norm_q_weight=torch.ones(C),
              norm_k_weight=torch.ones(C))
    want = attention_from_hidden_states(heads=H, **kw)
    kw[which].requires_grad_()
    with pytest.raises(NotImplementedError, match="backward"):
        attention_from_hidden_states(heads=H, **kw)
    with torch.no_grad():
        assert torch.equal(attention_from_hidden_states(heads=H, **kw), want)


# ---- the norm's kernels -------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("C", [256 * i + d for i in (1, 2, 3, 4, 5) for d in (-8, 0, 8)] + [1024 * i + d for i in (2, 3, 4, 5) for d in (-8, 0, 8)]
                         + [8192, 8200, 12288, 12296, 16376])
def test_norm_at_both_ends_of_every_width_of_vectors(C):
    """Rows of 16-byte words at the ends of every number of vectors a thread, both results against 64 bits.  Tolerance: a sum
    of C values in a tree is off by less than 2^-24 (log2(C) + 40) of its magnitudes, the norm's other steps by ten roundings:
    128 of 2^-24 of the magnitudes of what a value is made of, and half a spacing of bf16."""
    from xdit_b200.modulation import gated_residual_norm

    g = torch.Generator(device="cuda").manual_seed(C)
    x, y = (torch.randn(1, 3, C, device="cuda", generator=g).bfloat16() for _ in range(2))
    gate, scale = (torch.randn(1, 1, C, device="cuda", generator=g) for _ in range(2))
    h, z = gated_residual_norm(x, y, gate=gate, scale=scale, norm="rms")
    wh = x.double() + gate.double() * y.double()
    r = 1 / torch.sqrt((wh * wh).mean(-1, keepdim=True) + 1e-6)
    wz = wh * r * (1 + scale.double())
    mag = x.double().abs() + (gate.double() * y.double()).abs()
    zmag = (mag * r + wh.abs() * r * (mag * mag).mean(-1, keepdim=True) * r * r) * (1 + scale.double().abs())
    for got, want, m in ((h, wh, mag), (z, wz, zmag)):
        assert ((got.double() - want).abs() <= 128 * 2.0 ** -24 * m + want.abs() * 2.0 ** -8).all()


# ---- e4m3 kernels: outputs in an input's place ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 200, 3000])
def test_e4m3_kernels_refuse_results_in_an_input_s_place(M):
    """Rows of x and of w are read for as long as any tile runs."""
    from xdit_b200 import ops
    from xdit_b200._capi import XditError
    from xdit_b200.fp8_linear import quantize_rows, quantize_weight

    g, K = torch.Generator(device="cuda").manual_seed(4), 1024
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    rows, w = quantize_rows(x), quantize_weight(torch.randn(K, K, device="cuda", generator=g))
    q, s = ops.empty_fp8_rows(M, K, "cuda")
    kept = [t.clone() for t in (rows.data.view(torch.uint8), rows.scale, w.data.view(torch.uint8), w.scale, x)]
    for data, scale in ((rows.data, s), (q, rows.scale), (w.data[:M], s) if M <= K else (rows.data, s)):
        with pytest.raises(XditError) as e:
            ops.fp8_linear(rows.data, rows.scale, w.data, w.scale, out_q=data, out_scale=scale)
        assert e.value.code == -2
    lib, scale = _capi.load(), s.data_ptr()
    assert lib.xdit_quantize_rows(x.data_ptr(), 0, K, 0, 1, M, K, x.data_ptr(), scale, M, None) == -2
    assert lib.xdit_quantize_weight(x.data_ptr(), K, 0, M, K, x.data_ptr(), scale, None) == -2
    torch.cuda.synchronize()
    for a, b in zip(kept, (rows.data.view(torch.uint8), rows.scale, w.data.view(torch.uint8), w.scale, x)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_result_in_the_place_of_an_input_that_the_call_quantises():
    from xdit_b200 import ops
    from xdit_b200.fp8_linear import fp8_linear, quantize_weight

    g = torch.Generator(device="cuda").manual_seed(3)
    w = quantize_weight(torch.randn(1024, 1024, device="cuda", generator=g) / 32)
    for M in (3, 300, 9000):
        x = torch.randn(M, 1024, device="cuda", generator=g).bfloat16()
        want = fp8_linear(x, w)
        ops.fp8_linear(x.unsqueeze(0), None, w.data, w.scale, out=x)
        assert torch.equal(x, want)
