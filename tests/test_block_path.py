"""The operators around the attention as a DiT block uses them together: on the GPU a whole block against the same
steps in plain torch, and a compiled one; under two gloo ranks the attention from projections with a
``RotaryEmbedding`` in its three forms (tables, halves, positions of each sample's own)."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def angles(p, B, s):
    """[B, s, pairs] angles that an ``xdit_rotary_positions`` block in host memory stands for."""
    f, axis = np.array(p.frequencies[:p.pairs]), np.array(p.axis[:p.pairs])
    if p.kind == 0:
        n = p.start + np.arange(s)
        sides = list(p.grid[:p.axes])
        pos = np.stack(np.unravel_index(n % math.prod(sides), sides), -1) * (n < math.prod(sides))[:, None]
        pos = np.broadcast_to(pos, (B, s, p.axes))
    else:
        kind = {1: np.int32, 2: np.int64, 3: np.float32}[p.kind]
        size = np.dtype(kind).itemsize
        n = (B - 1) * p.stride_b + (s - 1) * p.stride_row + (p.axes - 1) * p.stride_axis + 1
        flat = np.frombuffer((C.c_char * (n * size)).from_address(p.positions), dtype=kind)
        pos = np.lib.stride_tricks.as_strided(flat, (B, s, p.axes), [v * size for v in (p.stride_b, p.stride_row, p.stride_axis)])
    return pos[..., axis] * f


def rotated(x, ang, halves):
    """``x`` [B, H, s, D] turned by ``ang`` [B, s, pairs] (numpy, 64 bits)."""
    n = ang.shape[-1]
    a_at, b_at = (slice(0, n), slice(n, 2 * n)) if halves else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y = x.copy()
    y[..., a_at], y[..., b_at] = x[..., a_at] * c - x[..., b_at] * s, x[..., a_at] * s + x[..., b_at] * c
    return y


def _fake_axes(q, k, p, halves, out_q, out_k):
    ang = angles(p, q.shape[0], q.shape[2])
    for t, o in ((q, out_q), (k, out_k)):
        if t is not None:
            o.copy_(torch.from_numpy(rotated(t.double().numpy(), ang, halves)))


def _fake_tables(p, s, D, device):
    ang = angles(p, 1, s)[0]
    full = np.zeros((s, D // 2))
    full[:, :p.pairs] = ang
    full = torch.from_numpy(np.repeat(full, 2, axis=1)).float()
    return full.cos(), full.sin()


def _worker(rank, world, port, U, R, errq):
    try:
        os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
        dist.init_process_group("gloo", rank=rank, world_size=world)
        torch.set_num_threads(1)
        import xdit_b200
        from oracle import usp_oracle as O
        from tests import fake_ops
        from xdit_b200 import ops
        from xdit_b200.prologue import attention_from_projections
        from xdit_b200.rotary import RotaryEmbedding

        fake_ops.install()
        ops.rotary_axes, ops.rotary_tables, ops._check_tensors = _fake_axes, _fake_tables, lambda *t: None
        xdit_b200.init_sequence_parallel(U, R, backend="gloo")
        B, S, H, D = 2, 48 * world, 4, 32
        s = S // world
        g = torch.Generator().manual_seed(5)
        q, k, v = (torch.randn(B, S, H * D, generator=g) for _ in range(3))
        w = 1 + 0.1 * torch.randn(H * D, generator=g)
        n64 = lambda t: t.double().numpy()  # noqa: E731
        qn, kn, vn = (x[0].transpose(1, 0, 2, 3) for x in O.attention_prologue(n64(q), n64(k), n64(v), H, n64(w), n64(w), 1e-6,
                                                                             False, None, None, 1))
        ids = torch.randint(0, 50, (B, S, 2), generator=g)
        local = slice(rank * s, (rank + 1) * s)
        forms = [dict(axes_dim=(12, 10, 10), grid=(3, 4, 8), start=rank * s),             # tables
                 dict(axes_dim=(12, 10, 10), grid=(3, 4, 8), start=rank * s, pairing="halves"),
                 dict(axes_dim=(16, 16), positions=ids[:, local].contiguous(), ladder="shared")]
        for form in forms:
            whole = dict(form, start=0) if "grid" in form else dict(form, positions=ids)
            ang = angles(RotaryEmbedding(**whole)._params(B, S), B, S)
            qr, kr = (rotated(x, ang, form.get("pairing") == "halves") for x in (qn, kn))
            want, _ = O.attention_dense(qr, kr, vn)
            want = want.transpose(0, 2, 1, 3).reshape(B, S, H * D)[:, local]
            got = attention_from_projections(q[:, local], k[:, local], v[:, local], H, norm_q_weight=w, norm_k_weight=w,
                                             rotary_emb=RotaryEmbedding(**form))
            err = np.abs(got.double().numpy() - want).max()
            assert err < 5e-5, (U, R, form, rank, err)
        dist.barrier()
        dist.destroy_process_group()
    except Exception as e:
        import traceback

        errq.put(f"rank {rank}: {e}\n{traceback.format_exc()}")
        raise


@pytest.mark.parametrize("U,R", [(2, 1), (1, 2)])
def test_rotary_embedding_under_two_ranks(U, R):
    import torch.multiprocessing as mp

    ctx = mp.get_context("spawn")
    errq = ctx.SimpleQueue()
    procs = [ctx.Process(target=_worker, args=(r, 2, 29810 + U, U, R, errq)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(300)
    errs = []
    while not errq.empty():
        errs.append(errq.get())
    for p in procs:
        if p.is_alive():
            p.terminate()
            errs.append("a rank did not finish")
    assert not errs and all(p.exitcode == 0 for p in procs), "\n".join(errs)


def _round8(x):
    """Rows of fp32 values as the quantisation rule leaves them."""
    p = torch.nn.functional.pad(x, (0, -x.shape[-1] % 128)).unflatten(-1, (-1, 128))
    m, e = torch.frexp(p.abs().amax(-1, keepdim=True))
    s = torch.where(m > 0, torch.exp2((e - 9 + (m > 0.875).int()).double()).float(), torch.ones_like(m))
    return ((p / s).to(torch.float8_e4m3fn).float() * s).flatten(-2)[..., :x.shape[-1]]


class _Block:
    """One DiT block, B=1..2: norm and modulation, attention, gated residual, norm and modulation, feed-forward, gated
    residual; weights quantised once."""

    def __init__(self, C_, heads, F, seed=0):
        from xdit_b200.fp8_linear import quantize_weight

        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s, scale=1.0: torch.randn(*s, device="cuda", generator=g) * scale  # noqa: E731
        self.heads, self.C = heads, C_
        self.w = {n: quantize_weight(rand(o, i, scale=i ** -0.5)) for n, o, i in
                  (("qkv", 3 * C_, C_), ("o", C_, C_), ("up", F, C_), ("down", C_, F))}
        self.b = {n: rand(w.data.shape[0], scale=0.1) for n, w in self.w.items()}
        self.nq, self.nk = (1 + rand(C_, scale=0.1)).bfloat16(), (1 + rand(C_, scale=0.1)).bfloat16()
        self.mod = rand(2, 6, C_, scale=0.3)

    def __call__(self, x, rotary):
        from xdit_b200.fp8_linear import fp8_linear
        from xdit_b200.modulation import gated_residual_norm
        from xdit_b200.prologue import attention_from_hidden_states

        s1, t1, g1, s2, t2, g2 = (self.mod[:x.shape[0], i:i + 1] for i in range(6))
        _, z = gated_residual_norm(x, scale=s1, shift=t1, quantize=True)
        a = attention_from_hidden_states(z, self.w["qkv"], self.heads, qkv_bias=self.b["qkv"], out_proj_weight=self.w["o"],
                                         out_proj_bias=self.b["o"], norm_q_weight=self.nq, norm_k_weight=self.nk,
                                         rotary_emb=rotary)
        h, z = gated_residual_norm(x, a, gate=g1, scale=s2, shift=t2, quantize=True)
        y = fp8_linear(z, self.w["up"], self.b["up"], activation="gelu_tanh", quantize_out=True)
        y = fp8_linear(y, self.w["down"], self.b["down"])
        return gated_residual_norm(h, y, gate=g2, norm=None)[0]

    def plain(self, x, cos, sin):
        """The same in fp32 torch operations, rounded where the block rounds."""
        bf = lambda t: t.bfloat16().float()  # noqa: E731
        val = lambda w: w.data.float() * w.scale.repeat_interleave(128, 0)[:w.data.shape[0]].repeat_interleave(128, 1)[:, :w.data.shape[1]]  # noqa: E731
        lin = lambda n, t: _round8(t) @ val(self.w[n]).T + self.b[n]  # noqa: E731
        ln = lambda t: torch.nn.functional.layer_norm(t, (self.C,), eps=1e-6)  # noqa: E731
        s1, t1, g1, s2, t2, g2 = (self.mod[:x.shape[0], i:i + 1] for i in range(6))
        x = x.float()
        B, s, _ = x.shape
        q, k, v = bf(lin("qkv", ln(x) * (1 + s1) + t1)).chunk(3, -1)
        rms = lambda t, w: bf(t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w.float())  # noqa: E731
        head = lambda t: t.view(B, s, self.heads, -1).transpose(1, 2)  # noqa: E731
        q, k, v = head(rms(q, self.nq)), head(rms(k, self.nk)), head(v)

        def turn(t):
            a, b = t[..., 0::2], t[..., 1::2]
            return bf(torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2))

        q, k = turn(q), turn(k)
        a = bf(torch.softmax(q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1]), -1) @ v).transpose(1, 2).flatten(2)
        h = x + g1 * bf(lin("o", a))
        z = ln(h) * (1 + s2) + t2
        h = bf(h)
        y = bf(lin("down", torch.nn.functional.gelu(lin("up", z), approximate="tanh")))
        return bf(h + g2 * y)


@pytest.mark.gpu
@pytest.mark.parametrize("B,grid,C_,heads", [(1, (3, 8, 16), 512, 4), (2, (1, 9, 11), 640, 10)])
def test_a_block_of_them(B, grid, C_, heads):
    """Against the plain steps with the same roundings.  The two differ where a value lies next to a rounding: the
    attention's probabilities are bf16 (2e-3 of its result), which moves one e4m3 rounding in about thirty by up to an eighth
    (0.07 in the mean square): 1.3e-2 of a projection's result; gates of 0.3 bring the two projections' share of the
    result, whose residual is of size one, below 1e-2.  2e-2 leaves room for both at once."""
    import xdit_b200
    from xdit_b200 import ops
    from xdit_b200.rotary import RotaryEmbedding

    xdit_b200.init_sequence_parallel(1, 1)
    s, D = math.prod(grid), C_ // heads
    block = _Block(C_, heads, 1280)
    x = torch.randn(B, s, C_, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    third = D // 8 * 2
    e = RotaryEmbedding((D - 2 * third, third, third), grid=grid)
    with torch.no_grad():
        got = block(x, e)
        n = torch.arange(s, device="cuda")
        pos = torch.stack((n // (grid[1] * grid[2]), n // grid[2] % grid[1], n % grid[2]), -1).double()
        f = torch.cat([10000.0 ** (-torch.arange(0, d, 2, device="cuda").double() / d) for d in e.axes_dim])
        axis = torch.tensor([a for a, d in enumerate(e.axes_dim) for _ in range(d // 2)], device="cuda")
        ang = pos[:, axis] * f
        want = block.plain(x, ang.cos().float(), ang.sin().float())
        torch.cuda.synchronize()
        ops.check_status()
    err = (got.float() - want).norm() / want.norm()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert float(err) < 2e-2, float(err)
    # ids of the tokens in place of the grid, on a second call: the same result to the bit
    with torch.no_grad():
        ids = RotaryEmbedding(e.axes_dim, positions=pos.to(torch.int32))
        assert torch.equal(block(x, ids), got)


@pytest.mark.gpu
def test_embeddings_behind_the_prologue():
    """Halves, and positions of each sample's own, through the attention's path: what rotary_embed makes of the normed
    heads (the prologue rounds them once more in between, as it does without a rotation)."""
    from xdit_b200.prologue import qk_norm_rope_heads
    from xdit_b200.rotary import RotaryEmbedding, rotary_embed

    B, s, H, D = 2, 70, 4, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    x = [torch.randn(B, s, H * D, device="cuda", generator=g).bfloat16() for _ in range(3)]
    w = (1 + 0.1 * torch.randn(H * D, device="cuda", generator=g)).bfloat16()
    ids = torch.randint(0, 90, (B, s, 2), device="cuda", generator=g)
    plain = qk_norm_rope_heads(*x, H, norm_q_weight=w, norm_k_weight=w)
    for e in (RotaryEmbedding((32, 32), grid=(7, 10), pairing="halves"), RotaryEmbedding((32, 32), positions=ids)):
        got = qk_norm_rope_heads(*x, H, norm_q_weight=w, norm_k_weight=w, rotary_emb=e)
        want = rotary_embed(plain[0], plain[1], e)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], plain[2])


@pytest.mark.gpu
def test_a_compiled_block_has_no_graph_break():
    """The steps are custom operators under torch.compile: the block traces as one graph and gives the same bits."""
    import torch._dynamo as dynamo
    from xdit_b200.fp8_linear import fp8_linear, quantize_weight
    from xdit_b200.modulation import gated_residual_norm
    from xdit_b200.rotary import RotaryEmbedding, rotary_embed

    g = torch.Generator(device="cuda").manual_seed(3)
    w1, w2 = (quantize_weight(torch.randn(o, i, device="cuda", generator=g)) for o, i in ((512, 256), (256, 512)))
    gate = torch.randn(1, 1, 256, device="cuda", generator=g)
    ids = torch.randint(0, 99, (40, 2), device="cuda", generator=g)

    def block(x):
        q = x.view(1, 40, 4, 64).transpose(1, 2)
        q, _ = rotary_embed(q, None, RotaryEmbedding((32, 32), positions=ids))
        h, z = gated_residual_norm(x, q.transpose(1, 2).flatten(2), gate=gate, quantize=True)
        y = fp8_linear(z, w1, activation="gelu_tanh", quantize_out=True)
        y = fp8_linear(y, w2) + fp8_linear(h, w1)[..., :256]
        return gated_residual_norm(h, y)

    x = torch.randn(1, 40, 256, device="cuda", generator=g).bfloat16()
    with torch.no_grad():
        want = block(x)
        dynamo.reset()
        got = torch.compile(block, fullgraph=True, backend="aot_eager")(x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_captured_blocks_replay_to_the_bits_of_the_eager_ones():
    """Two graphs of two blocks each, the second with positions of each sample's own, replayed in turn on changed inputs with
    eager calls between."""
    import xdit_b200
    from xdit_b200 import ops
    from xdit_b200.graph import GraphedStep
    from xdit_b200.rotary import RotaryEmbedding

    xdit_b200.init_sequence_parallel(1, 1)
    B, grid, C_, heads = 2, (2, 9, 11), 512, 4
    s, g = math.prod(grid), torch.Generator(device="cuda").manual_seed(7)
    blocks = [_Block(C_, heads, 1280, seed) for seed in (8, 9)]
    x = torch.randn(B, s, C_, device="cuda", generator=g).bfloat16()
    ids = torch.randint(0, 60, (B, s, 3), device="cuda", generator=g)
    embeddings = [RotaryEmbedding((48, 40, 40), grid=grid), RotaryEmbedding((48, 40, 40), positions=ids, ladder="shared")]

    def two(e):
        return blocks[1](blocks[0](x, e), e)

    with torch.no_grad():
        steps = [GraphedStep(lambda e=e: two(e)) for e in embeddings]
        for _ in range(3):
            x.copy_(torch.randn(B, s, C_, device="cuda", generator=g))
            ids.copy_(torch.randint(0, 60, (B, s, 3), device="cuda", generator=g))
            want = [two(e) for e in embeddings]
            for step, w in ((steps[1], want[1]), (steps[0], want[0]), (steps[1], want[1])):
                assert torch.equal(step.replay(), w)
        torch.cuda.synchronize()
        ops.check_status()
