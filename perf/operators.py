"""Cases of the operators around a DiT block's attention: rotary positions with several axes, the norms
before and after a sub-layer with their gate, modulation and residual scale, and the linear layers in
8-bit floating point with one scale for each block of 128.

A case is a dict of plain values; ``prepare`` makes its inputs from a seed, ``run`` makes one pass, in
elementary torch operations or (``own``) through this repository's entry points, ``exact`` gives the same
results from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BLOCK = 128


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _rotary(name, B, H, Hk, s, D, axes, where, kind, pairing="interleaved", ladder="axis", theta=10000.0, start=0):
    return dict(name=name, op="rotary", B=B, H=H, Hk=Hk, s=s, D=D, axes=axes, where=where, kind=kind, pairing=pairing,
                ladder=ladder, theta=theta, start=start)


def _norm(name, B, s, C, kind, branch=True, post="none", pre="layer", gate="batch", mod="batch", vec="same",
          affine=False, scale=1.0, N=0):
    return dict(name=name, op="norm", B=B, s=s, C=C, kind=kind, branch=branch, post=post, pre=pre, gate=gate, mod=mod,
                vec=vec, affine=affine, scale=scale, N=N)


def _linear(name, M, K, N, kind, given="tensor", bias=True, act="none", F=0):
    return dict(name=name, op="linear", M=M, K=K, N=N, kind=kind, given=given, bias=bias, act=act, F=F)


def listed():
    return [
        # one new token of a streaming model, two requests: its position is far along the time axis
        _rotary("rotary one token", 2, 40, 40, 1, 128, "44,42,42", "ids", "bf16"),
        # text and image tokens in one sequence with ids of their own per sample, shared heads of the keys, halves
        # rotated against each other, a head whose last elements are not rotated
        _rotary("rotary ids, shared keys", 3, 28, 4, 4093, 128, "32,40,40", "ids", "f16", "halves", "shared", 1e6),
        # the self-attention of a 720p video of 81 frames on one GPU: 21 x 45 x 80 tokens
        _rotary("rotary video grid", 1, 40, 40, 75600, 128, "44,42,42", "grid:21,45,80", "bf16"),
        # one token through the last norm of a small image model
        _norm("norm one token", 2, 1, 1152, "f32", branch=False, gate="none"),
        # the second half of a block of an image model at 2048 x 2048: 16,384 tokens, two samples
        _norm("norm image block", 2, 16384, 1152, "bf16"),
        # modulation of every token, a norm behind the branch, an odd width, a residual scale
        _norm("norm per token, odd", 3, 1021, 1155, "f16", post="rms", pre="rms", gate="token", mod="token",
              affine=True, scale=0.7071),
        # the same step of the video model on one GPU, modulation kept in 32 bits
        _norm("norm video block", 1, 75600, 5120, "bf16", vec="f32", pre="layer"),
        # the video model's norm on a rank of eight, followed by the projection that takes its quantised rows
        _norm("norm into projection", 1, 9450, 5120, "bf16", vec="f32", N=5120),
        # the modulation of one layer from the time embedding of two samples: weights are read for two rows
        _linear("linear two tokens", 2, 5120, 30720, "bf16"),
        # keys of the text's cross-attention, from rows that came quantised with scales of any value
        _linear("linear text, given rows", 509, 4096, 5120, "f16", given="rows", bias=False),
        # the feed-forward of the video model on a rank of eight: up, GELU, down
        _linear("feed-forward shard", 9450, 5120, 5120, "bf16", act="gelu_tanh", F=13824),
        # the fused q, k, v projection of the video model on one GPU
        _linear("linear video qkv", 75600, 5120, 15360, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "linear", "linear"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "rotary":
        axes = rng.choice([(44, 42, 42), (16, 56, 56), (32, 32), (16, 24, 24), (24, 24, 24), (64,), (32, 40, 40)])
        D = sum(axes) + rng.choice([0, 0, 0, 16])
        B, Hk = rng.randint(1, 4), rng.randint(1, 16)
        H = Hk * rng.choice([1, 1, 2, 3])
        s = _log(rng, 1, max(2, int(9e7 / (B * (H + Hk) * D))))
        if len(axes) == 3 and rng.random() < 0.5:
            w = _log(rng, 1, 90)
            h = _log(rng, 1, 60)
            where = "grid:%d,%d,%d" % (max(1, s // (h * w)), h, w)
            start = rng.randint(0, s)
        else:
            where, start = rng.choice(["ids", "float"]), 0
        c = _rotary("", B, H, Hk, s, D, ",".join(map(str, axes)), where, kind, rng.choice(["interleaved", "halves"]),
                    rng.choice(["axis", "shared"]), rng.choice([256.0, 10000.0, 1e6]), start)
    elif op == "norm":
        C = rng.choice([_log(rng, 64, 8192), 128 * rng.randint(1, 48)])
        B = rng.randint(1, 4)
        s = _log(rng, 1, max(2, int(6e7 / (B * C))))
        c = _norm("", B, s, C, kind, rng.random() < 0.8, rng.choice(["none", "none", "rms", "layer"]),
                  rng.choice(["layer", "rms"]), rng.choice(["none", "batch", "token"]),
                  rng.choice(["none", "batch", "batch", "token"]), rng.choice(["same", "f32"]), rng.random() < 0.5,
                  rng.choice([1.0, 0.5]))
        if not c["branch"]:
            c.update(post="none", gate="none")
        if C % 128 == 0 and kind != "f32" and rng.random() < 0.3:
            c["N"] = 16 * rng.randint(1, 320)
    else:
        K, N = 16 * _log(rng, 4, 512), 16 * _log(rng, 4, 960)
        M = _log(rng, 1, max(2, int(min(2e4, 6e11 / (K * N), 1e9 / (K + N)))))
        kind = rng.choice(["bf16", "f16"])
        given = rng.choice(["tensor", "rows"])
        c = _linear("", M, K, N, kind, given, rng.random() < 0.7, rng.choice(["none", "none", "gelu_tanh"]))
        if rng.random() < 0.25:
            c.update(F=16 * _log(rng, 4, 512), act="gelu_tanh")
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _positions(case, g):
    """[B, s, axes] positions as a model makes them: text counts along every axis alike, images and videos walk
    their grid from where the text ended; fractions where a model stretches its grid."""
    B, s, A = case["B"], case["s"], len(case["axes"].split(","))
    n = torch.arange(s, device="cuda")
    side = max(1, int(math.sqrt(max(1, s // 4))))
    text = torch.randint(0, 400, (B, 1), device="cuda", generator=g)
    m = (n[None] - text).clamp_min(0)
    grid = torch.stack([m // (side * side), m // side % side, m % side][-A:] if A <= 3 else [m] * A, -1)
    ids = torch.where((n[None] < text)[..., None], n[None, :, None].expand(B, s, A), grid + text[..., None])
    if s == 1:
        ids = torch.randint(0, 100000, (B, 1, A), device="cuda", generator=g)
    return ids.float() * 0.75 if case["where"] == "float" else ids


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["kind"]]

    def randn(*shape, kind=None, scale=1.0, shift=0.0):
        x = torch.randn(*shape, device="cuda", generator=g)
        return (x if scale == 1.0 and shift == 0.0 else x.mul_(scale).add_(shift)).to(kind or t)

    if case["op"] == "rotary":
        B, s, D = case["B"], case["s"], case["D"]
        st = {"case": case,
              # projections [B, s, heads * D] seen as [B, heads, s, D]
              "q": randn(B, s, case["H"], D).transpose(1, 2), "k": randn(B, s, case["Hk"], D).transpose(1, 2),
              "axes": tuple(int(a) for a in case["axes"].split(","))}
        if not case["where"].startswith("grid"):
            st["positions"] = _positions(case, g)
        return st
    if case["op"] == "norm":
        B, s, C = case["B"], case["s"], case["C"]
        vec = t if case["vec"] == "same" else torch.float32
        # a residual stream has channels that stand out
        st = {"case": case, "x": (randn(B, s, C, kind=torch.float32) * (1 + 10 * (torch.rand(C, device="cuda", generator=g) > 0.995))).to(t)}
        st["branch"] = randn(B, s, C) if case["branch"] else None

        def rows(how, shift=0.0):
            if how == "none":
                return None
            return randn(B, 1 if how == "batch" else s, C, kind=vec, scale=0.3, shift=shift)

        st["gate"], st["scale"], st["shift"] = rows(case["gate"], 0.5), rows(case["mod"]), rows(case["mod"])
        for n in ("post_weight", "weight"):
            st[n] = randn(C, kind=vec, scale=0.1, shift=1.0) if case["affine"] else None
        st["bias"] = randn(C, kind=vec, scale=0.1) if case["affine"] and case["pre"] == "layer" else None
        if case["N"]:
            st["w"], st["ws"] = _weight(case["N"], C, g)
        return st
    M, K, N, F = case["M"], case["K"], case["N"], case["F"]
    st = {"case": case}
    if case["given"] == "rows":
        st["x"] = _as8(randn(M, K, kind=torch.float32, scale=100.0))
        st["xs"] = torch.rand(M, -(-K // BLOCK), device="cuda", generator=g) * 0.02 + 1e-3
    else:
        st["x"] = randn(M, K)
    st["w"], st["ws"] = _weight(F or N, K, g)
    st["b"] = randn(F or N, scale=0.5) if case["bias"] else None
    if F:
        st["w2"], st["ws2"] = _weight(N, F, g)
        st["b2"] = randn(N, scale=0.5) if case["bias"] else None
    return st


def _as8(x):
    return x.clamp_(-448, 448).to(torch.float8_e4m3fn)


def _weight(N, K, g):
    """A quantised weight as a checkpoint holds it: e4m3 values, one 32-bit scale for each block of 128 x 128."""
    w = _as8(torch.randn(N, K, device="cuda", generator=g).mul_(120))
    ws = torch.rand(-(-N // BLOCK), -(-K // BLOCK), device="cuda", generator=g) * 1e-4 + 1e-4
    return w, ws


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(st):
    return {"rotary": _run_rotary, "norm": _run_norm, "linear": _run_linear}[st["case"]["op"]](st)


def _pairs(case):
    """Of each rotated pair: its axis and its angle at position one."""
    axes = [int(a) for a in case["axes"].split(",")]
    axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    n = sum(axes) // 2
    if case["ladder"] == "shared":  # one ladder of frequencies over the rotated elements, cut into the axes
        freq = [case["theta"] ** (-i / n) for i in range(n)]
    else:  # each axis has a ladder of its own
        freq = [case["theta"] ** (-2 * i / d) for d in axes for i in range(d // 2)]
    return axis, freq


def _grid(case):
    T, Hh, W = (int(v) for v in case["where"].split(":")[1].split(","))
    n = torch.arange(case["start"], case["start"] + case["s"], device="cuda")
    pos = torch.stack([n // (Hh * W), n // W % Hh, n % W], -1)
    return torch.where((n < T * Hh * W)[:, None], pos, 0)[None]  # rows behind the grid are not rotated


def _run_rotary(st):
    case = st["case"]
    if own:
        from xdit_b200.rotary import RotaryEmbedding, rotary_embed

        if case["where"].startswith("grid"):
            where = dict(grid=tuple(int(v) for v in case["where"].split(":")[1].split(",")), start=case["start"])
        else:
            where = dict(positions=st["positions"])
        e = RotaryEmbedding(st["axes"], theta=case["theta"], pairing=case["pairing"], ladder=case["ladder"], **where)
        return rotary_embed(st["q"], st["k"], e)
    pos = _grid(case) if case["where"].startswith("grid") else st["positions"]
    axis, freq = _pairs(case)
    ang = pos[..., axis].double() * torch.tensor(freq, dtype=torch.float64, device="cuda")
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]  # [B or 1, 1, s, pairs]
    return _rotate(st["q"].float(), cos, sin, case).to(st["q"].dtype), _rotate(st["k"].float(), cos, sin, case).to(st["k"].dtype)


def _rotate(x, cos, sin, case):
    n = cos.shape[-1]
    out = x.clone()
    if case["pairing"] == "halves":
        a, b, at, bt = x[..., :n], x[..., n:2 * n], slice(0, n), slice(n, 2 * n)
    else:
        a, b, at, bt = x[..., 0:2 * n:2], x[..., 1:2 * n:2], slice(0, 2 * n, 2), slice(1, 2 * n, 2)
    out[..., at] = a * cos - b * sin
    out[..., bt] = a * sin + b * cos
    return out


def _run_norm(st):
    case = st["case"]
    if own:
        from xdit_b200.fp8_linear import Fp8Weight, fp8_linear
        from xdit_b200.modulation import gated_residual_norm

        h, z = gated_residual_norm(st["x"], st["branch"], gate=st["gate"], residual_scale=case["scale"],
                                   post_norm=None if case["post"] == "none" else case["post"], post_weight=st["post_weight"] if case["post"] != "none" else None,
                                   norm=case["pre"], weight=st["weight"], bias=st["bias"], scale=st["scale"],
                                   shift=st["shift"], eps=1e-6, quantize=bool(case["N"]))
        if case["N"]:
            z = fp8_linear(z, Fp8Weight(st["w"], st["ws"]), out_dtype=st["x"].dtype)
        return (h, z) if case["branch"] else z
    t = st["x"].dtype
    h = st["x"].float()
    if case["branch"]:
        y = st["branch"].float()
        if case["post"] != "none":
            y = _normed(y, case["post"], st["post_weight"], None)
        if st["gate"] is not None:
            y = y * st["gate"].float()
        h = case["scale"] * h + y
    z = _normed(h, case["pre"], st["weight"], st["bias"])
    if st["scale"] is not None:
        z = z * (1 + st["scale"].float()) + st["shift"].float()
    if case["N"]:
        B, s, C = z.shape
        z = (_round8(z.view(B * s, C)) @ _dequantized(st["w"], st["ws"]).T).view(B, s, -1)
    return (h.to(t), z.to(t)) if case["branch"] else z.to(t)


def _normed(x, how, weight, bias):
    if how == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    x = x if weight is None else x * weight.float()
    return x if bias is None else x + bias.float()


def _round8(x):
    """The values that rows quantised to e4m3 stand for: each block of 128 of a row has the smallest power of two as
    its scale that brings the block's values within 448; an empty block has the scale 1."""
    M, K = x.shape
    x = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(M, -1, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)
    s = torch.where(top > 0, (e + (127 - 9) + (m > 0.875) << 23).view(torch.float32), 1.0)  # the exponent's bits
    return ((x / s).to(torch.float8_e4m3fn).float() * s).view(M, -1)[:, :K]


def _dequantized(w, ws):
    N, K = w.shape
    return w.float() * ws.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _run_linear(st):
    case = st["case"]
    t = TYPES[case["kind"]]
    if own:
        from xdit_b200.fp8_linear import Fp8Rows, Fp8Weight, fp8_linear

        x = Fp8Rows(st["x"], st["xs"]) if case["given"] == "rows" else st["x"]
        act = None if case["act"] == "none" else case["act"]
        y = fp8_linear(x, Fp8Weight(st["w"], st["ws"]), st["b"], activation=act, out_dtype=t, quantize_out=bool(case["F"]))
        return fp8_linear(y, Fp8Weight(st["w2"], st["ws2"]), st["b2"], out_dtype=t) if case["F"] else y
    if case["given"] == "rows":
        x = st["x"].float() * st["xs"].repeat_interleave(BLOCK, 1)[:, :case["K"]]
    else:
        x = _round8(st["x"].float())
    y = x @ _dequantized(st["w"], st["ws"]).T
    y = y if st["b"] is None else y + st["b"].float()
    y = _gelu(y) if case["act"] != "none" else y
    if case["F"]:
        y = _round8(y) @ _dequantized(st["w2"], st["ws2"]).T
        y = y if st["b2"] is None else y + st["b2"].float()
    return y.to(t)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    e = SIZE[case["kind"]]
    if case["op"] == "rotary":
        rows = case["B"] * case["s"]
        n = rows * (case["H"] + case["Hk"]) * case["D"]
        ids = 0 if case["where"].startswith("grid") else rows * len(case["axes"].split(",")) * (4 if case["where"] == "float" else 8)
        return {"bytes": 2 * n * e + ids, "flops": 3 * n}
    if case["op"] == "norm":
        n = case["B"] * case["s"] * case["C"]
        v = e if case["vec"] == "same" else 4
        b = n * e * (3 if case["branch"] else 1)
        for how, count in ((case["gate"], 1), (case["mod"], 2)):
            b += count * v * {"none": 0, "batch": case["B"] * case["C"], "token": n}[how]
        N, f = case["N"], 12 * n
        if N:  # the normed rows stay between the two steps; the projection's weight is read and its result written
            b += N * case["C"] + case["B"] * case["s"] * N * e
            f += 2 * n * N
        else:
            b += n * e
        return {"bytes": b, "flops": f}
    M, K, N, F = case["M"], case["K"], case["N"], case["F"]
    b = M * K * (1 if case["given"] == "rows" else e) + M * N * e + (K * F + F * N if F else K * N)
    b += M * -(-K // BLOCK) * 4 if case["given"] == "rows" else 0
    return {"bytes": b, "flops": 2 * M * ((K * F + F * N) if F else K * N)}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":  # the rows in pieces: 64 bits take room
        return torch.cat([_exact_linear(case, st, r, r + 16384) for r in range(0, case["M"], 16384)])
    return {"rotary": _exact_rotary, "norm": _exact_norm}[case["op"]](case, st)


def _exact_rotary(case, st):
    """A pair (a, b) as the complex number a + ib, turned by its angle."""
    if case["where"].startswith("grid"):
        sides = [int(v) for v in case["where"].split(":")[1].split(",")]
        n = torch.arange(case["s"], device="cuda", dtype=torch.float64) + case["start"]
        w = torch.remainder(n, sides[2])
        h = torch.remainder(torch.floor(n / sides[2]), sides[1])
        pos = torch.stack([torch.floor(n / (sides[1] * sides[2])), h, w])
        pos = (pos * (n < sides[0] * sides[1] * sides[2]))[None]  # [1, axes, s]
    else:
        pos = st["positions"].double().permute(0, 2, 1)
    axis, freq = _pairs(case)
    turn = torch.stack([torch.polar(torch.ones_like(pos[:, a]), pos[:, a] * f) for a, f in zip(axis, freq)], -1)[:, None]

    def turned(x):
        x = x.double()
        r = 2 * turn.shape[-1]
        if case["pairing"] == "interleaved":
            z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
            y = torch.cat([z.real, z.imag], -1)
        return torch.cat([y, x[..., r:]], -1)

    return turned(st["q"]), turned(st["k"])


def _exact_norm(case, st):
    def norm(v, how, weight, bias):
        if how == "layer":
            var, mean = torch.var_mean(v, -1, unbiased=False, keepdim=True)
            v = (v - mean) / torch.sqrt(var + 1e-6)
        else:
            v = v / torch.sqrt(torch.square(v).mean(-1, keepdim=True) + 1e-6)
        return (v if weight is None else v * weight.double()) + (0 if bias is None else bias.double())

    h = st["x"].double()
    if case["branch"]:
        y = st["branch"].double()
        y = norm(y, case["post"], st["post_weight"], None) if case["post"] != "none" else y
        h = h * case["scale"] + (y if st["gate"] is None else y * st["gate"].double())
    z = norm(h, case["pre"], st["weight"], st["bias"])
    if case["mod"] != "none":
        z = z + z * st["scale"].double() + st["shift"].double()
    if case["N"]:
        z = (_exact8(z.flatten(0, 1)) @ _exact_weight(st["w"], st["ws"])).unflatten(0, z.shape[:2])
    return (h, z) if case["branch"] else z


def _exact8(x):
    """Rows rounded to e4m3 by its definition: steps of 2^-3 of a value's power of two, of 2^-9 below 2^-6, ties to even."""
    M, K = x.shape
    y = torch.zeros(M, -(-K // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    y[:, :K] = x
    y = y.view(M, -1, BLOCK)
    top = y.abs().amax(-1, keepdim=True)
    s = 2.0 ** torch.floor(torch.log2(top.clamp_min(1e-300)) - 8)
    s = torch.where(448 * s < top, 2 * s, s)
    s = torch.where(448 * (s / 2) >= top, s / 2, s)
    s = torch.where(top > 0, s, 1.0)
    y = y / s
    step = torch.exp2(torch.frexp(y)[1].double().sub(1).clamp_min(-6) - 3)
    return (torch.round(y / step) * step * s).view(M, -1)[:, :K]


def _exact_weight(w, ws):
    """[K, N] of a quantised weight [N, K]."""
    n, k = torch.arange(w.shape[0], device="cuda") // BLOCK, torch.arange(w.shape[1], device="cuda") // BLOCK
    return (w.double() * ws.double()[n][:, k]).T


def _exact_linear(case, st, first, last):
    x = st["x"][first:last].double()
    if case["given"] == "rows":
        x = x * st["xs"][first:last].double()[:, torch.arange(case["K"], device="cuda") // BLOCK]
    else:
        x = _exact8(x)
    y = x @ _exact_weight(st["w"], st["ws"])
    y = y if st["b"] is None else y + st["b"].double()
    if case["act"] != "none":
        y = y * torch.sigmoid(2 * (2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3))
    if case["F"]:
        y = _exact8(y) @ _exact_weight(st["w2"], st["ws2"])
        y = y if st["b2"] is None else y + st["b2"].double()
    return y
