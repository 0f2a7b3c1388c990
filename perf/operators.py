"""The block-scaled linear layers that are timed, and their plain forms.

Three operators, as a denoising step of the dual-stream model uses them when its
feed-forwards and timestep modulations hold their weights in 8 and 4 bits:

* ``norm``   -- gated residual update, RMS norm and modulation of the stream's
                rows, the normalised rows in 8 bits (e4m3) with a power-of-two
                scale for every 32 channels; without a norm, the rows themselves.
* ``linear`` -- the product of such rows with such weights, bias and tanh-GELU
                in its epilogue, the result in bf16 or in 8 bits with scales again.
* ``row4``   -- a linear layer over a few rows (one per sample or frame) whose
                weight is held in 4 bits (e2m1) with a bf16 scale per group.

8-bit rows: codes [..., K] (float8_e4m3fn) and scales [ceil(K / 128), rows, 4]
(float8_e8m0fnu): the four scales of a row's 128 columns lie together.  A
block's scale is the smallest power of two, at least 2^-127, with which no
value of the block passes 448.  4-bit weights: two codes a byte, the lower
column in the low half, and scales [N, K / group].
"""
import math

import torch
import torch.nn.functional as F

own = False

BF = torch.bfloat16
E4 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu
DEV = "cuda"
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    mod = {"y": True, "gate": True, "norm": True}
    return [
        # between two layers of a block, 512x768 chunk (3 frames of 16x24), two samples, one timestep each
        {"name": "norm video", "op": "norm", "B": 2, "L": 1152, "C": 4096, **mod, "mod": "sample"},
        # 480x704 output with a timestep per frame: modulation rows per token
        {"name": "norm per token", "op": "norm", "B": 2, "L": 990, "C": 4096, **mod, "mod": "token"},
        # the audio stream of the chunk: 75 tokens
        {"name": "norm audio", "op": "norm", "B": 2, "L": 75, "C": 2048, **mod, "mod": "sample"},
        # rows that come from no norm, on their way into a linear: a single token of the smallest model
        {"name": "rows, one token", "op": "norm", "B": 1, "L": 1, "C": 512, "y": False, "gate": False, "norm": False,
         "mod": "none"},
        # the video feed-forward's two linears over the chunk
        {"name": "linear up video", "op": "linear", "M": 2304, "K": 4096, "N": 16384, "gelu": True, "out": "mx"},
        {"name": "linear down video", "op": "linear", "M": 2304, "K": 16384, "N": 4096, "gelu": False, "out": "bf16"},
        # the audio feed-forward's first
        {"name": "linear up audio", "op": "linear", "M": 150, "K": 2048, "N": 8192, "gelu": True, "out": "mx"},
        # one 15x22 frame of a model whose widths fill no tile
        {"name": "linear ragged", "op": "linear", "M": 331, "K": 1056, "N": 4099, "gelu": True, "out": "bf16"},
        # two rows: one per sample
        {"name": "linear two rows", "op": "linear", "M": 2, "K": 4096, "N": 16384, "gelu": False, "out": "bf16"},
        # the video modulation of a step, one row per sample: the largest of the timestep linears
        {"name": "row4 modulation", "op": "row4", "M": 2, "K": 4096, "N": 24576, "group": 32, "silu": True},
        # the first linear of a timestep embedding
        {"name": "row4 embedding", "op": "row4", "M": 1, "K": 256, "N": 4096, "group": 64, "silu": False},
        # the audio modulation with a timestep per frame of a 4-frame first block, two samples
        {"name": "row4 per frame", "op": "row4", "M": 8, "K": 2048, "N": 12288, "group": 128, "silu": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "row4"])
    if op == "norm":
        y = rng.random() < 0.8
        norm = rng.random() < 0.8
        return {"op": "norm", "B": rng.choice([1, 2, 2, 3]), "L": _log(rng, 1, 1152), "C": 32 * _log(rng, 4, 256),
                "y": y, "gate": y and rng.random() < 0.7, "norm": norm,
                "mod": rng.choice(["none", "sample", "sample", "token"]) if norm else "none"}
    if op == "row4":
        group = rng.choice([32, 64, 128])
        return {"op": "row4", "M": rng.randint(1, 16), "K": group * _log(rng, max(1, 128 // group), 4096 // group),
                "N": _log(rng, 1, 24576), "group": group, "silu": rng.random() < 0.6}
    out = rng.choice(["bf16", "mx"])
    c = {"op": "linear", "M": _log(rng, 1, 2304), "K": 32 * _log(rng, 4, 512), "N": _log(rng, 32, 16384),
         "gelu": rng.random() < 0.5, "out": out}
    if out == "mx":
        c["N"] = max(32, c["N"] // 32 * 32)
    while c["M"] * c["K"] * c["N"] > 2304 * 4096 * 16384:
        c["M"] = c["M"] // 2
    return c


def work(case):
    c = case
    if c["op"] == "norm":
        rows, C = c["B"] * c["L"], c["C"]
        b = rows * C * 2 + rows * C + rows * C // 32
        if c["y"]:
            b += 2 * rows * C * 2
        each = {"none": 0, "sample": c["B"], "token": rows}[c["mod"]]
        b += each * C * 2 * 2 + (max(each, c["B"]) * C * 2 if c["gate"] else 0)
        return {"bytes": b, "flops": rows * C * 8}
    M, K, N = c["M"], c["K"], c["N"]
    if c["op"] == "linear":
        b = (M + N) * K + (M + N) * K // 32 + N * 2
        b += M * N * 2 if c["out"] == "bf16" else M * N + M * N // 32
        return {"bytes": b, "flops": 2 * M * N * K}
    return {"bytes": N * K // 2 + N * K // c["group"] * 2 + M * K * 2 + N * 2 + M * N * 2, "flops": 2 * M * N * K}


# --------------------------------------------------------------------------
# the formats
# --------------------------------------------------------------------------
def _to_mx(v):
    """float32 rows [R, K] as 8-bit codes [R, K] and scales [ceil(K / 128), R, 4]."""
    R, K = v.shape
    blocks = v.reshape(R, K // 32, 32)
    top = blocks.abs().amax(-1)
    m, e = torch.frexp(top)                                  # top = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    k = e - 9 + (m > 0.875).to(e.dtype)
    k = torch.where(top == 0, torch.full_like(k, -127), k).clamp(-127, 127)
    codes = torch.ldexp(blocks, -k[..., None]).to(E4).reshape(R, K)
    scales = F.pad((k + 127).to(torch.uint8), (0, -(K // 32) % 4))
    return codes, scales.reshape(R, -1, 4).transpose(0, 1).contiguous().view(E8)


def _of_mx(codes, scales):
    """The float32 rows that 8-bit codes [R, K] and their scales stand for."""
    R, K = codes.shape
    s = scales.view(torch.uint8).transpose(0, 1).reshape(R, -1)[:, :K // 32].to(torch.int32) - 127
    return torch.ldexp(codes.float().reshape(R, K // 32, 32), s[..., None]).reshape(R, K)


def _to_4(w, group):
    """float32 weights [N, K] as packed e2m1 codes [N, K / 2] and bf16 scales [N, K / group]."""
    N, K = w.shape
    g = w.reshape(N, K // group, group)
    s = (g.abs().amax(-1) / 6.0).to(BF)
    t = g / s.float().clamp_min(1e-30)[..., None]
    grid = torch.tensor(E2M1, device=w.device)
    code = torch.bucketize(t.abs(), (grid[1:] + grid[:-1]) / 2).to(torch.uint8) | (t < 0).to(torch.uint8) << 3
    code = code.reshape(N, K // 2, 2)
    return code[..., 0] | code[..., 1] << 4, s


def _of_4(packed, scales, group):
    """The float32 weights [N, K] that packed codes and their scales stand for."""
    N = packed.shape[0]
    grid = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=packed.device)
    code = torch.stack([packed & 15, packed >> 4], -1).reshape(N, -1)
    w = grid[code.long()].reshape(N, -1, group)
    return (w * scales.float()[..., None]).reshape(N, -1)


# --------------------------------------------------------------------------
# the inputs
# --------------------------------------------------------------------------
def _stream_rows(shape, g):
    """Rows of a residual stream: normal values, a few channels far larger."""
    C = shape[-1]
    spread = torch.ones(C, device=DEV)
    spread[torch.randperm(C, generator=g, device=DEV)[:max(1, C // 128)]] = 12.0
    return torch.randn(shape, generator=g, device=DEV) * spread


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    if c["op"] == "norm":
        B, L, C = c["B"], c["L"], c["C"]
        s = {"case": c, "x": _stream_rows((B, L, C), g).to(BF), "y": None, "gate": None, "scale": None, "shift": None}
        if c["y"]:
            s["y"] = randn(B, L, C).to(BF)
        rows = L if c["mod"] == "token" else 1
        if c["gate"]:
            s["gate"] = (0.5 * randn(B, rows, C)).to(BF)
        if c["mod"] != "none":
            s["scale"] = (0.3 * randn(B, rows, C)).to(BF)
            s["shift"] = (0.3 * randn(B, rows, C)).to(BF)
        return s
    M, K, N = c["M"], c["K"], c["N"]
    s = {"case": c, "bias": (0.1 * randn(N)).to(BF)}
    if c["op"] == "linear":
        s["a"] = _to_mx(_stream_rows((M, K), g))
        s["w"] = _to_mx(randn(N, K) / math.sqrt(K))
        return s
    s["x"] = randn(M, K).to(BF)
    s["w"] = _to_4(randn(N, K) / math.sqrt(K), c["group"])
    if own:
        from taomate_amd import quant
        s["packed"] = quant.Group4Weight.from_codes(*s["w"])
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"] == "norm":
        x = s["x"].float()
        if s["y"] is not None:
            y = s["y"].float()
            x = x + (y if s["gate"] is None else y * s["gate"].float())
        n = x
        if c["norm"]:
            n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            if s["scale"] is not None:
                n = n * (1.0 + s["scale"].float()) + s["shift"].float()
        codes, scales = _to_mx(n.reshape(-1, c["C"]))
        out = {"codes": codes.view(n.shape), "scales": scales}
        if s["y"] is not None:
            out["x"] = x.to(BF)
        return out
    if c["op"] == "linear":
        y = _of_mx(*s["a"]) @ _of_mx(*s["w"]).t() + s["bias"].float()
        if c["gelu"]:
            y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
        if c["out"] == "bf16":
            return {"y": y.to(BF)}
        codes, scales = _to_mx(y)
        return {"codes": codes, "scales": scales}
    x = s["x"].float()
    if c["silu"]:
        x = x / (1.0 + torch.exp(-x))
    return {"y": (x @ _of_4(*s["w"], c["group"]).t() + s["bias"].float()).to(BF)}


def _own(s, c):
    from taomate_amd import kernels, quant
    if c["op"] == "norm":
        x = torch.empty_like(s["x"]) if s["y"] is not None else None
        n = kernels.adaln_mx(s["x"], y=s["y"], gate=s["gate"], x_out=x, scale=s["scale"], shift=s["shift"],
                             eps=EPS if c["norm"] else None)
        out = {"codes": n.codes, "scales": n.scales}
        if x is not None:
            out["x"] = x
        return out
    if c["op"] == "linear":
        a, w = quant.MXRows(*s["a"]), quant.MXRows(*s["w"])
        y = kernels.mx_linear(a, w, s["bias"], gelu=c["gelu"], quantize=c["out"] == "mx")
        return {"codes": y.codes, "scales": y.scales} if c["out"] == "mx" else {"y": y}
    return {"y": kernels.group4_linear(s["x"], s["packed"], s["bias"], silu=c["silu"])}


# --------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------
def _e4m3_value(t):
    """The e4m3 value nearest each float64 |t| <= 448, ties to the even code: steps of 2^-3 of
    the value's power of two, of 2^-9 below 2^-6."""
    _, e = torch.frexp(t)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3.0)
    return torch.round(t / step) * step


def _mx_value(v):
    """Codes and scales of float64 rows, as the values they stand for by themselves."""
    R, K = v.shape
    blocks = v.view(R, K // 32, 32)
    top = blocks.abs().amax(-1)
    k = torch.ceil(torch.log2((top / 448.0).clamp_min(2.0 ** -130)))
    k = torch.where(top > 448.0 * torch.exp2(k), k + 1, k)         # the logarithm's own rounding, both ways
    k = torch.where(top <= 448.0 * torch.exp2(k - 1), k - 1, k).clamp(-127, 127)
    k = torch.where(top == 0, torch.full_like(k, -127.0), k)
    codes = _e4m3_value(blocks / torch.exp2(k)[..., None]).reshape(R, K)
    full = torch.full((R, -(-K // 128) * 4), 2.0 ** -127, dtype=torch.float64, device=v.device)
    full[:, :K // 32] = torch.exp2(k)
    return codes, full.view(R, -1, 4).permute(1, 0, 2).contiguous()


def _mx_double(codes, scales):
    R, K = codes.shape
    power = torch.exp2(scales.view(torch.uint8).double() - 127.0).permute(1, 0, 2).reshape(R, -1)
    return codes.double() * power[:, :K // 32].repeat_interleave(32, dim=1)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "norm":
        x = s["x"].double()
        if c["y"]:
            x = torch.addcmul(x, s["y"].double(), s["gate"].double()) if c["gate"] else x + s["y"].double()
        n = x
        if c["norm"]:
            n = x / torch.sqrt(x.square().sum(-1, keepdim=True) / c["C"] + EPS)
            if c["mod"] != "none":
                n = n + n * s["scale"].double() + s["shift"].double()
        codes, scales = _mx_value(n.reshape(-1, c["C"]))
        out = {"codes": codes.view(n.shape), "scales": scales}
        if c["y"]:
            out["x"] = x
        return out
    if c["op"] == "linear":
        y = torch.addmm(s["bias"].double(), _mx_double(*s["a"]), _mx_double(*s["w"]).t())
        if c["gelu"]:
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * y * (1.0 + 0.044715 * y.square()))
        if c["out"] == "bf16":
            return {"y": y}
        codes, scales = _mx_value(y)
        return {"codes": codes, "scales": scales}
    packed, scales = s["w"]
    code = torch.empty(packed.shape[0], packed.shape[1] * 2, dtype=torch.int64, device=DEV)
    code[:, 0::2], code[:, 1::2] = packed & 15, packed >> 4
    mag = code & 7
    w = torch.where(mag < 2, mag * 0.5, (1 + (mag & 1) * 0.5) * torch.exp2((mag >> 1).double() - 1.0))
    w = torch.where(code >= 8, -w, w) * scales.double().repeat_interleave(c["group"], dim=1)
    x = s["x"].double()
    if c["silu"]:
        x = x * torch.sigmoid(x)
    return {"y": torch.addmm(s["bias"].double(), x, w.t())}
