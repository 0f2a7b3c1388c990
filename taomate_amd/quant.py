"""Tensors of the block-scaled linear layers: 8-bit rows and 4-bit weights.

``MXRows``: rows [..., K] in the OCP microscaling form with e4m3 elements, one
power-of-two scale for every 32 columns.  Activations get it from
``kernels.adaln_mx`` and ``kernels.mx_linear(..., quantize=True)``, weights
from ``quantize_mx``.

``Group4Weight``: a weight [N, K] in e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives) with a bf16 scale for every group of 32, 64 or 128 columns,
packed in the order in which ``kernels.group4_linear`` feeds the matrix cores.

The functions here are plain torch, on any device: they run once, when a
weight is laid out.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

MX_BLOCK = 32
E4M3_MAX = 448.0
E2M1_MAX = 6.0
GROUPS = (32, 64, 128)
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class MXRows:
    """8-bit rows: ``codes`` float8_e4m3fn [..., K] and ``scales`` float8_e8m0fnu
    [ceil(K / 128), rows, 4], both contiguous; the scale of column c of row r is
    scales[c // 128, r, c % 128 // 32].  Scales past K are 2^-127 (byte 0)."""
    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        self.codes, self.scales = codes, scales

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def tensors(self):
        return self.codes, self.scales

    def dequantize(self) -> torch.Tensor:
        """The float32 values that the codes stand for."""
        K, rows = self.codes.shape[-1], self.scales.shape[1]
        s = self.scales.view(torch.uint8).transpose(0, 1).flatten(1)[:, :K // MX_BLOCK].to(torch.int32) - 127
        v = self.codes.to(torch.float32).reshape(rows, K // MX_BLOCK, MX_BLOCK)
        v = torch.ldexp(v, s.unsqueeze(-1)).masked_fill((s == 128).unsqueeze(-1), float("nan"))   # byte 255
        return v.reshape(self.codes.shape)


def quantize_mx(x: torch.Tensor) -> MXRows:
    """Rows [..., K] (K a multiple of 32) in 8 bits, as the kernels quantise
    their results: a block's scale is the smallest power of two, at least
    2^-127, with which no finite value of the block passes 448; each value is
    rounded once to nearest even.  Values that are not finite become NaN and
    do not count in their block's maximum."""
    K = x.shape[-1] if x.dim() else 0
    if K == 0 or K % MX_BLOCK:
        raise ValueError(f"quantize_mx: the last dimension must be a multiple of {MX_BLOCK}, got {tuple(x.shape)}")
    if not x.is_floating_point() or x.dtype == torch.float64:
        raise TypeError(f"quantize_mx takes float32, bfloat16 or float16 rows, got {x.dtype}")
    v = x.detach().to(torch.float32).reshape(x.numel() // K, K // MX_BLOCK, MX_BLOCK)
    top = torch.where(v.isfinite(), v, torch.zeros_like(v)).abs().amax(-1)
    m, e = torch.frexp(top)                       # top = m 2^e, m in [0.5, 1), and 448 = 0.875 * 2^9
    k = e - 9 + (m > E4M3_MAX / 512).to(e.dtype)
    k = torch.where(top == 0, torch.full_like(k, -127), k.clamp(min=-127))
    codes = torch.ldexp(v, -k.unsqueeze(-1)).to(torch.float8_e4m3fn).reshape(x.shape)
    scales = F.pad((k + 127).to(torch.uint8), (0, -(K // MX_BLOCK) % 4))
    scales = scales.reshape(v.shape[0], scales.shape[1] // 4, 4).transpose(0, 1).contiguous()
    return MXRows(codes, scales.view(torch.float8_e8m0fnu))


class Group4Weight:
    """A weight [N, K] in 4 bits, zero-padded to whole tiles of 16 rows and 128
    columns: ``codes`` uint8 [ceil(N / 16), ceil(K / 128), 4, 16, 16] and
    ``scales`` bf16 [ceil(N / 16), ceil(K / 128), 16, 128 / group].  Byte
    [t, c, p, r, 4 j + i] holds row 16 t + r, columns 128 c + 32 j + 8 p + 2 i
    (low half) and the next one (p, j, i in [0, 4))."""
    __slots__ = ("codes", "scales", "rows", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, columns: int):
        self.codes, self.scales, self.rows, self.columns = codes, scales, int(rows), int(columns)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.columns))

    @property
    def group(self) -> int:
        return 128 // self.scales.shape[3]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def tensors(self):
        return self.codes, self.scales

    @classmethod
    def from_codes(cls, packed: torch.Tensor, scales: torch.Tensor) -> "Group4Weight":
        """From codes in column order, two a byte with the lower column in the
        low half (uint8 [N, K / 2]), and bf16 scales [N, K / group]."""
        if packed.dtype != torch.uint8 or packed.dim() != 2 or scales.dtype != torch.bfloat16 or scales.dim() != 2 \
                or scales.shape[0] != packed.shape[0]:
            raise ValueError("Group4Weight: codes must be uint8 [N, K / 2] and scales bf16 [N, K / group]")
        N, K = packed.shape[0], packed.shape[1] * 2
        if K == 0 or scales.shape[1] == 0 or K % scales.shape[1] or K // scales.shape[1] not in GROUPS:
            raise ValueError(f"Group4Weight: {K} columns in {scales.shape[1]} groups: groups must be 32, 64 or 128 columns")
        per, chunks, tiles = 128 * scales.shape[1] // K, -(-K // 128), -(-N // 16)
        if K % 128 or N % 16:
            packed = F.pad(packed, (0, chunks * 64 - K // 2, 0, tiles * 16 - N))
            scales = F.pad(scales, (0, chunks * per - scales.shape[1], 0, tiles * 16 - N))
        codes = packed.reshape(tiles, 16, chunks, 4, 4, 4)
        # tile, row, chunk, j, p, i -> tile, chunk, p, row, j, i
        codes = codes.permute(0, 2, 4, 1, 3, 5).reshape(tiles, chunks, 4, 16, 16).contiguous()
        scales = scales.reshape(tiles, 16, chunks, per).transpose(1, 2).clone(memory_format=torch.contiguous_format)
        return cls(codes, scales, N, K)

    def dequantize(self) -> torch.Tensor:
        """The float32 values that the codes stand for."""
        tiles, chunks = self.codes.shape[:2]
        rows = self.codes.reshape(tiles, chunks, 4, 16, 4, 4).permute(0, 3, 1, 4, 2, 5).reshape(tiles * 16, chunks * 64)
        code = torch.stack([rows & 15, rows >> 4], -1).reshape(tiles * 16, chunks * 128)
        grid = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=rows.device)
        scales = self.scales.transpose(1, 2).reshape(tiles * 16, chunks * 128 // self.group).to(torch.float32)
        w = grid[code.long()] * scales.repeat_interleave(self.group, dim=1)
        return w[:self.rows, :self.columns].contiguous()


def quantize_group4(weight: torch.Tensor, group: int = 32) -> Group4Weight:
    """A weight [N, K] in 4 bits: each group's scale is its largest magnitude
    over 6, in bf16, each value the nearest e2m1 step under that scale (ties to
    the even code)."""
    if group not in GROUPS:
        raise ValueError(f"quantize_group4: group must be 32, 64 or 128, got {group}")
    if weight.dim() != 2 or weight.shape[1] == 0 or weight.shape[1] % group:
        raise ValueError(f"quantize_group4: a weight [N, K] with K a multiple of {group}, got {tuple(weight.shape)}")
    N, K = weight.shape
    w = weight.detach().to(torch.float32).reshape(N, K // group, group)
    if not bool(w.isfinite().all()):
        raise ValueError("quantize_group4: the weight holds values that are not finite (4-bit codes have none)")
    scales = (w.abs().amax(-1) / E2M1_MAX).to(torch.bfloat16)
    t = w.abs() / scales.to(torch.float32).clamp_min(2.0 ** -133).unsqueeze(-1)   # bf16's smallest
    grid = torch.tensor(_E2M1, device=w.device)
    mid = (grid[1:] + grid[:-1]) / 2
    # below or on a midpoint: the lower code; on one whose lower code is odd: the upper
    code = torch.bucketize(t, mid)
    on = t == mid[code.clamp(max=6)]
    code = torch.where(on & (code % 2 == 1) & (code < 7), code + 1, code).to(torch.uint8)
    code = (code | ((w < 0).to(torch.uint8) << 3)).reshape(N, K // 2, 2)
    return Group4Weight.from_codes(code[..., 0] | (code[..., 1] << 4), scales)


class Packed:
    """What a linear's weight was packed into, as long as it holds: ``holds(lin)``
    tells whether ``lin.weight`` is still the parameter, in the memory and at the
    version, that was packed (a change through ``.data`` in place goes unseen).
    Keeps the memory of the weight alive, so that nothing else can come to lie there,
    until ``lapse``: the caller's, once the packing holds no more.  The rows stay for
    captured graphs, and the packing never holds again.
    ``into``: an earlier packing whose rows are overwritten, so that captured graphs
    read the new ones.  Rows on a GPU that have another layout (shape, group or
    device) are refused instead of being freed under such a graph.  A deep copy or
    pickle carries no rows and never holds: versions count anew there."""
    __slots__ = ("rows", "weight", "source", "at", "version")

    def __init__(self, lin: torch.nn.Linear, rows, into: "Packed | None" = None):
        if lin.weight.is_inference():
            raise ValueError("a weight made in inference mode does not tell when it is changed: it cannot be packed")
        old = None if into is None else into.rows
        if old is not None and old.shape == rows.shape and all(
                a.shape == b.shape and a.device == b.device for a, b in zip(old.tensors(), rows.tensors())):
            for a, b in zip(old.tensors(), rows.tensors()):
                a.view(torch.uint8).copy_(b.view(torch.uint8))
            rows = old
        elif old is not None and old.device.type == "cuda":
            raise ValueError(f"packed rows {tuple(old.shape)} on {old.device} have another layout, and a captured graph "
                             "may read them: drop them first (False)")
        self.rows = rows
        self.weight = lin.weight
        self.source = lin.weight.detach()
        self.at = self.source.data_ptr()   # source itself follows a storage that is allocated anew
        self.version = lin.weight._version

    def lapse(self) -> None:
        self.weight = self.source = None

    @classmethod
    def _lapsed(cls) -> "Packed":
        p = cls.__new__(cls)
        p.rows = p.weight = p.source = p.at = p.version = None
        return p

    def __reduce__(self):
        return Packed._lapsed, ()

    def holds(self, lin: torch.nn.Linear) -> bool:
        w = lin._parameters.get("weight")
        return (w is not None and w is self.weight and w.data_ptr() == self.at and w._version == self.version
                and w.shape == self.source.shape and w.dtype == self.source.dtype and w.device == self.source.device)
