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
        return torch.ldexp(v, s.unsqueeze(-1)).reshape(self.codes.shape)


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
    """A weight [N, columns] in 4 bits: ``codes`` uint8 [N, ceil(K / 128) * 64] in
    the kernel's order (byte c * 64 + p * 16 + j * 4 + i of a row holds columns
    c * 128 + j * 32 + p * 8 + 2 i, in the low half, and the next one) and
    ``scales`` bf16 [N, K / group]."""
    __slots__ = ("codes", "scales", "columns")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, columns: int):
        self.codes, self.scales, self.columns = codes, scales, int(columns)

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], self.columns))

    @property
    def group(self) -> int:
        return self.columns // self.scales.shape[1]

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
        if scales.shape[1] == 0 or K % scales.shape[1] or K // scales.shape[1] not in GROUPS:
            raise ValueError(f"Group4Weight: {K} columns in {scales.shape[1]} groups: groups must be 32, 64 or 128 columns")
        chunks = -(-K // 128)
        rows = F.pad(packed, (0, -packed.shape[1] % 64)).reshape(N, chunks, 4, 4, 4)    # chunk, j, p, i
        return cls(rows.transpose(2, 3).reshape(N, chunks * 64).contiguous(), scales.contiguous(), K)

    def dequantize(self) -> torch.Tensor:
        """The float32 values that the codes stand for."""
        N, K = self.shape
        rows = self.codes.reshape(N, -(-K // 128), 4, 4, 4).transpose(2, 3).flatten(1)[:, :K // 2]
        code = torch.stack([rows & 15, rows >> 4], -1).reshape(N, K)
        grid = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=rows.device)
        w = grid[code.long()].reshape(N, K // self.group, self.group) * self.scales.to(torch.float32).unsqueeze(-1)
        return w.reshape(N, K)


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
    t = w.abs() / scales.to(torch.float32).clamp_min(torch.finfo(torch.float32).tiny).unsqueeze(-1)
    grid = torch.tensor(_E2M1, device=w.device)
    mid = (grid[1:] + grid[:-1]) / 2
    # below or on a midpoint: the lower code; on one whose lower code is odd: the upper
    code = torch.bucketize(t, mid)
    on = t == mid[code.clamp(max=6)]
    code = torch.where(on & (code % 2 == 1) & (code < 7), code + 1, code).to(torch.uint8)
    code = (code | ((w < 0).to(torch.uint8) << 3)).reshape(N, K // 2, 2)
    return Group4Weight.from_codes(code[..., 0] | (code[..., 1] << 4), scales)
