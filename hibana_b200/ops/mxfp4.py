"""MXFP4: e2m1 values with one power-of-two scale per block of 32 elements along K (the OCP microscaling format).

A block's scale is 2^(b - 127), b a byte: b = max(floor(log2(max |x|)) - 2 + 127, 0); its elements are x / scale rounded to
the nearest e2m1 value (ties to the even code), saturating at 6. A block with an infinity or a NaN gets b = 255, the
format's NaN. There is no per-tensor scale, so activations need no calibration.

Values are packed two per byte (low nibble first). Scale bytes are kept in the 128 x 4 blocks that the tensor cores consume,
as for NVFP4 (ops/nvfp4.py), four bytes being 128 elements of a row here. Published checkpoints hold both row-major:
`from_blocks` takes those. The torch functions are the reference of csrc/mxfp4.cu and what runs on CPU.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _native as nv
from .nvfp4 import e2m1_codes, e2m1_values, swizzle_blocks, unswizzle_sf

BLOCK = 32
NAN_SCALE = 255

nv.register("hb_quant_mxfp4", [nv.P, nv.I, nv.L, nv.I, nv.I, nv.I, nv.P, nv.P, nv.P, nv.I, nv.I, nv.P])
nv.register("hb_dequant_mxfp4", [nv.P, nv.P, nv.I, nv.I, nv.I, nv.P, nv.I, nv.P])

IN_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def k_atoms(k: int) -> int:
    """Number of 128-element K atoms of a scale tensor, padded to a whole 256-element K tile."""
    return ((k + 255) // 256) * 2


def quantize_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Reference quantiser. x [M, K] -> (packed uint8 [M, K / 2], row-major scale bytes uint8 [M, K / 32])."""
    m, k = x.shape
    v = x.float().reshape(m, k // BLOCK, BLOCK)
    amax = v.abs().amax(dim=-1)
    bad = ~torch.isfinite(amax)
    # frexp: amax = f * 2^e with f in [0.5, 1), so floor(log2(amax)) = e - 1
    e = torch.frexp(torch.where(bad, torch.ones_like(amax), amax)).exponent
    b = torch.where(amax > 0, e - 1 - 2 + 127, torch.zeros_like(e)).clamp_min(0)
    inv = torch.ldexp(torch.ones_like(amax), 127 - b)
    codes = e2m1_codes(torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v) * inv.unsqueeze(-1)).view(m, k)
    b = torch.where(bad, torch.full_like(b, NAN_SCALE), b).to(torch.uint8)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8), b


def scale_values(b: torch.Tensor) -> torch.Tensor:
    """Scale bytes -> fp32 factors (255 is NaN)."""
    s = torch.ldexp(torch.ones(b.shape, device=b.device), b.int() - 127)
    return torch.where(b == NAN_SCALE, torch.full_like(s, float("nan")), s)


def dequantize_ref(packed: torch.Tensor, sfb: torch.Tensor) -> torch.Tensor:
    """(packed [M, K / 2], scale bytes [M, K / 32]) -> fp32 [M, K]."""
    m, kh = packed.shape
    p = packed.int()
    vals = e2m1_values(torch.stack((p & 15, p >> 4), dim=-1).view(m, kh * 2)).view(m, kh * 2 // BLOCK, BLOCK)
    return (vals * scale_values(sfb).unsqueeze(-1)).view(m, kh * 2)


@dataclass
class Mxfp4Tensor:
    """A quantised [rows, k] matrix: packed values and scale blocks. Scale bytes of the rows that pad the last 128 are
    not part of it and may hold anything."""

    q: torch.Tensor          # uint8 [rows, k / 2]
    sf: torch.Tensor         # uint8 [ceil(rows / 128), k_atoms, 512]
    rows: int
    k: int

    @property
    def ka(self) -> int:
        return self.sf.shape[1]

    def to(self, device) -> "Mxfp4Tensor":
        return Mxfp4Tensor(self.q.to(device), self.sf.to(device), self.rows, self.k)

    def scales(self) -> torch.Tensor:
        """Row-major scale bytes [rows, k / 32]."""
        return unswizzle_sf(self.sf, self.rows, self.k // BLOCK)

    def dequantize(self) -> torch.Tensor:
        return dequantize(self, torch.float32)


def from_blocks(packed: torch.Tensor, scales: torch.Tensor) -> Mxfp4Tensor:
    """Wraps a checkpoint's row-major tensors: packed uint8 [rows, K / 2] (or [rows, K / 32, 16]) and scale bytes uint8
    [rows, K / 32]. The packed values are used where they are; the scales are laid out once."""
    if packed.dim() == 3:
        packed = packed.flatten(1)
    if packed.dtype != torch.uint8 or scales.dtype != torch.uint8 or packed.dim() != 2 or scales.dim() != 2:
        raise ValueError("MXFP4 blocks: uint8 packed values [rows, K / 2] and uint8 scales [rows, K / 32] expected")
    rows, k = packed.shape[0], packed.shape[1] * 2
    if rows < 1 or k < BLOCK or k % BLOCK or scales.shape != (rows, k // BLOCK):
        raise ValueError(f"MXFP4 blocks: packed {tuple(packed.shape)} and scales {tuple(scales.shape)} do not fit together")
    packed = packed.contiguous()
    if packed.data_ptr() % 16:             # the kernels fetch 16-byte pieces
        packed = packed.clone()
    return Mxfp4Tensor(packed, swizzle_blocks(scales, k_atoms(k)), rows, k)


def cut(packed: torch.Tensor, scales: torch.Tensor, rows, c0: int, c1: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows (slice or index tensor) and columns c0 .. c1 (whole blocks) of a matrix in row-major blocks; nothing is
    requantised."""
    if c0 % BLOCK or c1 % BLOCK:
        raise ValueError(f"MXFP4: columns [{c0}, {c1}) are not whole blocks of {BLOCK}")
    return packed[rows][:, c0 // 2:c1 // 2], scales[rows][:, c0 // BLOCK:c1 // BLOCK]


def _check(x: torch.Tensor) -> tuple[int, int]:
    shape = x.shape
    if len(shape) != 2 or x.dtype not in IN_TYPES:
        raise ValueError(f"MXFP4: a bf16, fp16 or fp32 matrix expected, got {x.dtype} {tuple(shape)}")
    m, k = shape
    if k < BLOCK or k % BLOCK:
        raise ValueError(f"MXFP4: K must be a positive multiple of {BLOCK}, got {k}")
    if m and x.stride(1) != 1:
        raise ValueError("MXFP4: the elements of a row must be contiguous")
    return m, k


def _alloc(m: int, k: int, device: torch.device) -> tuple[torch.Tensor, torch.Tensor]:
    rb = (m + 127) // 128
    rb += rb & 1 if rb > 1 else 0          # whole 256-row tiles (see nvfp4.swizzle_sf)
    return (torch.empty(m, k // 2, dtype=torch.uint8, device=device),
            torch.empty(rb, k_atoms(k), 512, dtype=torch.uint8, device=device))


def empty(m: int, k: int, device: torch.device) -> Mxfp4Tensor:
    """An MXFP4 matrix with nothing in it yet."""
    return Mxfp4Tensor(*_alloc(m, k, device), m, k)


def quantize(x: torch.Tensor) -> Mxfp4Tensor:
    """Rows [M, K] (bf16, fp16 or fp32; any row stride, K a multiple of 32) -> MXFP4."""
    m, k = _check(x)
    if nv.use_native(x):
        q, sf = _alloc(m, k, x.device)
        if m:
            _launch(x, m, k, q, sf, None, m, 0)
        return Mxfp4Tensor(q, sf, m, k)
    packed, sfb = quantize_ref(x)
    return Mxfp4Tensor(packed, swizzle_blocks(sfb, k_atoms(k)), m, k)


def _launch(x, m, k, q, sf, pos, rows, topk) -> None:
    with nv.on_device(x):
        nv.check(nv.lib().hb_quant_mxfp4(x.data_ptr(), IN_TYPES[x.dtype], x.stride(0), m, k, k_atoms(k), q.data_ptr(),
                                         sf.data_ptr(), nv.ptr(pos), rows, topk, nv.stream()), "hb_quant_mxfp4")


def quantize_pairs(x: torch.Tensor, pos: torch.Tensor, topk: int, rows: int) -> Mxfp4Tensor:
    """Into the expert-sorted buffer of a mixture-of-experts layer (CUDA only), [rows, K]: pair p of `pos` (int32, one number a
    token and expert) becomes row pos[p], from x[p // topk] or, with topk 0, from x[pos[p]]. Pairs whose number is negative or
    not below `rows` are left out, and rows that no pair names are left unwritten. A row that two pairs name holds either's."""
    m, k = _check(x)
    n = pos.numel()
    if not x.is_cuda or pos.dtype != torch.int32 or pos.device != x.device or not pos.is_contiguous():
        raise ValueError("MXFP4: row numbers are a contiguous int32 tensor on the rows' CUDA device")
    if topk < 0 or (n != m * topk if topk else rows > m) or rows < 0:
        raise ValueError(f"MXFP4: {n} row numbers (top {topk}) of {rows} rows do not fit {m} rows")
    nv.use_native(x)
    out = empty(rows, k, x.device)
    if n and rows:
        _launch(x, n, k, out.q, out.sf, pos, rows, topk)
    return out


def quantize_weight(w: torch.Tensor) -> Mxfp4Tensor:
    """A weight matrix [N, K] of any float type."""
    return quantize(w.contiguous() if w.dtype in IN_TYPES else w.float().contiguous())


def dequantize(t: Mxfp4Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values an MXFP4 matrix stands for, [rows, k]. Exact in bf16 and fp32; fp16 rounds what it cannot hold."""
    if dtype not in IN_TYPES:
        raise ValueError(f"MXFP4 values come as bf16, fp16 or fp32, not {dtype}")
    if nv.use_native(t.q, t.sf):
        out = torch.empty(t.rows, t.k, dtype=dtype, device=t.q.device)
        if t.rows:
            with nv.on_device(t.q):
                nv.check(nv.lib().hb_dequant_mxfp4(t.q.data_ptr(), t.sf.data_ptr(), t.rows, t.k, t.ka, out.data_ptr(),
                                                   IN_TYPES[dtype], nv.stream()), "hb_dequant_mxfp4")
        return out
    return dequantize_ref(t.q, t.scales()).to(dtype)
