"""Weight-only 4-bit (W4A16) tensors in the MFMA-operand-native layout.

``pack_w4`` turns integer weights ``q[N, K]`` (0..15), zero points ``z[N, K/G]``
and scales ``s[N, K/G]`` into

* ``qw  [N/16, K/128, 64, 4] int32`` - tile ``(nt, kb)`` is 1 KiB; lane
  ``c + 16 g`` holds row ``16 nt + c``, columns ``128 kb + 32 g + 8 w + e`` in word
  ``w``, element ``e`` in nibble ``(e >> 1) + 4 (e & 1)``;
* ``sz  [N/16, K/G, 16, 2]`` in the activation dtype - ``(scale, OFF + zero)``
  with ``OFF`` = 128 (bf16) or 1024 (fp16), the value whose exponent bits the
  kernel ORs onto a nibble to make it a float.

The kernels in ``csrc/quant_gemm.hip`` consume this layout; the functions here
are the layout's definition and the reference semantics (``unpack_w4`` +
``F.linear``).  AWQ checkpoints (the reference's documented model is AWQ,
``.env.server:11``) are converted with ``awq_unpack`` + ``pack_w4`` after the
tensor-parallel shards have been cut.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

_AWQ_ORDER = [0, 4, 1, 5, 2, 6, 3, 7]
_NIBBLE_OF_ELEM = [(e >> 1) + 4 * (e & 1) for e in range(8)]


def w4_offset(dtype: torch.dtype) -> float:
    if dtype in (torch.bfloat16, torch.float32):      # fp32 only on the reference path
        return 128.0
    if dtype == torch.float16:
        return 1024.0
    raise TypeError(f"W4A16 needs bf16/fp16 activations, got {dtype}")


def awq_unpack(packed: torch.Tensor) -> torch.Tensor:
    """AWQ ``[R, C/8] int32`` -> ``[R, C] uint8`` (nibble order 0,4,1,5,2,6,3,7)."""
    shifts = torch.tensor([4 * _AWQ_ORDER.index(i) for i in range(8)], dtype=torch.int32,
                          device=packed.device)
    u = (packed.unsqueeze(-1) >> shifts) & 0xF
    return u.reshape(packed.shape[0], -1).to(torch.uint8)


def awq_pack(vals: torch.Tensor) -> torch.Tensor:
    """Inverse of ``awq_unpack``: ``[R, C]`` ints in 0..15 -> ``[R, C/8] int32``."""
    r, c = vals.shape
    v = vals.to(torch.int64).reshape(r, c // 8, 8)
    out = torch.zeros((r, c // 8), dtype=torch.int64, device=vals.device)
    for i in range(8):
        out |= v[..., i] << (4 * _AWQ_ORDER.index(i))
    out = torch.where(out >= (1 << 31), out - (1 << 32), out)
    return out.to(torch.int32)


def gptq_to_awq(name: str, w: torch.Tensor, zero_offset: int = 1) -> torch.Tensor:
    """One tensor of a 4-bit GPTQ linear (``qweight [in/8, out]``: eight input rows per word, low nibble
    first; ``qzeros [in/g, out/8]``: eight output columns per word in natural order, stored minus
    ``zero_offset`` by the original format; ``scales [in/g, out]``) in the AWQ arrangement the
    W4A16 path consumes (``qweight [in, out/8]``, ``qzeros [in/g, out/8]``, AWQ nibble order).
    The two formats hold the same integers: only the packing differs."""
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=w.device)
    if name.endswith(".qweight"):
        rows = ((w.unsqueeze(1) >> shifts.view(1, 8, 1)) & 0xF)           # [in/8, 8, out]
        return awq_pack(rows.reshape(-1, w.shape[1]))
    if name.endswith(".qzeros"):
        z = ((w.unsqueeze(-1) >> shifts) & 0xF).reshape(w.shape[0], -1) + zero_offset
        if int(z.max()) > 15:
            raise NotImplementedError(f"{name}: a GPTQ zero point of 16 does not fit the 4-bit zero points "
                                      "of the W4A16 kernels (load with --quantization awq-dequant)")
        return awq_pack(z)
    return w


def pack_w4(q: torch.Tensor, z: torch.Tensor, s: torch.Tensor, dtype: torch.dtype,
            ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q [N, K]``, ``z [N, K/G]``, ``s [N, K/G]`` -> ``(qw, sz)`` as described above."""
    n, k = q.shape
    ng = s.shape[1]
    assert n % 16 == 0 and k % 128 == 0 and k % ng == 0 and (k // ng) % 128 == 0, (n, k, ng)
    assert z.shape == s.shape == (n, ng)
    v = q.to(torch.int64).reshape(n // 16, 16, k // 128, 4, 4, 8)        # nt c kb g w e
    v = v.permute(0, 2, 3, 1, 4, 5).reshape(n // 16, k // 128, 64, 4, 8)  # nt kb (g c) w e
    word = torch.zeros(v.shape[:-1], dtype=torch.int64, device=q.device)
    for e in range(8):
        word |= v[..., e] << (4 * _NIBBLE_OF_ELEM[e])
    word = torch.where(word >= (1 << 31), word - (1 << 32), word)
    qw = word.to(torch.int32).contiguous()
    off = w4_offset(dtype)
    sc = s.to(torch.float32).reshape(n // 16, 16, ng).permute(0, 2, 1)
    zc = z.to(torch.float32).reshape(n // 16, 16, ng).permute(0, 2, 1) + off
    sz = torch.stack([sc, zc], dim=-1).to(dtype).contiguous()
    return qw, sz


def unpack_w4(qw: torch.Tensor, sz: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Inverse of ``pack_w4``: ``(q [N,K] uint8, z [N,K/G] f32, s [N,K/G] f32)``."""
    nt, kb = qw.shape[0], qw.shape[1]
    w = qw.to(torch.int64) & 0xFFFFFFFF
    elems = [(w >> (4 * _NIBBLE_OF_ELEM[e])) & 0xF for e in range(8)]
    v = torch.stack(elems, dim=-1).reshape(nt, kb, 4, 16, 4, 8)          # nt kb g c w e
    q = v.permute(0, 3, 1, 2, 4, 5).reshape(nt * 16, kb * 128).to(torch.uint8)
    ng = sz.shape[1]
    s = sz[..., 0].to(torch.float32).permute(0, 2, 1).reshape(nt * 16, ng)
    z = sz[..., 1].to(torch.float32).permute(0, 2, 1).reshape(nt * 16, ng) - w4_offset(sz.dtype)
    return q, z, s


def w4_dequant(qw: torch.Tensor, sz: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Dense ``[N, K]`` weights ``(q - z) * s`` (reference path)."""
    q, z, s = unpack_w4(qw, sz)
    g = q.shape[1] // s.shape[1]
    w = (q.to(torch.float32) - z.repeat_interleave(g, dim=1)) * s.repeat_interleave(g, dim=1)
    return w.to(dtype)


def w4a16_gemm(x: torch.Tensor, qw: torch.Tensor, sz: torch.Tensor) -> torch.Tensor:
    """Reference ``x [M, K] -> [M, N]``: fp32 accumulation over exact ``(q-z)*s``."""
    return (x.to(torch.float32) @ w4_dequant(qw, sz).t()).to(x.dtype)


def quantize_w4(w: torch.Tensor, group: int = 128) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Asymmetric round-to-nearest 4-bit quantisation of dense ``w [N, K]`` per
    ``group`` input columns: ``(q, z, s)`` with ``w ~ (q - z) * s``."""
    n, k = w.shape
    wg = w.to(torch.float32).reshape(n, k // group, group)
    lo, hi = wg.amin(-1), wg.amax(-1)
    s = ((hi - lo) / 15.0).clamp_min(1e-8)
    z = (-lo / s).round().clamp(0, 15)
    q = (wg / s.unsqueeze(-1) + z.unsqueeze(-1)).round().clamp(0, 15)
    return q.reshape(n, k).to(torch.uint8), z, s


# ------------------------------------------------------------------ NVFP4
# E2M1 code -> value; code bit 3 is the sign (``Dockerfile:5-6`` of the
# reference installs the fp4 kernels its documented deployments rely on).
FP4_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def fp4_lut(device=None) -> torch.Tensor:
    v = torch.tensor(FP4_VALUES, dtype=torch.float32, device=device)
    return torch.cat([v, -v])


def pack_fp4(packed: torch.Tensor, block_scale: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """NVFP4 checkpoint tensors -> kernel layout.  ``packed [N, K/2] uint8``
    holds element ``2i`` in the low nibble of byte ``i``; ``block_scale
    [N, K/16]`` is ``float8_e4m3fn`` (one scale per 16 input columns).  Returns
    ``qw [N/16, K/128, 64, 4] int32`` (same tiles as ``pack_w4``, element ``e`` in
    nibble ``e``) and ``fs [N/16, K/128, 64] int32`` - lane ``c + 16 g`` holds the
    scales of row ``c``, blocks ``8 kb + 2 g`` (low half) and ``8 kb + 2 g + 1``
    (high half), as bf16 bit patterns (every e4m3 value is exact in bf16)."""
    n, kh = packed.shape
    k = kh * 2
    assert packed.dtype == torch.uint8 and n % 16 == 0 and k % 128 == 0, (packed.dtype, n, k)
    assert block_scale.shape == (n, k // 16), (block_scale.shape, n, k)
    words = packed.contiguous().view(torch.int32).reshape(n // 16, 16, k // 128, 4, 4)      # nt c kb g w
    qw = words.permute(0, 2, 3, 1, 4).reshape(n // 16, k // 128, 64, 4).contiguous()
    sb = block_scale.to(torch.float32).to(torch.bfloat16).reshape(n // 16, 16, k // 128, 4, 2)   # nt c kb g j
    fs = sb.permute(0, 2, 3, 1, 4).reshape(n // 16, k // 128, 64, 2).contiguous().view(torch.int32)
    return qw, fs.reshape(n // 16, k // 128, 64)


def unpack_fp4(qw: torch.Tensor, fs: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Inverse of ``pack_fp4``: ``(codes [N, K] uint8 in 0..15, block_scale [N, K/16] f32)``."""
    nt, kb = qw.shape[0], qw.shape[1]
    w = qw.reshape(nt, kb, 4, 16, 4).permute(0, 3, 1, 2, 4).contiguous()               # nt c kb g w
    by = w.view(torch.uint8).reshape(nt * 16, kb * 64)                                # [N, K/2]
    codes = torch.stack([by & 0xF, by >> 4], dim=-1).reshape(nt * 16, kb * 128)
    sb = fs.contiguous().view(torch.bfloat16).reshape(nt, kb, 4, 16, 2).permute(0, 3, 1, 2, 4)
    return codes, sb.reshape(nt * 16, kb * 8).to(torch.float32)


def fp4_dequant(qw: torch.Tensor, fs: torch.Tensor, alpha: torch.Tensor = None,
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Dense ``[N, K]`` weights ``e2m1 * block_scale * alpha[row]`` (reference path)."""
    codes, sc = unpack_fp4(qw, fs)
    w = fp4_lut(qw.device)[codes.long()] * sc.repeat_interleave(16, dim=1)
    if alpha is not None:
        w = w * alpha.to(torch.float32).reshape(-1, 1)
    return w.to(dtype)


def fp4a16_gemm(x: torch.Tensor, qw: torch.Tensor, fs: torch.Tensor, alpha: torch.Tensor = None) -> torch.Tensor:
    return (x.to(torch.float32) @ fp4_dequant(qw, fs, alpha).t()).to(x.dtype)


def quantize_fp4(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Round-to-nearest NVFP4 quantisation of dense ``w [N, K]``:
    ``(packed [N, K/2] uint8, block_scale [N, K/16] float8_e4m3fn, global_scale [1] f32)``
    with ``w ~ e2m1 * block_scale / global_scale`` - the tensors (and the
    divide-by-global-scale convention) of a compressed-tensors
    ``nvfp4-pack-quantized`` checkpoint."""
    n, k = w.shape
    wf = w.to(torch.float32)
    amax = wf.abs().max().clamp_min(1e-12)
    gscale = (448.0 * 6.0 / amax).reshape(1)
    blocks = wf.reshape(n, k // 16, 16)
    bs = (blocks.abs().amax(-1) / 6.0 * gscale).clamp(max=448.0).to(torch.float8_e4m3fn)
    eff = (bs.to(torch.float32) / gscale).clamp_min(1e-30).unsqueeze(-1)
    lut = torch.tensor(FP4_VALUES, dtype=torch.float32, device=w.device)
    mag = (blocks.abs() / eff).clamp(max=6.0)
    code = (mag.unsqueeze(-1) - lut).abs().argmin(-1)
    code = (code + 8 * (blocks < 0)).to(torch.uint8).reshape(n, k // 2, 2)
    packed = code[..., 0] | (code[..., 1] << 4)
    return packed.contiguous(), bs, gscale


# ------------------------------------------------------------------ microscaled formats (blocks of 32 values, one power of two each)
MX_BLOCK = 32
MX_LARGEST = {8: 448.0, 4: 6.0}      # largest element: e4m3, e2m1


def _ceil_to(n: int, m: int) -> int:
    return -(-n // m) * m


class MxRows:
    """Rows in microscaled 8- or 4-bit floating point: a value is ``element * 2^(scale byte - 127)``, one scale for each 32
    neighbours of a row; a scale byte of 255 makes its block NaN.

    ``q`` ``[M, K]`` float8_e4m3fn (8 bits) or ``[M, K/2]`` uint8 (4 bits, the even element in the low half of a byte), ``s``
    ``[M, K/32]`` float8_e8m0fnu; ``dtype``: the type that products of these rows have.  Both are views of ``payload`` and ``scales``,
    whose rows are padded (elements with zeros to a multiple of 128 columns, scales to 16 bytes), which is what the kernels read."""
    __slots__ = ("payload", "scales", "width", "bits", "dtype")

    def __init__(self, payload: torch.Tensor, scales: torch.Tensor, width: int, bits: int, dtype: torch.dtype):
        self.payload, self.scales, self.width, self.bits, self.dtype = payload, scales, width, bits, dtype

    @staticmethod
    def empty(rows: int, width: int, bits: int, dtype: torch.dtype, device) -> "MxRows":
        """Buffers for a kernel to fill (uninitialised)."""
        if bits != 8 and bits != 4:
            raise ValueError(f"microscaled rows hold 8 or 4 bits a value, not {bits}")
        if width <= 0 or width % MX_BLOCK:
            raise ValueError(f"{width} columns are not whole blocks of {MX_BLOCK}")
        kp = (width + 127) // 128 * 128
        # (sizes as numbers: a tuple of them takes torch half as long again, 1.6 us)
        payload = (torch.empty(rows, kp, dtype=torch.float8_e4m3fn, device=device) if bits == 8
                   else torch.empty(rows, kp // 2, dtype=torch.uint8, device=device))
        return MxRows(payload, torch.empty(rows, (kp + 511) // 512 * 16, dtype=torch.float8_e8m0fnu, device=device), width, bits, dtype)

    @staticmethod
    def of(q: torch.Tensor, s: torch.Tensor, dtype: torch.dtype) -> "MxRows":
        """Rows from elements and scales that come from elsewhere (``q`` and ``s`` as the properties have them, ``s`` also uint8)."""
        bits = 8 if q.dtype == torch.float8_e4m3fn else 4
        if q.dtype not in (torch.float8_e4m3fn, torch.uint8) or s.dtype not in (torch.float8_e8m0fnu, torch.uint8):
            raise TypeError(f"microscaled rows of {q.dtype} elements and {s.dtype} scales")
        width = q.shape[-1] * (8 // bits)
        if q.dim() != 2 or s.dim() != 2 or width % MX_BLOCK or tuple(s.shape) != (q.shape[0], width // MX_BLOCK):
            raise ValueError(f"elements {tuple(q.shape)} and scales {tuple(s.shape)} are not rows of blocks of {MX_BLOCK}")
        r = MxRows.empty(q.shape[0], width, bits, dtype, q.device)
        r.payload.view(torch.uint8).zero_()
        r.payload.view(torch.uint8)[:, :q.shape[1]] = q.view(torch.uint8)
        r.scales.view(torch.uint8).zero_()
        r.scales.view(torch.uint8)[:, :s.shape[1]] = s.view(torch.uint8)
        return r

    def take(self, rows: torch.Tensor) -> "MxRows":
        """The rows of these numbers."""
        return MxRows(self.payload.view(torch.uint8).index_select(0, rows).view(self.payload.dtype),
                      self.scales.view(torch.uint8).index_select(0, rows).view(self.scales.dtype), self.width, self.bits, self.dtype)

    @property
    def q(self) -> torch.Tensor:
        n = self.width * self.bits // 8
        return self.payload if self.payload.shape[1] == n else self.payload[:, :n]

    @property
    def s(self) -> torch.Tensor:
        n = self.width // MX_BLOCK
        return self.scales if self.scales.shape[1] == n else self.scales[:, :n]

    @property
    def shape(self) -> Tuple[int, int]:
        return (self.payload.shape[0], self.width)

    @property
    def device(self) -> torch.device:
        return self.payload.device

    @property
    def is_cuda(self) -> bool:
        return self.payload.is_cuda


class MxWeight(NamedTuple):
    """A 4-bit microscaled weight (or several of one shape) in the kernels' layout, and its number of rows without padding.

    ``qw [.., N/16, K/128, 64, 4] int32``: tiles as ``pack_fp4`` lays them out; ``ws [.., N/16, K/512, 64, 4] uint8``: byte ``i``
    of lane ``c + 16 g`` is the scale of row ``c`` of the tile, block ``16 j + 4 i + g`` of its columns.  Rows are padded with zeros
    to a multiple of 16, columns to 128 (of ``ws`` to 512)."""
    qw: torch.Tensor
    ws: torch.Tensor
    rows: int


def pack_mx(packed: torch.Tensor, scales: torch.Tensor, halves: int = 1) -> MxWeight:
    """4-bit blocks in the order checkpoints have them (``packed [.., N, K/2] uint8``, the even element in the low half;
    ``scales [.., N, K/32]`` biased exponents, uint8 or float8_e8m0fnu) -> ``MxWeight``.  ``halves`` 2: the rows are
    ``[gate ; up]``, each padded to a multiple of 128 (the columns of the projection that follows come in whole steps)."""
    lead, n, k = packed.shape[:-2], packed.shape[-2], packed.shape[-1] * 2
    if packed.dtype != torch.uint8 or k % MX_BLOCK or tuple(scales.shape) != (*lead, n, k // MX_BLOCK):
        raise ValueError(f"codes {tuple(packed.shape)} {packed.dtype} and scales {tuple(scales.shape)} are not 4-bit blocks of {MX_BLOCK}")
    if halves not in (1, 2) or n % halves or n % (8 * halves):
        raise ValueError(f"{n} rows in {halves} part(s): multiples of 8 are wanted")
    sb = scales.view(torch.uint8)
    np_ = _ceil_to(n // halves, 128 if halves == 2 else 16) * halves
    kp, ks = _ceil_to(k, 128), _ceil_to(k, 512)
    pad_rows = (np_ - n) // halves

    def padded(t: torch.Tensor, cols: int) -> torch.Tensor:
        t = t.reshape(*lead, halves, n // halves, t.shape[-1])
        t = torch.nn.functional.pad(t, (0, cols - t.shape[-1], 0, pad_rows))
        return t.reshape(*lead, np_, cols)
    nl = len(lead)
    order = list(range(nl))
    words = padded(packed, kp // 2).contiguous().view(torch.int32).reshape(*lead, np_ // 16, 16, kp // 128, 4, 4)      # nt c kb g w
    qw = words.permute(*order, nl, nl + 2, nl + 3, nl + 1, nl + 4).reshape(*lead, np_ // 16, kp // 128, 64, 4).contiguous()
    sc = padded(sb, ks // MX_BLOCK).reshape(*lead, np_ // 16, 16, ks // 512, 4, 4)                                     # nt c j i g
    ws = sc.permute(*order, nl, nl + 2, nl + 4, nl + 1, nl + 3).reshape(*lead, np_ // 16, ks // 512, 64, 4).contiguous()
    return MxWeight(qw, ws, np_ if halves == 2 else n)


def pad_mx_bias(bias: torch.Tensor, halves: int = 1) -> torch.Tensor:
    """``bias [.., N]`` for the padded rows of ``pack_mx``."""
    n = bias.shape[-1] // halves
    np_ = _ceil_to(n, 128) if halves == 2 else n
    b = bias.reshape(*bias.shape[:-1], halves, n)
    return torch.nn.functional.pad(b, (0, np_ - n)).reshape(*bias.shape[:-1], halves * np_).contiguous()


def unpack_mx(w: MxWeight) -> Tuple[torch.Tensor, torch.Tensor]:
    """Inverse of ``pack_mx`` up to the padding: ``(packed [.., N, Kp/2], scales [.., N, Kp/32])``."""
    lead, (nt, kb), nj = w.qw.shape[:-4], w.qw.shape[-4:-2], w.ws.shape[-3]
    nl = len(lead)
    order = list(range(nl))
    q = w.qw.reshape(*lead, nt, kb, 4, 16, 4).permute(*order, nl, nl + 3, nl + 1, nl + 2, nl + 4).contiguous()     # nt c kb g w
    q = q.view(torch.uint8).reshape(*lead, nt * 16, kb * 64)[..., :w.rows, :]
    s = w.ws.reshape(*lead, nt, nj, 4, 16, 4).permute(*order, nl, nl + 3, nl + 1, nl + 4, nl + 2)                  # nt c j i g
    return q, s.reshape(*lead, nt * 16, nj * 16)[..., :w.rows, :kb * 4]


def mx_blocks(x: torch.Tensor, bits: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [.., K]`` -> (elements as numbers ``[.., K/32, 32]``, scale bytes ``[.., K/32]``), in 32 bits: the definition."""
    b = x.to(torch.float32).reshape(*x.shape[:-1], x.shape[-1] // MX_BLOCK, MX_BLOCK)
    a = b.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(b).all(-1, keepdim=True)
    a = torch.where(finite, a, torch.zeros_like(a))
    m, e = torch.frexp(a)
    # the smallest e with a <= largest * 2^e; 448 = 0.875 * 2^9, 6 = 0.75 * 2^3
    e = e - (9 if bits == 8 else 3) + (m > (0.875 if bits == 8 else 0.75)).to(e.dtype)
    e = torch.where(a > 0, e, torch.full_like(e, -127)).clamp(-127, 127)
    u = torch.ldexp(torch.where(finite, b, torch.zeros_like(b)), -e)
    if bits == 8:
        u = u.to(torch.float8_e4m3fn).to(torch.float32)
    else:
        t = u.abs()
        step = torch.where(t < 2, 0.5, torch.where(t < 4, 1.0, 2.0))
        u = torch.copysign(torch.round(t / step) * step, u)
    byte = torch.where(finite, e + 127, torch.full_like(e, 255))
    return u, byte.squeeze(-1).to(torch.uint8)


def mx_quantize(x: torch.Tensor, bits: int, dtype: Optional[torch.dtype] = None) -> MxRows:
    """Reference path of ``ops.mx_quantize``."""
    u, byte = mx_blocks(x, bits)
    if bits == 8:
        q = u.reshape(x.shape).to(torch.float8_e4m3fn)
    else:
        code = torch.tensor([0, 1, 2, 3, 4, 0, 5, 0, 6, 0, 0, 0, 7], dtype=torch.uint8, device=x.device)[(u.abs() * 2).long()]
        code = (code | (torch.signbit(u).to(torch.uint8) << 3)).reshape(*x.shape[:-1], x.shape[-1] // 2, 2)
        q = code[..., 0] | (code[..., 1] << 4)
    return MxRows.of(q, byte, dtype or x.dtype)


def _mx_scaled(u: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    e = byte.to(torch.int32) - 127
    v = torch.ldexp(u.to(torch.float32), e.unsqueeze(-1))
    return torch.where((byte == 255).unsqueeze(-1), torch.full_like(v, float("nan")), v)


def mx_dequantize(rows: MxRows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Reference path of ``ops.mx_dequantize``."""
    s = rows.s.view(torch.uint8)
    if rows.bits == 8:
        u = rows.q.to(torch.float32)
    else:
        u = fp4_lut(rows.device)[torch.stack([rows.q & 15, rows.q >> 4], dim=-1).long()]
    return _mx_scaled(u.reshape(*s.shape, MX_BLOCK), s).reshape(rows.shape).to(dtype)


def mx_weight_dense(w: MxWeight) -> torch.Tensor:
    """The weight as fp32 ``[.., N, Kp]`` (columns from K on are zeros)."""
    q, s = unpack_mx(w)
    u = fp4_lut(q.device)[torch.stack([q & 15, q >> 4], dim=-1).long()]
    return _mx_scaled(u.reshape(*s.shape, MX_BLOCK), s).reshape(*q.shape[:-1], -1)


def mx_product(rows: MxRows, w: MxWeight, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Reference product in fp32."""
    y = mx_dequantize(rows) @ mx_weight_dense(w)[:, :rows.width].t()
    return y if bias is None else y + bias.to(torch.float32)


def mx_gated(h: torch.Tensor, limit: float, alpha: float) -> torch.Tensor:
    """The gated activation of ``h = [gate | up]``: SiLU(gate) * up, or with a limit the clamped form of gpt-oss."""
    g, u = h.chunk(2, dim=-1)
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return (u + 1) * g * torch.sigmoid(alpha * g)
    return g * torch.sigmoid(g) * u
