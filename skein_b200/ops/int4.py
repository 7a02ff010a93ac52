"""Products with weights of 4 bits and group scales: W[f, k] = scale[f, k / group] (code[f, k] - zero[f, k / group]).

Codes are 0 .. 15, a zero is 0 .. 15 (8 where there is none), a group is 32, 64 or 128 neighbours along K, scales are bf16 or fp16. Activations are
bf16 and are not quantised; sums, the scales' products included, are fp32, and nothing is rounded before the result. Beside ops/fp8.py this is the other
form of weights narrower than the activations: half its bytes, scales of finer groups.

A weight is laid out once (`pack_weight` from codes, `quantize_weight` from a matrix) for the kernels: csrc/kernels/int4.cuh has the layout. On CPU the
same mathematics run through the reference (dequantise, matmul; reference_int4.py).
"""
from __future__ import annotations

import torch

from . import _lib, functional as F, reference_int4 as ri

GROUPS = (32, 64, 128)
STEP = 128                 # elements of K of a packed block (16 rows)
CODES = 16 * STEP // 2     # its bytes of codes
MAX_EXPERTS = 1024
MAX_ROW = 1 << 16       # of K in the kernel of few rows, which keeps whole rows of x in shared memory


def _data_shape(shape, group, pair, scales, zeros):
    """Of the packed weight [rows, K] or [experts, rows, K]."""
    if len(shape) not in (2, 3) or min(shape) < 1 or group not in GROUPS or shape[-1] % group:
        raise ValueError(f"int4 weight: [rows, K] or [experts, rows, K] with K a multiple of the group ({GROUPS}), not {tuple(shape)} in groups of {group}")
    n, rows = shape[0] if len(shape) == 3 else 1, shape[-2]
    if n > MAX_EXPERTS:
        raise ValueError(f"int4 weight: at most {MAX_EXPERTS} experts")
    if pair and rows % 2:
        raise ValueError("int4 weight: a pair has as many up rows as gate rows")
    if scales not in (torch.bfloat16, torch.float16):
        raise ValueError("int4 weight: scales are bf16 or fp16")
    tiles = -(-rows // 2 // 64) if pair else -(-rows // 128)
    return (n, tiles, -(-shape[-1] // STEP), 8 * (CODES + STEP // group * (48 if zeros else 32)))


class Int4Weight:
    """data uint8 [matrices, tiles, steps, bytes]: codes, scales and zeros of 128 rows x 128 of K (csrc/kernels/int4.cuh). `shape` is the logical [rows, K]
    or [experts, rows, K]; `pair`: gate rows, then up rows, packed side by side for the SwiGLU product."""

    def __init__(self, data, shape, group, pair, scales, zeros):
        want = _data_shape(shape, group, pair, scales, zeros)
        if data.dtype != torch.uint8 or data.shape != want or not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError(f"int4 weight: data must be contiguous uint8 {want} on a 16-byte boundary")
        self.data, self.shape, self.group, self.pair = data, tuple(shape), group, pair
        self.scales, self.zeros = scales, zeros
        self.K, self.matrices = shape[-1], want[0]
        self.features = shape[-2] // 2 if pair else shape[-2]
        self.flags = int(pair) | (2 if scales == torch.float16 else 0) | (8 if zeros else 0)

    # (asked of the storage each time: a copied, pickled or moved weight has another one)
    @property
    def is_cuda(self):
        return self.data.is_cuda

    @property
    def device(self):
        return self.data.device

    @property
    def ptr(self):
        return self.data.data_ptr()

    def nbytes(self) -> int:
        return self.data.numel()

    def parts(self):
        """(codes [..., rows, K / 2], scale [..., rows, K / group], zero or None) as pack_weight takes them."""
        *lead, rows, K = self.shape
        n, per = self.data.shape[0], STEP // self.group
        S, B = 8 * self.data.shape[1], self.data.shape[2]
        codes, scale, zero = self.data.split((8 * CODES, 8 * 32 * per, 8 * 16 * per if self.zeros else 0), -1)
        w = codes.contiguous().view(torch.int32).view(n, S // 8, B, 8, 2, 4, 8, 2, 2).permute(0, 1, 3, 7, 6, 2, 4, 8, 5)   # [n, S, half, g, B, j, h, t]
        w = _rows_out(w.reshape(n, S, 2, 8, B * 16), self.pair, rows)[:, :, :K // 8]

        def back(t):
            u = t.view(n, S // 8, B, 8, 8, per, 2).permute(0, 1, 3, 6, 4, 2, 5).reshape(n, S, 2, 8, -1)
            return _rows_out(u, self.pair, rows)[:, :, :K // self.group].reshape(*lead, rows, K // self.group)
        return (_interleave(w.contiguous()).view(torch.uint8).reshape(*lead, rows, K // 2), back(scale.contiguous().view(self.scales)),
                back(zero.contiguous()) if self.zeros else None)

    def dequant(self) -> torch.Tensor:
        """The weight in fp32, in its logical shape."""
        return ri.dequant(*self.parts(), self.group)

    def copy_(self, src: "Int4Weight"):
        """In-place update (hot swap keeps the storage that captured CUDA graphs point at)."""
        if (src.shape, src.group, src.pair, src.scales, src.zeros) != (self.shape, self.group, self.pair, self.scales, self.zeros):
            raise ValueError("int4 weight: another shape, group, pairing or type of scales")
        self.data.copy_(src.data)
        return self


def _deinterleave(w):
    """Words of eight codes in order -> codes of even k in the low half, of odd k in the high half."""
    def squeeze(v):
        v = (v | (v >> 4)) & 0x00FF00FF
        return (v | (v >> 8)) & 0x0000FFFF
    return squeeze(w & 0x0F0F0F0F) | (squeeze((w >> 4) & 0x0F0F0F0F) << 16)


def _interleave(w):
    def spread(v):
        v = (v | (v << 8)) & 0x00FF00FF
        return (v | (v << 4)) & 0x0F0F0F0F
    return spread(w & 0xFFFF) | (spread((w >> 16) & 0xFFFF) << 4)


def _rows_in(t, pair, strips):
    """[n, rows, ...] -> [n, strips, 2, 8, ...], rows padded with zeros."""
    n, rows = t.shape[:2]
    parts = t.reshape(n, 2, rows // 2, *t.shape[2:]) if pair else t.unsqueeze(1)
    pad = strips * (8 if pair else 16) - parts.shape[2]
    if pad:
        parts = torch.cat((parts, parts.new_zeros(*parts.shape[:2], pad, *parts.shape[3:])), 2)
    if pair:
        return parts.reshape(n, 2, strips, 8, *t.shape[2:]).transpose(1, 2)
    return parts.reshape(n, strips, 2, 8, *t.shape[2:])


def _rows_out(t, pair, rows):
    """[n, strips, 2, 8, m] -> [n, rows, m]."""
    n, S, _, _, m = t.shape
    if pair:
        return t.transpose(1, 2).reshape(n, 2, S * 8, m)[:, :, :rows // 2].reshape(n, rows, m)
    return t.reshape(n, S * 16, m)[:, :rows]


def pack_weight(codes, scale, zero=None, pair=False) -> Int4Weight:
    """codes uint8 [rows, K / 2] or [experts, rows, K / 2], two to a byte (the even k in the low half); scale bf16 or fp16 [.., rows, K / group]; zero
    uint8 of scale's shape, 0 .. 15, or None (all 8). pair: the first half of the rows are the gate, the second half the up projection of a SwiGLU."""
    if codes.dim() not in (2, 3) or codes.dtype != torch.uint8 or codes.numel() == 0:
        raise ValueError("int4 weight: codes must be uint8 [rows, K / 2] or [experts, rows, K / 2]")
    *lead, rows, half = codes.shape
    K = 2 * half
    if scale.dtype not in (torch.bfloat16, torch.float16) or scale.shape[:-1] != codes.shape[:-1] or scale.shape[-1] == 0 or K % scale.shape[-1]:
        raise ValueError("int4 weight: scale must be bf16 or fp16 [.., rows, K / group]")
    group = K // scale.shape[-1]
    if group not in GROUPS:
        raise ValueError(f"int4 weight: groups of {group}; they are {GROUPS}")
    if zero is not None:
        if zero.dtype != torch.uint8 or zero.shape != scale.shape:
            raise ValueError("int4 weight: zero must be uint8 of scale's shape")
        if int(zero.max()) > 15:
            raise ValueError("int4 weight: zeros are 0 .. 15")
    if any(t is not None and t.device != codes.device for t in (scale, zero)):
        raise ValueError("int4 weight: codes, scale and zero lie on different devices")
    n, tiles, B, _ = size = _data_shape((*lead, rows, K), group, pair, scale.dtype, zero is not None)
    S = 8 * tiles
    codes = codes.reshape(n, rows, half).contiguous()
    if codes.storage_offset() % 4:           # (a part of a buffer of bytes)
        codes = codes.clone()
    w = _rows_in(_deinterleave(codes.view(torch.int32)), pair, S)                                            # [n, S, half, g, K / 8]
    w = torch.nn.functional.pad(w, (0, B * 16 - w.shape[-1])) if w.shape[-1] < B * 16 else w
    per = STEP // group
    data = codes.new_empty(size)
    to = data[..., :8 * CODES].view(torch.int32).view(n, S // 8, B, 8, 2, 4, 8, 2, 2)                        # [n, tile, B, strip, j, t, g, half, h]
    to.copy_(w.reshape(n, S // 8, 8, 2, 8, B, 2, 2, 4).permute(0, 1, 5, 2, 6, 8, 4, 3, 7))

    def lay(t, first, size):
        t = _rows_in(t.reshape(n, rows, -1), pair, S)
        if t.shape[-1] < B * per:
            t = torch.nn.functional.pad(t, (0, B * per - t.shape[-1]))
        to = data[..., first:first + size].view(t.dtype).view(n, S // 8, B, 8, 8, per, 2)                    # [n, tile, B, strip, g, group, half]
        to.copy_(t.reshape(n, S // 8, 8, 2, 8, B, per).permute(0, 1, 5, 2, 4, 6, 3))
    lay(scale, 8 * CODES, 8 * 32 * per)
    if zero is not None:
        lay(zero, 8 * (CODES + 32 * per), 8 * 16 * per)
    return Int4Weight(data, (*lead, rows, K), group, bool(pair), scale.dtype, zero is not None)


def quantize_weight(w: torch.Tensor, group: int = 128, symmetric: bool = True, pair: bool = False) -> Int4Weight:
    """Nearest codes of a weight [rows, K] or [experts, rows, K]. symmetric: a group's scale maps its largest magnitude to 7 (codes 1 .. 15 around 8);
    else scale and zero map its range, zero included, onto 0 .. 15. Scales are bf16. K must be a multiple of the group, the weight finite."""
    if w.dim() not in (2, 3) or group not in GROUPS or w.shape[-1] % group:
        raise ValueError(f"int4 weight: [.., rows, K] with K a multiple of the group ({GROUPS})")
    v = w.float().unflatten(-1, (-1, group))
    if symmetric:
        s, zero = v.abs().amax(-1) / 7, None
    else:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        s = (hi - lo) / 15
    if not bool(s.isfinite().all()):
        raise ValueError("int4 weight: a group holds what is not finite, or spans more than 32-bit numbers do")
    s = torch.where(s > 0, s, torch.ones_like(s)).to(torch.bfloat16)
    if not symmetric:
        zero = (-lo / s.float()).round().clamp(0, 15).to(torch.uint8)
    z = 8.0 if zero is None else zero.float()[..., None]
    q = ((v / s.float()[..., None]).round() + z).clamp(0, 15).to(torch.uint8).flatten(-2)
    return pack_weight(q[..., 0::2] | (q[..., 1::2] << 4), s, zero, pair)


def _check(what, x, w: Int4Weight, pair, dims):
    if not isinstance(w, Int4Weight) or len(w.shape) != dims:
        raise ValueError(f"{what}: the weight must be an Int4Weight of {dims} dimensions")
    if w.pair != pair:
        raise ValueError(f"{what}: the weight is {'' if w.pair else 'not '}packed as a gate / up pair")
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != w.K or x.stride(1) != 1:
        raise ValueError(f"{what}: x must be bf16 [rows, {w.K}] with contiguous rows")
    if x.device != w.data.device:
        raise ValueError(f"{what}: x is on {x.device}, the weight on {w.device}")


def _meet(a, b) -> bool:
    """Whether two matrices with contiguous rows share a byte. Rows of the same distance (columns of one buffer, every other row of it) are compared at once,
    others row by row, and only where the spans meet."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    if a.shape[0] > b.shape[0]:
        a, b = b, a
    p, n, step, size = a.data_ptr(), a.shape[0], a.stride(0) * a.element_size(), a.shape[1] * a.element_size()
    q, m, other, wide = b.data_ptr(), b.shape[0], b.stride(0) * b.element_size(), b.shape[1] * b.element_size()
    if p + (n - 1) * step + size <= q or q + (m - 1) * other + wide <= p:
        return False
    if m == 1 or other == 0:        # (a row that repeats is one row)
        m = other = 1
    if n == 1 or step == 0:
        n, step = 1, other
    if step == other:               # rows i and j meet where (i - j) step lies between q - p - size and q - p + wide: the first that does
        d = max((q - p - size) // step + 1, 1 - m)
        return d < n and d * step < q - p + wide
    for at in range(p, p + n * step, step):
        j = max((at - wide - q) // other + 1, 0)
        if j < m and q + j * other < at + size:
            return True
    return False


def _check_out(what, out, x, rows, w, dtype):
    if out.shape != (rows, w.features) or out.dtype != dtype or out.device != x.device or out.stride(1) != 1 or (rows > 1 and out.stride(0) < w.features):
        raise ValueError(f"{what}: out must be {dtype} [{rows}, {w.features}] with contiguous rows that do not overlap")
    p, q = out.data_ptr(), x.data_ptr()
    size = 4 if dtype is torch.float32 else 2
    # (the spans first: a call that takes 10 us has no 2 for the rest)
    if p < q + 2 * ((x.shape[0] - 1) * x.stride(0) + w.K) and q < p + size * ((rows - 1) * out.stride(0) + w.features) and _meet(out, x):
        raise ValueError(f"{what}: out lies on x, which is read until the end")


def _few_rows(hint: int, K: int, grouped: bool) -> bool:
    """Whether a product with `hint` rows per matrix runs on the kernel of few rows (csrc/kernels/int4_rows.cu) instead of the one on tensor memory
    (int4_tc.cu), which has more to set up and is the quicker one from where a warp's share of the rows of x costs more than the conversion. Measured, few
    rows / tensor memory, us: 4096 x 4096 7.4 / 9.6 at 1 row, 9.8 / 9.9 at 8, 12.7 / 10.0 at 16; 4096 x 14336 13.9 / 17.4 at 1, 16.9 / 17.6 at 4, 25.5 / 17.6
    at 7; gate / up 14336 x 4096 25.3 / 29.8 at 1, 29.1 / 29.8 at 8, 37.8 / 29.8 at 16.
    With experts the tensor-memory kernel takes two tiles at a time, and the mean of unequal rows is asked. 8 experts, gate / up 14336 x 4096: 35.4 / 43.6 at 1
    token, 90 / 92 at a mean of 2 rows, 117 / 124 at 3, 130 / 125 at 4; 4096 x 14336 61 / 75 at 2, 66 / 75 at 3, 79 / 75 at 4. 64 experts, gate / up 1408 x
    2048: 26.9 / 31 at 0.4, 41.9 / 41.9 at 0.75, 53 / 54 at 1.5, 61 / 55 at 2.3; 2048 x 1408 26 / 24 at 0.75, 35 / 25 at 1.5. 128 experts, 2048 x 768: 21 / 20
    at 0.25, 32 / 25 at 1."""
    if grouped:
        return hint << 10 < min(K, 1 << 12) and K <= MAX_ROW
    return hint <= 8 and hint * K <= MAX_ROW


_STATUS: dict = {}      # device -> address of the status word of its workspace, which is made once


def _status(device) -> int:
    at = _STATUS.get(device)
    if at is None:
        at = _STATUS[device] = F.workspace(device).status.data_ptr()
    return at


def _launch(what, x, w: Int4Weight, out, residual, counts, offsets, src_row, rows, hint, flags, cfg=None):
    """cfg: None (the rule) or (n_tile, split) of the tensor-memory kernel, (0, team) of the kernel of few rows."""
    L, dev = _lib.lib(), x.device
    xp, x_ld = x.data_ptr(), x.stride(0) if x.shape[0] > 1 else w.K
    few = _few_rows(hint, w.K, counts is not None) if cfg is None else cfg[0] == 0
    if xp % 16 or x_ld % 8:
        if w.K > MAX_ROW:
            raise ValueError(f"{what}: rows of x off 16-byte boundaries have at most {MAX_ROW} elements, not {w.K}")
        if not few:     # (few rows are read two bytes at a time; 1000 rows of gate / up 18944 x 3584 so took 1770 us, laid out anew 253)
            x = x.clone(memory_format=torch.contiguous_format)
            xp, x_ld = x.data_ptr(), w.K
    args = (xp, x_ld, None if src_row is None else src_row.data_ptr(), w.data.data_ptr(), None if residual is None else residual.data_ptr(), out.data_ptr(),
            out.stride(0), None if counts is None else counts.data_ptr(), None if counts is None else offsets.data_ptr(), rows, x.shape[0], w.matrices,
            w.features, w.K, w.group, hint, flags)
    if few:
        rc = L.skein_int4_rows(*args, cfg[1] if cfg else 0, _status(dev), _lib.stream_on(dev))
    else:
        rc = L.skein_int4_tc(*args, *(cfg or (0, 0)), _status(dev), _lib.stream_on(dev))
    _lib.check(rc, what)
    _lib.count_launch()


def linear(x, w: Int4Weight, out=None, residual=None, out_f32=False, _cfg=None):
    """y[t, f] = sum_k x[t, k] W[f, k] (+ residual[t, f]) for bf16 x [T, K] (rows may be strided). out_f32: y and the residual are fp32, else both are
    bf16. out may be a run of columns of a wider matrix; it shares no memory with x, nor with the residual unless it is the residual."""
    _check("int4 linear", x, w, False, 2)
    return _dense("int4 linear", x, w, out, residual, out_f32, _cfg)


def swiglu_linear(x, w: Int4Weight, out=None, _cfg=None):
    """silu(x Wg^T) * (x Wu^T) with both products from one pass over x; w is packed as a pair; out as in `linear`."""
    _check("int4 swiglu_linear", x, w, True, 2)
    return _dense("int4 swiglu_linear", x, w, out, None, False, _cfg)


def _dense(what, x, w, out, residual, out_f32, cfg):
    T = x.shape[0]
    dtype = torch.float32 if out_f32 else torch.bfloat16
    given = out is not None
    if given:
        _check_out(what, out, x, T, w, dtype)
    else:
        out = torch.empty((T, w.features), dtype=dtype, device=x.device)
    if residual is not None and (residual.shape != out.shape or residual.dtype != out.dtype or residual.device != out.device
                                 or residual.stride(1) != 1 or (T > 1 and residual.stride(0) != out.stride(0))):
        raise ValueError(f"{what}: the residual must have the result's shape, type and strides")
    if given and residual is not None and residual.data_ptr() != out.data_ptr() and _meet(residual, out):
        raise ValueError(f"{what}: the residual is out itself or lies beside it")
    if T == 0:
        return out
    if not x.is_cuda:
        return out.copy_(ri.product(x, w.dequant(), residual, out_f32, w.pair))
    with _lib.on_device(x):
        _launch(what, x, w, out, residual, None, None, None, T, T, w.flags | (4 if out_f32 else 0), cfg)
    return out


def grouped_linear(x, w: Int4Weight, counts, offsets, swiglu=False, src_row=None, out=None, rows_hint=None, _cfg=None):
    """Per-expert linear over expert-sorted rows. counts / offsets are int32 device tensors of E (offsets may have E + 1) entries: rows of expert e are
    offsets[e] : offsets[e] + counts[e] of the result, no row belongs to two. They read the same rows of x, or with src_row (int32, one entry per row of the result) rows
    src_row[r]: the tokens themselves, without a sorted copy. Rows not covered by any expert are left untouched (uninitialised in a result that the call
    makes); out shares no memory with x. rows_hint: rows expected over all experts, on which the choice of kernel depends (default: all of the result's)."""
    what = "int4 grouped_linear"
    _check(what, x, w, bool(swiglu), 3)
    E = w.shape[0]
    for t, name, least in ((counts, "counts", E), (offsets, "offsets", E)):
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] < least or not t.is_contiguous() or t.device != x.device:
            raise ValueError(f"{what}: {name} must be int32 [{E}] on x's device")
    if src_row is not None and (src_row.dtype != torch.int32 or src_row.dim() != 1 or not src_row.is_contiguous() or src_row.device != x.device):
        raise ValueError(f"{what}: src_row must be int32 [rows] on x's device")
    rows = x.shape[0] if src_row is None else src_row.shape[0]
    if out is None:
        out = torch.empty((rows, w.features), dtype=torch.bfloat16, device=x.device)
    else:
        _check_out(what, out, x, rows, w, torch.bfloat16)
    if rows == 0:
        return out
    if x.shape[0] == 0:
        raise ValueError(f"{what}: src_row names rows of an empty x")
    if not x.is_cuda:
        return ri.grouped_product(x, w.dequant(), counts[:E], offsets[:E], swiglu, src_row, out)
    hint = -(-(rows if rows_hint is None else max(1, min(int(rows_hint), rows))) // E)
    with _lib.on_device(x):
        _launch(what, x, w, out, None, counts, offsets, src_row, rows, hint, w.flags, _cfg)
    return out
