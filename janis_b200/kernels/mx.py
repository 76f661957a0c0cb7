"""8-bit rows and 4-bit weights: the two microscaling forms, and the kernels that make and take them.

32 values that lie together along a row share a scale that is a power of two.  Rows of activations (`MxRows`) hold e4m3 values,
weights (`MxWeight`) e2m1 values.  A group's scale is the smallest power of two that brings its largest magnitude under the
type's largest value (448 and 6), so nothing saturates; a group of zeros has scale 1, a group that holds an infinity or a NaN stands
for NaN.  `codes` is uint8: [rows, K'] for e4m3 and [N, K' / 2] for e2m1 (the lower half of a byte first), K' the width
padded to a multiple of 128 with zeros.  `scales` is uint8 [rows / 128, K' / 128, 512] (rounded up): s stands for 2^(s - 127), 255
for NaN; a block of 512 is [row % 32][row / 32][group], as the tensor cores take it.

The names here are also those of `ops`, whose `rmsnorm`, `add_rmsnorm` and `gated_act` take `MxRows` as their `out`.
"""
from __future__ import annotations

import struct

import torch

from . import ops as _ops

GROUP, BLOCK = 32, 128

# The two calls of a decode step hand their arguments over as one block of 8-byte fields: ctypes takes 1.8 us to convert
# sixteen arguments and 0.4 us for a block, of some 5 us that a call of a few rows lasts on the device.
_PRODUCT = struct.Struct("=12q3dq").pack
_NORM = struct.Struct("=6qd1qd6q").pack


def _padded(k: int) -> int:
    return (k + BLOCK - 1) // BLOCK * BLOCK


_U8, _F32 = torch.uint8, torch.float32


class _Mx:
    """`rows` x `width` values in one of the two forms."""

    __slots__ = ("codes", "scales", "rows", "width")
    bits = 0

    def __init__(self, codes, scales, rows: int, width: int):
        try:
            kp = (width + 127) // 128
            fine = (rows >= 0 < width and codes.is_cuda and scales.is_cuda and codes.dtype is _U8 and scales.dtype is _U8
                    and codes.shape == (rows, kp * 16 * self.bits) and scales.shape == ((rows + 127) // 128, kp, 512)
                    and codes.is_contiguous() and scales.is_contiguous() and not (codes.data_ptr() | scales.data_ptr()) & 31)
        except (AttributeError, TypeError):
            fine = False
        if not fine:
            self._refuse(codes, scales, rows, width)
        self.codes, self.scales, self.rows, self.width = codes, scales, rows, width

    def _refuse(self, codes, scales, rows, width):
        """Says what is wrong with them."""
        if not isinstance(rows, int) or not isinstance(width, int) or rows < 0 or width < 1:
            raise _ops.KernelError(f"{type(self).__name__}: {rows} rows of {width} values")
        kp = _padded(width)
        _ops._t(codes, "codes", torch.uint8, (rows, kp * self.bits // 8))
        _ops._t(scales, "scales", torch.uint8, (_padded(rows) // BLOCK, kp // BLOCK, 512))
        raise _ops.KernelError(f"{type(self).__name__}: codes and scales must start on 32 bytes")

    @classmethod
    def empty(cls, rows: int, width: int, device="cuda"):
        """Room for `rows` x `width` values, all zero."""
        kp = _padded(width)
        return cls(torch.zeros(rows, kp * cls.bits // 8, dtype=torch.uint8, device=device),
                   torch.full((_padded(rows) // BLOCK, kp // BLOCK, 512), 127, dtype=torch.uint8, device=device), rows, width)

    @property
    def shape(self):
        return (self.rows, self.width)

    @property
    def device(self):
        return self.codes.device

    def values(self, out=None):
        """The values it stands for, [rows, width] (float32 where no `out` is given)."""
        if out is None:
            out = torch.empty(self.rows, self.width, dtype=torch.float32, device=self.codes.device)
        lib = _ops.low_bits()
        _ops._check(lib, lib.janis_mx_values(self.codes.data_ptr(), self.scales.data_ptr(), self.bits,
                                             _ops._t(out, "out", _ops._FLOATS, self.shape), _ops._DT[out.dtype], self.rows, self.width,
                                             _ops._stream()))
        return out


class MxRows(_Mx):
    """Rows of activations in 8 bits."""
    __slots__ = ()
    bits = 8


class MxWeight(_Mx):
    """Rows of a weight matrix in 4 bits."""
    __slots__ = ()
    bits = 4

    def __getitem__(self, rows: slice) -> "MxWeight":
        """Its first rows, over the same memory."""
        if not isinstance(rows, slice) or rows.start not in (None, 0) or rows.step not in (None, 1):
            raise IndexError("4-bit weights are cut behind their first rows only: w[:n]")
        n = len(range(*rows.indices(self.rows)))
        return MxWeight(self.codes[:n], self.scales[:_padded(n) // BLOCK], n, self.width)


def _rows(x, name, rows, width):
    if type(x) is not MxRows:
        raise _ops.KernelError(f"{name}: expected MxRows, found {type(x).__name__}")
    if x.rows != rows or x.width != width:
        raise _ops.KernelError(f"{name}: shape {x.shape} does not match {(rows, width)}")
    return x.codes.data_ptr(), x.scales.data_ptr()


def mx_rows(x, out: MxRows) -> MxRows:
    """out = x [R, K] in 8 bits."""
    R, K = x.shape
    lib = _ops.low_bits()
    _ops._check(lib, lib.janis_mx_rows(_ops._t(x, "x", _ops._FLOATS), _ops._DT[x.dtype], -1, 0.0, 0.0, 0.0, *_rows(out, "out", R, K), R, K,
                                       _ops._stream()))
    return out


def mx_weight(w) -> MxWeight:
    """A weight matrix w [N, K] in 4 bits."""
    N, K = w.shape
    p, out, lib = _ops._t(w, "w", _ops._FLOATS), MxWeight.empty(N, K, w.device), _ops.low_bits()
    _ops._check(lib, lib.janis_mx_weight(p, _ops._DT[w.dtype], out.codes.data_ptr(), out.scales.data_ptr(), N, K, _ops._stream()))
    return out


def norm_to_rows(h, res, w_post, eps_post, w_next, eps_next, out: MxRows, n_part: int = 1, rows=None) -> MxRows:
    """`rmsnorm` (res None) and `add_rmsnorm` with 8-bit rows as their output."""
    lib = _ops._low_bits or _ops.low_bits()
    shape, wide = h.shape, (out.width,)
    # what a decode step calls, checked at once; whatever is not this is looked at one by one below
    if (res is not None and w_next is not None and n_part == 1 and rows is None and shape == (out.rows, out.width) == res.shape
            and (w_post is None or (w_post.dtype is _F32 and w_post.shape == wide and w_post.is_contiguous() and w_post.is_cuda))
            and w_next.dtype is _F32 and w_next.shape == wide and w_next.is_contiguous() and w_next.is_cuda
            and h.dtype is _F32 and h.is_contiguous() and h.is_cuda and res.is_contiguous() and res.is_cuda and res.dtype in _ops._DT):
        _ops._check(lib, lib.janis_mx_norm_rows(_NORM(
            h.data_ptr(), res.data_ptr(), _ops._DT[res.dtype], 1, 0, w_post.data_ptr() if w_post is not None else 0, eps_post,
            w_next.data_ptr(), eps_next, 0, out.codes.data_ptr(), out.scales.data_ptr(), out.rows, out.width, _ops._stream())))
        return out
    H = shape[1]
    R = out.rows if res is None else shape[0]
    if n_part < 1:
        raise _ops.KernelError("add_rmsnorm: n_part must be >= 1")
    if w_next is None:
        raise _ops.KernelError("add_rmsnorm: 8-bit rows are the second norm's output, which has no weight here")
    t = _ops._t
    if res is None:
        if rows is None and h.shape[0] != R:
            raise _ops.KernelError(f"rmsnorm: {h.shape[0]} input rows for {R} output rows")
        p_res, dt, stride = 0, 0, 0
    else:
        p_res, dt, stride = t(res, "res", _ops._FLOATS, (R, H) if n_part == 1 else (n_part, R, H)), _ops._DT[res.dtype], R * H
    block = _NORM(t(h, "h", torch.float32, (None, H)), p_res, dt, n_part, stride,
                  t(w_post, "w_post", torch.float32, (H,)) if w_post is not None else 0, eps_post,
                  t(w_next, "w_next", torch.float32, (H,)), eps_next, t(rows, "rows", torch.int32, (R,)) if rows is not None else 0,
                  *_rows(out, "out", R, H), R, H, _ops._stream())
    _ops._check(lib, lib.janis_mx_norm_rows(block))
    return out


def gated_to_rows(gu, out: MxRows, act: int, group: int, limit: float, alpha: float, up_add: float) -> MxRows:
    """`gated_act` with 8-bit rows as its output."""
    R, I2 = gu.shape
    if group != _ops.GATE_GROUP:
        raise _ops.KernelError(f"gated_act: 8-bit rows come from gates and ups in groups of {_ops.GATE_GROUP}, found {group}")
    if act not in (_ops.ACT_GELU_TANH, _ops.ACT_SILU, _ops.ACT_CLAMPED):
        raise _ops.KernelError(f"gated_act: unknown activation {act}")
    lib = _ops.low_bits()
    _ops._check(lib, lib.janis_mx_rows(_ops._t(gu, "gu", _ops._FLOATS, (R, I2 // 2 * 2)), _ops._DT[gu.dtype], int(act), float(limit), float(alpha), float(up_add),
                                       *_rows(out, "out", R, I2 // 2), R, I2 // 2, _ops._stream()))
    return out


def mx_set_few(split: int = 0, stages: int = 0) -> None:
    """Fixes how many CTAs share K (1, 2, 4, 8) and the depth of the ring in products of few rows (0: chosen).  For tests and tuning."""
    _ops.low_bits().janis_mx_set_few(int(split), int(stages))


def mx_set_kernel(kernel: int = 0) -> None:
    """Fixes the kernel of products: 0 chosen by their sizes, 1 few rows, 2 and 3 many rows by pairs of CTAs and by one, 4 many rows whose K
    is shared by the CTAs of `mx_set_few`, 5, 6 and 7 the same by 2, 4 and 8 of them.  For tests and tuning."""
    _ops.low_bits().janis_mx_set_kernel(int(kernel))


def linear_mx(x: MxRows, w: MxWeight, out, epilogue: int = 0, limit: float = 0.0, alpha: float = 1.0, up_add: float = 0.0):
    """out[T, N] = x w^T of 8-bit rows and 4-bit weights, float sums; out bfloat16 or float32.  With a gated epilogue
    (EPI_GATED_GELU, EPI_GATED_SILU, EPI_GATED_CLAMP with its three numbers) the rows of w alternate 8 gates, 8 ups and
    out[T, N / 2] = act(gate) * up; it may be `MxRows` then.  Like every product of this library it takes w for a constant: its first
    tiles are fetched while the kernel in front of this one still runs."""
    if type(x) is not MxRows or type(w) is not MxWeight:
        raise _ops.KernelError(f"linear_mx: x must be MxRows and w MxWeight, found {type(x).__name__} and {type(w).__name__}")
    T, K, N = x.rows, x.width, w.rows
    if w.width != K:
        raise _ops.KernelError(f"linear_mx: x has {K} columns and w {w.width}")
    cols = N // 2 if epilogue else N                      # (EPI_NONE is 0)
    if type(out) is MxRows:
        if not epilogue:
            raise _ops.KernelError("linear_mx: 8-bit rows are a gated epilogue's output")
        p_out, dt, (pc, ps) = 0, 0, _rows(out, "out", T, cols)
    else:
        dt = _ops._DT.get(getattr(out, "dtype", None))
        if dt is None or out.shape != (T, cols) or not out.is_cuda or not out.is_contiguous():
            _ops._t(out, "out", _ops._FLOATS, (T, cols))                  # (says what is wrong with it)
        p_out, pc, ps = out.data_ptr(), 0, 0
    lib = _ops._low_bits or _ops.low_bits()
    _ops._check(lib, lib.janis_mx_product(_PRODUCT(
        x.codes.data_ptr(), x.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), p_out, dt, pc, ps, T, N, K, epilogue,
        limit, alpha, up_add, _ops._stream())))
    return out
