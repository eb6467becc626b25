"""Matrices in microscaled 4-bit floating point (MXFP4) and the operations on them.

The format (OCP Microscaling Formats, MXFP4): every 32 neighbouring elements of a row share a scale
2^(e - 127), one byte (255: the block reads as NaN), and an element is a sign and one of the
magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6: 4.25 bits an element.  ``Mx4Matrix`` holds such a matrix as
the matrix cores take it (csrc/mx4.h says how it lies).
"""
import ctypes

import torch

from ..errors import KernelError

_vp, _i, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t

BLOCK = 32              # elements that share a scale
TILE_ROWS, QUAD = 16, 512      # a tile holds 16 rows by whole quads of 512 elements

SIGNATURES = {
    "llm_mx4_quantize": [_vp, _i, _sz, _i, _i, _vp, _vp, _vp],
    "llm_mx4_dequantize": [_vp, _vp, _vp, _i, _i, _i, _vp],
    "llm_mx4_pack": [_vp, _sz, _vp, _i, _i, _vp, _vp, _vp],
    "llm_pad_rows": [_vp, _sz, _vp, _i, _i, _i, _vp],
    "llm_gemm_mx4_rows": [_vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp],
    "llm_gemm_mx4_many": [_vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp],
    "llm_mx4_join": [_vp, _i, _vp, _vp, _i, _i, _i, _i, _vp],
}


def tiled_sizes(rows: int, width: int):
    """(bytes of codes, bytes of scales) of a matrix of these sizes, whole tiles."""
    tiles, quads = -(-rows // TILE_ROWS), -(-width // QUAD)
    return tiles * quads * 4096, tiles * quads * 256


class Mx4Matrix:
    """A matrix ``[rows, width]`` in MXFP4: ``codes`` and ``scales`` are uint8 tensors in the order
    the matrix cores read them.  What ``HipOps.quantize_mx4`` and ``HipOps.mx4_from_codes`` return, and the
    products take as a weight, or on both sides."""
    dtype = "mxfp4"

    def __init__(self, shape, codes, scales):
        self.shape, self.codes, self.scales = tuple(shape), codes, scales

    @property
    def device(self):
        return self.codes.device

    def leading_rows(self, rows: int) -> "Mx4Matrix":
        """The first ``rows`` rows, a multiple of 16, in the same storage."""
        if rows % TILE_ROWS or not 0 < rows <= self.shape[0]:
            raise KernelError("the leading rows of an MXFP4 matrix are a multiple of %d (asked for %d of %d)"
                              % (TILE_ROWS, rows, self.shape[0]))
        codes, scales = tiled_sizes(rows, self.shape[1])
        return Mx4Matrix((rows, self.shape[1]), self.codes[:codes], self.scales[:scales])


class Mx4Ops:
    """The operations of ``HipOps`` on matrices in MXFP4."""

    MX4_ROWS = 32           # most rows that go to the product for few rows

    def _mx4_empty(self, rows, width):
        if rows <= 0 or width <= 0:
            raise KernelError("an MXFP4 matrix has rows and columns, not [%d, %d]" % (rows, width))
        if max(rows, width) >= 1 << 30:
            raise KernelError("an MXFP4 matrix of [%d, %d] is too large" % (rows, width))
        codes, scales = tiled_sizes(rows, width)
        return Mx4Matrix((rows, width), torch.empty(codes, dtype=torch.uint8, device=self.device),
                         torch.empty(scales, dtype=torch.uint8, device=self.device))

    def _mx4(self, q, what):
        """Checks a matrix in MXFP4; returns the pointers to its codes and scales."""
        if not isinstance(q, Mx4Matrix):
            raise KernelError("%s is no MXFP4 matrix" % what)
        codes, scales = tiled_sizes(*q.shape)
        return (self._dev(q.codes, what + " codes", torch.uint8, (codes,)),
                self._dev(q.scales, what + " scales", torch.uint8, (scales,)))

    def quantize_mx4(self, x) -> Mx4Matrix:
        """The matrix ``x`` (bfloat16 or float32, rows contiguous; they may lie further apart than
        their length) in MXFP4.  The scale of a block is 2^(floor(log2(max |x|)) - 2), at least
        2^-127; an element is divided by it and rounded to the nearest code, ties to the even one,
        6 beyond 6.  A block that holds an infinity or a NaN reads as NaN."""
        from .ops import _code
        self._weight(x, "the matrix to quantise")
        q = self._mx4_empty(*x.shape)
        self._check(self.lib.llm_mx4_quantize(
            x.data_ptr(), _code(x.dtype), max(x.stride(0), x.shape[1]), x.shape[0], x.shape[1], q.codes.data_ptr(), q.scales.data_ptr(),
            self._stream()), "quantize_mx4")
        return q

    def dequantize_mx4(self, q: Mx4Matrix, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers that ``q`` stands for, exactly (a scale above 2^125 can give an infinity)."""
        from .ops import _code
        codes, scales = self._mx4(q, "the matrix to read")
        out = torch.empty(q.shape, dtype=dtype, device=self.device)
        self._check(self.lib.llm_mx4_dequantize(codes, scales, out.data_ptr(), _code(dtype), q.shape[0], q.shape[1],
                                                self._stream()), "dequantize_mx4")
        return out

    def mx4_from_codes(self, codes, scales, width=None) -> Mx4Matrix:
        """A matrix that is in MXFP4 already, as files hold it: ``codes`` uint8
        ``[rows, ceil(width / 2)]`` or wider, two elements a byte, the even one in the low half, and
        ``scales`` uint8 ``[rows, ceil(width / 32)]``.  ``width``: twice the columns of ``codes``
        unless it is given (an odd width, padded rows)."""
        if codes.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise KernelError("mx4_from_codes: codes and scales are matrices of uint8")
        self._weight(codes, "the matrix of codes")
        rows, columns = codes.shape
        width = 2 * columns if width is None else int(width)
        if not 0 < -(-width // 2) <= columns:
            raise KernelError("mx4_from_codes: %d columns of codes do not hold rows of %d elements" % (columns, width))
        self._dev(scales, "the matrix of scales", torch.uint8, (rows, -(-width // BLOCK)))
        q = self._mx4_empty(rows, width)
        self._check(self.lib.llm_mx4_pack(codes.data_ptr(), max(codes.stride(0), columns), scales.data_ptr(), rows, width,
                                          q.codes.data_ptr(), q.scales.data_ptr(), self._stream()), "mx4_from_codes")
        return q

    def _mx4_rows(self, x, k, piece):
        """Rows for a product with an MXFP4 weight that reads ``piece`` elements of them at a time:
        (pointer, pointer to scales or None, row stride, what keeps them alive).  bfloat16 rows
        whose length, distance or address does not allow that are copied to a padded buffer first."""
        if isinstance(x, Mx4Matrix):
            codes, scales = self._mx4(x, "linear input")
            return codes, scales, 0, x
        if x.device != self.device:
            raise KernelError("linear input lies on %s, not on %s" % (x.device, self.device))
        if x.dtype != torch.bfloat16:
            raise KernelError("linear: an MXFP4 weight takes rows in bfloat16 or MXFP4, not %s" % (x.dtype,))
        if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < k):
            raise KernelError("linear input must be a matrix with contiguous rows")
        ld = max(x.stride(0), k)
        if k % piece == 0 and ld % piece == 0 and x.data_ptr() % 16 == 0:
            return x.data_ptr(), None, ld, x
        ldp = -(-k // piece) * piece
        padded = torch.empty((x.shape[0], ldp), dtype=torch.bfloat16, device=self.device)
        self._check(self.lib.llm_pad_rows(x.data_ptr(), ld, padded.data_ptr(), x.shape[0], k, ldp, self._stream()),
                    "pad_rows")
        return padded.data_ptr(), None, ldp, padded

    _MX4_FORMS = ((256, 256), (256, 128), (128, 128), (64, 128))
    mx4_force = None

    def _mx4_form(self, m, n, k, epilogue, four):
        if self.mx4_force:
            form, ks = self.mx4_force
            quads = -(-k // QUAD)
            per = -(-quads // min(ks, quads))
            return form, -(-quads // per)
        return 0, 1

    def _mx4_product(self, x, w, out, epilogue, bias=None):
        from .ops import _code
        n, k = w.shape
        m = out.shape[0]
        codes, scales = self._mx4(w, "MXFP4 weight")
        if m == 0:
            return out
        bptr = None if bias is None else self._dev(bias, "bias", torch.float32, (n,))
        if m <= self.MX4_ROWS:
            xp, xs, ldx, alive = self._mx4_rows(x, k, 8)
            # (where rows were padded, K is their padded length: the weight's codes there are zero)
            self._check(self.lib.llm_gemm_mx4_rows(xp, xs, ldx, codes, scales, bptr, out.data_ptr(), epilogue,
                                                   _code(out.dtype), m, n, -(-k // 8) * 8, self._stream()), "gemm_mx4_rows")
            return out
        xp, xs, ldx, alive = self._mx4_rows(x, k, 128)
        form, ks = self._mx4_form(m, n, k, epilogue, xs is not None)
        kp = -(-k // 128) * 128
        if ks == 1:
            self._check(self.lib.llm_gemm_mx4_many(xp, xs, ldx, codes, scales, bptr, out.data_ptr(), epilogue,
                                                   _code(out.dtype), m, n, kp, form, 1, self._stream()), "gemm_mx4_many")
            return out
        parts = torch.empty((ks, m, n), dtype=torch.float32, device=self.device)
        self._check(self.lib.llm_gemm_mx4_many(xp, xs, ldx, codes, scales, None, parts.data_ptr(), self._EPI_NONE,
                                               _code(torch.float32), m, n, kp, form, ks, self._stream()), "gemm_mx4_many")
        self._check(self.lib.llm_mx4_join(parts.data_ptr(), ks, bptr, out.data_ptr(), epilogue, _code(out.dtype), m, n,
                                          self._stream()), "mx4_join")
        return out

    def _linear_mx4(self, x, w, bias, out_dtype, residual=None):
        """``linear`` with an MXFP4 weight.  With ``residual`` the product is returned, for the norm
        that comes next to add."""
        from .ops import NormedRows
        if isinstance(x, NormedRows):
            x = self._materialise(x, torch.bfloat16)
        m, k = x.shape
        n = w.shape[0]
        if k != w.shape[1]:
            raise KernelError("linear: x is [%d, %d] but the weight is [%d, %d]" % (m, k, n, w.shape[1]))
        return self._mx4_product(x, w, torch.empty((m, n), dtype=out_dtype, device=self.device), self._EPI_NONE, bias)

    def _linear_swiglu_mx4(self, x, w, dtype, activation):
        """The gated product with a stacked MXFP4 weight.  Gate and up stay in 32 bits until the
        result is rounded."""
        from .ops import NormedRows
        if isinstance(x, NormedRows):
            x = self._materialise(x, torch.bfloat16)
        if dtype is None:
            dtype = torch.bfloat16
        m, k = x.shape
        act = self._act(activation)
        if w.shape[0] % 2:
            raise KernelError("linear_swiglu: the stacked weight has an odd number of rows")
        if k != w.shape[1]:
            raise KernelError("linear_swiglu: x is [%d, %d] but the weight is %s" % (m, k, w.shape))
        inter = w.shape[0] // 2
        if dtype == torch.bfloat16 and inter % TILE_ROWS == 0:
            out = torch.empty((m, inter), dtype=torch.bfloat16, device=self.device)
            return self._mx4_product(x, w, out, self._EPI_SWIGLU | (act << 4))
        # up's rows begin inside a tile, or the result is wanted in 32 bits: the product in 32 bits, then the gate
        out = self.silu_mul(self._linear_mx4(x, w, None, torch.float32), activation)
        return out if out.dtype == dtype else out.to(dtype)
