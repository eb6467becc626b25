"""Matrices in microscaled 4-bit floating point (MXFP4) and the operations on them.

The format (OCP Microscaling Formats, MXFP4): every 32 neighbouring elements of a row share a scale
2^(e - 127), one byte (255: the block reads as NaN), and an element is a sign and one of the
magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6: 4.25 bits an element.  ``Mx4Matrix`` holds such a matrix as
the matrix cores take it (csrc/mx4.h says how it lies).
"""
import ctypes

import torch

from ..errors import KernelError

_vp, _i, _f, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t

BLOCK = 32                      # elements that share a scale
TILE_ROWS, QUAD = 16, 512       # a tile holds 16 rows by whole quads of 512 elements

SIGNATURES = {
    "llm_mx4_quantize": [_vp, _i, _sz, _i, _i, _vp, _vp, _vp],
    "llm_mx4_dequantize": [_vp, _vp, _vp, _i, _i, _i, _vp],
    "llm_mx4_pack": [_vp, _sz, _vp, _i, _i, _vp, _vp, _vp],
    "llm_pad_rows": [_vp, _sz, _vp, _i, _i, _i, _vp],
    "llm_gemm_mx4_rows": [_vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _f, _vp],
    "llm_gemm_mx4_rows_rope": [_vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp, _vp, _i, _vp, _vp, _vp, _vp, _i,
                               _vp, _vp, _i, _i, _vp, _f, _vp],
    "llm_gemm_mx4_many": [_vp, _vp, _i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _i, _vp],
    "llm_mx4_join": [_vp, _i, _vp, _vp, _i, _i, _i, _i, _vp],
}


def tiled_sizes(rows: int, width: int):
    """(bytes of codes, bytes of scales) of a matrix of these sizes, whole tiles."""
    cells = -(-rows // TILE_ROWS) * -(-width // QUAD)
    return cells * 4096, cells * 256


class Mx4Matrix:
    """A matrix ``[rows, width]`` in MXFP4: ``codes`` and ``scales`` are flat uint8 tensors in the
    order the matrix cores read them, zero where rows and columns are filled up.  What
    ``HipOps.quantize_mx4`` and ``HipOps.mx4_from_codes`` return, and the products take as a weight, or
    on both sides."""
    dtype = "mxfp4"
    __slots__ = ("shape", "device", "codes_ptr", "scales_ptr", "_storage")

    def __init__(self, shape, codes, scales):
        rows, width = shape
        want = tiled_sizes(rows, width)
        for t, size, what in ((codes, want[0], "codes"), (scales, want[1], "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != (size,) or not t.is_contiguous() or t.data_ptr() % 16:
                raise KernelError("the %s of an MXFP4 matrix [%d, %d] are %d bytes in a row, 16-byte aligned"
                                  % (what, rows, width, size))
        if codes.device != scales.device:
            raise KernelError("codes and scales of an MXFP4 matrix lie on %s and %s" % (codes.device, scales.device))
        self.shape, self.device, self._storage = (rows, width), codes.device, (codes, scales)
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _new(cls, rows, width, device, blank):
        """Room for a matrix: one allocation, the codes first."""
        q = cls.__new__(cls)
        cells = -(-rows // TILE_ROWS) * -(-width // QUAD)
        q._storage = both = blank.new_empty(cells * 4352)
        q.shape, q.device, q.codes_ptr = (rows, width), device, both.data_ptr()
        q.scales_ptr = q.codes_ptr + cells * 4096
        return q

    @property
    def codes(self):
        return self._parts()[0]

    @property
    def scales(self):
        return self._parts()[1]

    def _parts(self):
        if not isinstance(self._storage, tuple):
            size = tiled_sizes(*self.shape)[0]
            self._storage = (self._storage[:size], self._storage[size:])
        return self._storage

    def leading_rows(self, rows: int) -> "Mx4Matrix":
        """The first ``rows`` rows, a multiple of 16, in the same storage."""
        if rows % TILE_ROWS or not 0 < rows <= self.shape[0]:
            raise KernelError("the leading rows of an MXFP4 matrix are a multiple of %d (asked for %d of %d)"
                              % (TILE_ROWS, rows, self.shape[0]))
        codes, scales = tiled_sizes(rows, self.shape[1])
        return Mx4Matrix((rows, self.shape[1]), self.codes[:codes], self.scales[:scales])


class Mx4Ops:
    """The operations of ``HipOps`` on matrices in MXFP4."""

    MX4_ROWS = 32           # rows that go to the product for few rows in any case
    MX4_PLANS = 4096        # launch plans kept, by sizes
    MX4_FAR = 1 << 22       # most elements between two rows in bfloat16 for the product for many rows: a block's offsets have 32 bits

    # ---- conversions
    def _mx4_empty(self, rows, width):
        if rows <= 0 or width <= 0:
            raise KernelError("an MXFP4 matrix has rows and columns, not [%d, %d]" % (rows, width))
        if rows > 1 << 27 or width > 65535 * QUAD:          # (threads of a launch, blocks along the second axis of a grid)
            raise KernelError("an MXFP4 matrix of [%d, %d] is too large" % (rows, width))
        return Mx4Matrix._new(rows, width, self.device, self._blank[torch.uint8])

    def _mx4(self, q, what):
        if not isinstance(q, Mx4Matrix):
            raise KernelError("%s is no MXFP4 matrix" % what)
        if q.device is not self.device and q.device != self.device:
            raise KernelError("%s lies on %s, not on %s" % (what, q.device, self.device))
        return q

    def quantize_mx4(self, x) -> Mx4Matrix:
        """The matrix ``x`` (bfloat16 or float32, rows contiguous; they may lie further apart than
        their length) in MXFP4.  The scale of a block is 2^(floor(log2(max |x|)) - 2), at least
        2^-127; an element is divided by it and rounded to the nearest code, ties to the even one,
        6 beyond 6.  A block that holds an infinity or a NaN reads as NaN.  A matrix without rows is refused."""
        self._matrix(x, "the matrix to quantise")
        m, k = x.shape
        q = self._mx4_empty(m, k)
        self._launch("llm_mx4_quantize", x.data_ptr(), self._dtype_code(x.dtype), max(x.stride(0), k), m, k,
                     q.codes_ptr, q.scales_ptr)
        return q

    def dequantize_mx4(self, q: Mx4Matrix, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers that ``q`` stands for, exactly (with a scale of 2^126 or 2^127 those of 2^128 and more
        are infinities)."""
        self._mx4(q, "the matrix to read")
        code = self._dtype_code(dtype)
        m, k = q.shape
        out = self._blank[dtype].new_empty(m, k)
        self._launch("llm_mx4_dequantize", q.codes_ptr, q.scales_ptr, out.data_ptr(), code, m, k)
        return out

    def mx4_from_codes(self, codes, scales, width=None) -> Mx4Matrix:
        """A matrix that is in MXFP4 already, as files hold it: ``codes`` uint8
        ``[rows, ceil(width / 2)]`` or wider, two elements a byte, the even one in the low half, and
        ``scales`` uint8 ``[rows, ceil(width / 32)]``.  ``width``: twice the columns of ``codes``
        unless it is given (an odd width, padded rows).  Every byte is taken; of scales of 253 and 254
        ``linear`` says what becomes."""
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise KernelError("mx4_from_codes: codes and scales are matrices of uint8")
        self._matrix(codes, "the matrix of codes")
        rows, columns = codes.shape
        width = 2 * columns if width is None else int(width)
        if not 0 < -(-width // 2) <= columns:
            raise KernelError("mx4_from_codes: %d columns of codes do not hold rows of %d elements" % (columns, width))
        self._dev(scales, "the matrix of scales", torch.uint8, (rows, -(-width // BLOCK)))
        q = self._mx4_empty(rows, width)
        self._launch("llm_mx4_pack", codes.data_ptr(), max(codes.stride(0), columns), scales.data_ptr(), rows, width,
                     q.codes_ptr, q.scales_ptr)
        return q

    def _matrix(self, x, what):
        """A matrix on the device with contiguous rows."""
        if x.is_contiguous() and x.get_device() == self._index and x.dim() == 2:
            return
        if x.device != self.device:
            raise KernelError("%s lies on %s, not on %s" % (what, x.device, self.device))
        if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
            raise KernelError("%s must be a matrix with contiguous rows" % what)

    # ---- products
    def _mx4_few(self, m, n, k, four):
        """Whether the product goes to the kernel for few rows (times of plain products over warm weights; over
        cold ones, with the stream or the cache to write, 64 rows of K 4,096 take 14.5 us for 4,096 outputs and 16.3
        for 6,144).  Up to 32 rows always (us, 32 rows, that
        kernel against the other: K 14,336, 4,096 outputs 19.5 against 23.0, gate and up of 4,096 x 14,336
        22.7 against 22.8).  Up to 64, where it reads W twice, if W is small and has two tiles a compute
        unit at most (MXFP4: one and a half), so that the other cannot fill the units (64 rows, bfloat16:
        K 2,048, 6,144 outputs 8.9 against 10.4, K 8,192, 2,048 outputs 12.3 against 13.4, but K 2,048, 10,240
        outputs 12.9 against 10.8, K 14,336, 2,048 outputs 18.2 against 16.6; MXFP4, in the same order, 6.1
        against 6.5, 7.0 against 10.6, 8.4 against 6.8, 9.8 against 12.6: wide rows count for less there).
        Beyond 64 while its blocks, a tile of W by 32 rows each, are two a compute unit (MXFP4: two and a
        half) and read little of X in all (K 2,048, 2,048 outputs, 128 / 192 rows: bfloat16 9.3 / 12.7 against
        9.5 / 9.6, MXFP4 4.3 / 5.8 against 5.7 / 5.8; K 2,048, 512 outputs, 512 rows: 8.3 against 10.3 and
        4.1 against 6.1)."""
        if m <= self.MX4_ROWS:
            return True
        tiles = -(-n // TILE_ROWS)
        if m <= 2 * self.MX4_ROWS:
            return 2 * tiles <= (3 if four else 4) * self.units and n * k <= 1 << 25 and k <= 1 << (14 if four else 13)
        blocks = tiles * -(-m // 32)
        return 2 * blocks <= (5 if four else 4) * self.units and blocks * k <= (2 if four else 1) << 20

    # The product for many rows, by form (csrc/gemm_mx4_many.hip): rows of X and of W a block, the us that
    # 128 elements of K take with one, two, three, four blocks a compute unit (beyond, as much again for
    # every four), and as how many such elements more a block's begin and end count.  Fitted to 135
    # products of each kind (warm weights, plain epilogue), 128 to 14,336 elements of K, 64 to 4,096 rows, 2,048 to 28,672 outputs, in every
    # form: what this says is best takes 0.1 % longer than the best on average, 4 % at most.
    _MX4_FORMS = {
        False: ((0, 256, 256, (2.56, 5.12, 7.68, 10.24), 1.5), (1, 128, 256, (1.255, 2.51, 3.765, 5.02), 4.5),
                (2, 64, 128, (0.69, 0.92, 1.07, 1.75), 0), (3, 64, 128, (0.58, 1.15, 1.73, 2.31), 0.5),
                (4, 64, 64, (0.58, 1.17, 1.75, 2.34), 0)),
        True: ((0, 256, 256, (0.83, 1.66, 2.48, 3.31), 0), (1, 128, 128, (0.265, 0.36, 1.26, 1.34), 0),
               (2, 64, 128, (0.25, 0.26, 0.51, 1.13), 0), (3, 64, 128, (0.21, 0.42, 0.63, 0.84), 1),
               (4, 64, 64, (0.17, 0.34, 0.51, 0.68), 0)),
    }

    def _mx4_form(self, m, n, k, four):
        """(form, slices of K) of the product for many rows: those for which blocks, times and the
        adding of the slices (each written and read in 32 bits, and a launch) come out lowest."""
        quads, all_units = -(-k // QUAD), -(-k // 128)
        best = None
        for form, rows, cols, times, more in self._MX4_FORMS[four]:
            blocks = -(-m // rows) * -(-n // cols)
            for ks in range(1, min(quads, 16) + 1):
                if ks > 1 and blocks * ks > 2 * self.units:
                    break
                per = -(-quads // ks)
                if -(-quads // per) != ks:
                    continue
                a_unit = -(-blocks * ks // self.units)
                cost = (min(4 * per, all_units) + more) * (times[3] * ((a_unit - 1) // 4) + times[(a_unit - 1) % 4])
                if ks > 1:
                    cost += 5.0 + ks * m * n * 8 / 3e6
                if best is None or cost < best[0]:
                    best = (cost, form, ks)
        return best[1:]

    def _mx4_plan(self, m, n, n_out, k, four):
        """(form, slices of K), form -1 being the kernel for few rows.  Kept by sizes: choosing takes
        longer than a small product."""
        key = (m, n, n_out, k, four)
        plan = self._mx4_plans.get(key)
        if plan is None:
            if len(self._mx4_plans) >= self.MX4_PLANS:
                self._mx4_plans.clear()
            few = self._mx4_few(m, n, k, four) or (k > self.MX4_FAR and not four)
            plan = (-1, 1) if few else self._mx4_form(m, n, k, four)
            self._mx4_plans[key] = plan
        return plan

    def _mx4_rows(self, x, k, piece):
        """bfloat16 rows for a kernel that reads ``piece`` elements of them at a time: ``x`` itself, or a
        padded copy where its length, distance or address does not allow that; with its address and
        the distance of its rows."""
        at = x.data_ptr()
        if x.dtype != torch.bfloat16:
            raise KernelError("linear: an MXFP4 weight takes rows in bfloat16 or MXFP4, not %s" % (x.dtype,))
        self._matrix(x, "linear input")
        ld = max(x.stride(0), k)
        if k % piece == 0 and ld % piece == 0 and at % 16 == 0 and ld <= (self.MX4_FAR if piece > 8 else 1 << 30):
            return x, at, ld
        ldp = -(-k // piece) * piece
        padded = torch.empty((x.shape[0], ldp), dtype=torch.bfloat16, device=self.device)
        self._launch("llm_pad_rows", at, ld, padded.data_ptr(), x.shape[0], k, ldp)
        return padded, padded.data_ptr(), ldp

    def _mx4_product(self, x, w, n_out, out_dtype, epilogue, bias=None, stack=False):
        """The product of ``x`` (a matrix, MXFP4 rows, or a record of normed rows whose norm is
        prepared) with ``w``.  ``stack``: where K goes in slices their products may come back
        unadded, ``[slices, m, n]`` in 32 bits."""
        if w.device is not self.device:
            self._mx4(w, "the weight")
        n, k = w.shape
        four, ssq, eps = False, None, 0.0
        if not isinstance(x, torch.Tensor):
            if isinstance(x, Mx4Matrix):
                self._mx4(x, "linear input")
                four = True
            else:
                x, ssq, eps = x.pre.raw, x.pre.ssq.data_ptr(), x.pre.eps
        m, k2 = x.shape
        if k != k2:
            raise KernelError("linear: x is [%d, %d] but the weight is [%d, %d]" % (m, k2, n, k))
        code = self._dtype_code(out_dtype)
        bptr = None if bias is None else self._dev(bias, "bias", torch.float32, (n,))
        if m == 0:
            return self._blank[out_dtype].new_empty(m, n_out)
        form, ks = self._mx4_plans.get((m, n, n_out, k, four)) or self._mx4_plan(m, n, n_out, k, four)
        piece = 8 if form < 0 else 128
        if four:
            xp, xs, ldx = x.codes_ptr, x.scales_ptr, 0
        else:
            xp, xs, ldx = x.data_ptr(), None, k
            if not (x.dtype is torch.bfloat16 and k % piece == 0 and xp % 16 == 0 and x.is_contiguous()
                    and x.get_device() == self._index):
                x, xp, ldx = self._mx4_rows(x, k, piece)
        kp = -(-k // piece) * piece         # (where rows were padded, their length: the weight's codes there are zero)
        wp, ws = w.codes_ptr, w.scales_ptr
        if ks == 1:
            out = self._blank[out_dtype].new_empty(m, n_out)
            if form < 0:
                self._launch("llm_gemm_mx4_rows", xp, xs, ldx, wp, ws, bptr, out.data_ptr(), epilogue, code, m, n, kp,
                             None, None, None, ssq, eps)
            else:
                self._launch("llm_gemm_mx4_many", xp, xs, ldx, wp, ws, bptr, out.data_ptr(), epilogue, code, m, n, kp,
                             form, 1)
            return out
        parts = self._blank[torch.float32].new_empty(ks, m, n)
        self._launch("llm_gemm_mx4_many", xp, xs, ldx, wp, ws, None, parts.data_ptr(), self._EPI_NONE,
                     self._dtype_code(torch.float32), m, n, kp, form, ks)
        if stack and bias is None and epilogue == self._EPI_NONE:
            return parts
        out = self._blank[out_dtype].new_empty(m, n_out)
        self._launch("llm_mx4_join", parts.data_ptr(), ks, bptr, out.data_ptr(), epilogue, code, m, n)
        return out

    def _mx4_input(self, x, w):
        """``x`` for a product with ``w``: a matrix as it is; a record of normed rows goes in as it is where the product before
        has prepared its norm and the product for few rows takes it, else the norm kernel runs."""
        if isinstance(x, (torch.Tensor, Mx4Matrix)):
            return x
        if x.pre is not None and x.pre.raw.shape[0] <= self.ACCUM_ROWS and w.shape[1] == x.pre.raw.shape[1]:
            return x
        return self._materialise(x, torch.bfloat16)

    def _linear_mx4(self, x, w, bias, out_dtype, residual=None, then_norm=None):
        """``linear`` with an MXFP4 weight.  With ``residual`` the product for few rows adds into it;
        the other returns the product, or its slices of K, for the norm that comes next to add."""
        if not isinstance(x, torch.Tensor):
            x = self._mx4_input(x, w)
        n, k = w.shape
        if residual is None or bias is not None or not isinstance(x, torch.Tensor):
            return self._mx4_product(x, w, n, out_dtype, self._EPI_NONE, bias, residual is not None)
        m = x.shape[0]
        if m == 0 or x.shape[1] != k or self._mx4_plan(m, n, n, k, False)[0] >= 0:
            return self._mx4_product(x, w, n, out_dtype, self._EPI_NONE, None, True)
        self._mx4(w, "the weight")
        self._dev(residual, "residual stream", torch.float32, (m, n))
        x, xp, ldx = self._mx4_rows(x, k, 8)
        record, nw, raw, ssq = None, None, None, None
        if then_norm is not None and self.fold_norms and m <= self.ACCUM_ROWS and n % 16 == 0:
            weight, eps = then_norm
            nw = self._dev(weight, "norm weight", torch.float32, (n,))
            record = self._prenormed(m, n, weight, eps)
            raw, ssq = record.raw.data_ptr(), record.ssq.data_ptr()
        self._launch("llm_gemm_mx4_rows", xp, None, ldx, w.codes_ptr, w.scales_ptr, None, residual.data_ptr(),
                     self._EPI_ACCUM, self._dtype_code(torch.float32), m, n, -(-k // 8) * 8, nw, raw, ssq, None, 0.0)
        return record

    def _linear_swiglu_mx4(self, x, w, dtype, activation):
        """The gated product with a stacked MXFP4 weight.  Gate and up stay in 32 bits until the
        result is rounded."""
        x = self._mx4_input(x, w)
        act = self._act(activation)
        dtype = dtype or torch.bfloat16
        n = w.shape[0]
        if n % 2:
            raise KernelError("linear_swiglu: the stacked weight has an odd number of rows")
        if dtype == torch.bfloat16 and n // 2 % TILE_ROWS == 0:
            return self._mx4_product(x, w, n // 2, dtype, self._EPI_SWIGLU | (act << 4))
        # up's rows begin inside a tile, or the result is wanted in 32 bits: the product in 32 bits, then the gate
        code = self._dtype_code(dtype)
        y = self._mx4_product(x, w, n, torch.float32, self._EPI_NONE, None, True)
        out = torch.empty((y.shape[-2], n // 2), dtype=dtype, device=self.device)
        if y.shape[-2]:
            self._launch("llm_mx4_join", y.data_ptr(), y.shape[0] if y.dim() == 3 else 1, None, out.data_ptr(),
                         self._EPI_SWIGLU | (act << 4), code, y.shape[-2], n)
        return out

    def _qkv_rope_mx4(self, x, w, bias, n_heads, n_kv, hd, cos, sin, rot_dim, ctx, kv, write):
        """The stacked projection with its rotation and cache write in one kernel, or None where the
        product for few rows does not take it."""
        x = self._mx4_input(x, w)
        if isinstance(x, Mx4Matrix):
            return None, x
        pre = None if isinstance(x, torch.Tensor) else x.pre
        rows = x if pre is None else pre.raw
        m, k = rows.shape
        n = w.shape[0]
        if m == 0 or k != w.shape[1] or self._mx4_plan(m, n, n, k, False)[0] >= 0:
            return None, x
        self._mx4(w, "qkv weight")
        rows, xp, ldx = self._mx4_rows(rows, k, 8)
        cptr, sptr, bptr, kptr, vptr, tptr, stride = self._rope_operands("qkv_rope", cos, sin, rot_dim, bias, n, ctx, kv, write,
                                                                         n_kv, hd, torch.bfloat16)
        q = torch.empty((m, n_heads * hd), dtype=torch.bfloat16, device=self.device)
        self._launch("llm_gemm_mx4_rows_rope", xp, ldx, w.codes_ptr, w.scales_ptr, bptr, q.data_ptr(), m,
                     -(-k // 8) * 8, n_heads, n_kv, hd, cptr, sptr, rot_dim, ctx.tok_pos.data_ptr(), ctx.tok_seq.data_ptr(),
                     ctx.seq_slot.data_ptr(), tptr, stride, kptr, vptr, 64, 1 if write else 0,
                     pre.ssq.data_ptr() if pre is not None else None, pre.eps if pre is not None else 0.0)
        return q, x
