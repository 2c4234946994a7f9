"""Matrices in 4 bits (microscaled e2m1): quantisation, and products of a block-sparse matrix with dense ones.

Formats, layouts and roundings are those of the C ABI (include/smat_b200.h, "matrices in 4 bits"):
  "nvfp4"  groups of 16 columns share an e4m3 scale, every row has an fp32 scale (a power of two where it is computed here)
  "mxfp4"  groups of 32 columns share a scale 2^e

    A4 = Fp4SparseMatrix.quantize(A)              # A: SparseMatrix
    plan = Fp4Plan(A4)
    plan.spmm(x, C)                               # decoding: x [N, K] in fp16 or bf16, C [M, N] of the same type
    plan.spmm(Fp4Matrix.quantize(x), C)           # prefilling: both in 4 bits on the tensor cores

The reference multiplies fp16 only (src/cuda_hgemm/src/mma/mmaCBT.cu:13-88)."""
import ctypes as C

import torch

from . import api
from .api import Matrix, SmatError, SparseMatrix, _check, lib

_FORMATS = {"nvfp4": 0, "mxfp4": 1}
_GROUP = {"nvfp4": 16, "mxfp4": 32}
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_LIB = None


def _lib():
    global _LIB
    if _LIB is None:
        L = lib()
        vp, sz, i = C.c_void_p, C.c_size_t, C.c_int
        L.smat_fp4_quantize.argtypes = [vp, i, sz, sz, sz, i, vp, vp, vp, vp]
        L.smat_fp4_dequantize.argtypes = [vp, vp, vp, i, sz, sz, vp, i, sz, vp]
        L.smat_fp4_quantize_blocks.argtypes = [vp, i, vp, vp, sz, sz, i, vp, vp, vp, vp]
        L.smat_fp4_dequantize_blocks.argtypes = [vp, vp, vp, i, vp, sz, sz, vp, i, vp]
        L.smat_fp4_plan_create.argtypes = [C.POINTER(vp), vp, vp, vp, i, vp, vp, sz, sz, sz, sz, sz, i, vp]
        L.smat_fp4_plan_set_values.argtypes = [vp, vp]
        L.smat_fp4_plan_spmm.argtypes = [vp, vp, i, vp, sz, vp]
        L.smat_fp4_plan_spmm_fp4.argtypes = [vp, vp, vp, vp, i, vp, i, sz, vp]
        L.smat_fp4_plan_destroy.argtypes = [vp]
        _LIB = L
    return _LIB


def _refuse(text):
    raise SmatError(-1, text)


def _format(fmt):
    if fmt not in _FORMATS:
        _refuse(f"unknown 4-bit format {fmt!r}: 'nvfp4' or 'mxfp4'")
    return _FORMATS[fmt]


def _dtype(dtype, most=2):
    code = _DTYPES.get(dtype, 3)
    if code > most:
        _refuse(f"element type {dtype} is not one of {[str(d) for d, c in _DTYPES.items() if c <= most]}")
    return code


_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # a tensor on a GPU has initialised CUDA


def _on_current_device(t):
    if not t.is_cuda or t.get_device() != _device():
        _refuse(f"tensor on {t.device}: it has to be on the current CUDA device")


def _bytes_like(t, shape, name, device):
    """t as uint8 (fp8 and other 8-bit types by their bits), of the given shape, contiguous."""
    t = t if t.dtype == torch.uint8 else t.view(torch.uint8) if t.element_size() == 1 else _refuse(f"{name}: 8-bit elements expected, not {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        _refuse(f"{name}: shape {tuple(shape)} expected, not {tuple(t.shape)}")
    return t.to(device).contiguous()


def _row_scales(row_scale, fmt, rows, device):
    """float32[rows] or None; a single number stands for all rows."""
    if row_scale is None:
        return None
    if fmt != "nvfp4":
        _refuse("row scales go with nvfp4")
    t = torch.as_tensor(row_scale, dtype=torch.float32, device=device)
    if t.numel() == 1:
        return t.reshape(1).expand(rows).contiguous()
    if tuple(t.shape) != (rows,):
        _refuse(f"row_scale: one number or {rows} expected, not shape {tuple(t.shape)}")
    return t.contiguous()


def _valid_scales(scales, fmt):
    """e4m3 scales without their sign bit (no scale is negative)."""
    return scales & 0x7F if fmt == "nvfp4" else scales


def _ptr(t):
    return None if t is None else t.data_ptr()


class Fp4Matrix:
    """Dense matrix [N, K] in 4 bits, K a multiple of 16: the activations of a product.

    ``codes`` uint8 [N, 32 * ceil(K / 64)], ``scales`` uint8 (tiled, see the C header; ``group_scales()`` gives them as
    [N, groups]), ``row_scale`` float32 [N] or None."""

    def __init__(self, N, K, fmt="nvfp4", device="cuda"):
        if fmt not in _FORMATS:
            _format(fmt)
        if N < 0 or K < 0 or K % 16:
            _refuse(f"N ({N}) must not be negative, and K ({K}) a multiple of 16")
        self.N, self.K, self.fmt = N, K, fmt
        self.quads = quads = (K + 63) // 64
        # One piece of memory; the tensors in it are made when they are asked for (a microsecond each).
        self._scales_at = at = (N * quads * 32 + 15) // 16 * 16
        self._row_at = end = at + (N + 127) // 128 * quads * 512
        self._memory = torch.empty(end + (4 * N if fmt == "nvfp4" else 0), dtype=torch.uint8, device=device)
        self._codes = self._scales = self._row = None
        self._has_row = fmt == "nvfp4"

    @property
    def _at(self):
        """Addresses of codes, scales and row scales (None: there are none)."""
        p = self._memory.data_ptr()
        return p, p + self._scales_at, p + self._row_at if self._has_row else None

    def __getstate__(self):  # of a copy: the tensors in its memory are made again, as parts of its own
        return {**self.__dict__, "_codes": None, "_scales": None, "_row": None}

    @property
    def device(self):
        return self._memory.device

    @property
    def codes(self):
        if self._codes is None:
            self._codes = self._memory[:self.N * self.quads * 32].view(self.N, self.quads * 32)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._memory[self._scales_at:self._row_at]
        return self._scales

    @property
    def row_scale(self):
        if self._row is None and self._has_row:
            self._row = self._memory[self._row_at:].view(torch.float32)
        return self._row

    @row_scale.setter
    def row_scale(self, value):
        t = _row_scales(value, self.fmt, self.N, self.device)
        self._row, self._has_row = None, t is not None
        if self._has_row:  # a copy: quantize(out=...) writes to it later
            self._memory[self._row_at:].view(torch.float32).copy_(t)

    @classmethod
    def quantize(cls, X, fmt="nvfp4", out=None):
        """X: Matrix or tensor [N, K] in fp16, bf16 or fp32 (rows may be strided, 16-byte aligned).  ``out``: an Fp4Matrix of this
        size and format to write to instead of a new one."""
        x = X.data if isinstance(X, Matrix) else X
        f = _format(fmt)
        d = _dtype(x.dtype)
        if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
            _refuse("a matrix [N, K] with consecutive columns is expected")
        _on_current_device(x)
        N, K = x.shape
        if out is None:
            out = cls(N, K, fmt, x.device)
        elif (out.N, out.K, out.fmt, out.device) != (N, K, fmt, x.device):
            _refuse("out has another size, format or device")
        elif f == 0 and not out._has_row:
            _refuse("out has no row scales")
        codes, scales, row = out._at
        rc = (_LIB or _lib()).smat_fp4_quantize(x.data_ptr(), d, N, K, x.stride(0) if N > 1 else K, f, codes, scales, row, api._stream())
        if rc:
            _check(rc)
        return out

    @classmethod
    def from_codes(cls, codes, scales, K, fmt="nvfp4", row_scale=None, device="cuda"):
        """From arrays as checkpoints and other programs have them: codes uint8 [N, K / 2] (the even column in the low half),
        scales 8-bit [N, ceil(K / 16 or 32)] (e4m3, or e8m0 bytes), row_scale one number or [N]."""
        codes, scales = torch.as_tensor(codes), torch.as_tensor(scales)
        if codes.dim() != 2:
            _refuse(f"codes: a matrix [N, {K // 2}] is expected, not shape {tuple(codes.shape)}")
        N = codes.shape[0]
        self = cls(N, K, fmt, device)
        dev = self.device
        self.codes.zero_()
        self.codes[:, :K // 2] = _bytes_like(codes, (N, K // 2), "codes", dev)
        groups, per = -(-K // _GROUP[fmt]), 64 // _GROUP[fmt]
        s = _valid_scales(_bytes_like(scales, (N, groups), "scales", dev), fmt)
        full = torch.zeros((-(-N // 128) * 128, self.quads, 4), dtype=torch.uint8, device=dev)
        flat = torch.zeros((N, self.quads * per), dtype=torch.uint8, device=dev)
        flat[:, :groups] = s
        full[:N, :, :per] = flat.view(N, self.quads, per)
        self.scales.copy_(full.view(-1, 4, 32, self.quads, 4).permute(0, 3, 2, 1, 4).reshape(-1))
        self.row_scale = row_scale
        return self

    def group_scales(self):
        """The scales as uint8 [N, ceil(K / 16 or 32)]."""
        per = 64 // _GROUP[self.fmt]
        s = self.scales.view(-1, self.quads, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, self.quads, 4)[:self.N, :, :per]
        return s.reshape(self.N, -1)[:, :-(-self.K // _GROUP[self.fmt])].contiguous()

    def dequantize(self, dtype=torch.float16, out=None):
        """The values as a tensor [N, K] in fp16, bf16 or fp32; ``out``: a tensor to write to.  Code * scale is exact; times the row
        scale it is rounded to fp32 (powers of two change nothing), then to the type."""
        d = _dtype(dtype if out is None else out.dtype)
        _on_current_device(self._memory)
        if out is None:
            out, ld = torch.empty((self.N, self.K), dtype=dtype, device=self.device), self.K
        else:
            if tuple(out.shape) != (self.N, self.K) or (self.K > 1 and out.stride(1) != 1) or out.device != self.device:
                _refuse("out has another size, strided columns or another device")
            ld = out.stride(0) if self.N > 1 else self.K
        codes, scales, row = self._at
        rc = _lib().smat_fp4_dequantize(codes, scales, row, _FORMATS[self.fmt], self.N, self.K, out.data_ptr(), d, ld, api._stream())
        if rc:
            _check(rc)
        return out


class Fp4SparseMatrix:
    """Block-sparse matrix with its 16x16 blocks in 4 bits: the structure of a SparseMatrix (``bcsrRowPtr``, ``bcsrColIdx``),
    ``codes`` uint8 [nnzb, 16, 8], ``scales`` uint8 [nnzb, 16], ``row_scale`` float32 [M] or None."""

    def __init__(self):
        self.M = self.K = self.nnzb = 0
        self.fmt = "nvfp4"
        self.bcsrRowPtr = self.bcsrColIdx = self.codes = self.scales = self.row_scale = None
        self._checked = ()

    def _arrays(self):
        return self.codes, self.scales, self.row_scale, self.bcsrRowPtr, self.bcsrColIdx

    def _check_arrays(self):
        """Refuses arrays that are not what the kernels take them for.  Those that were looked over before are not again (0.4 instead of
        4 us)."""
        c = self._checked
        if c and self.codes is c[0] and self.scales is c[1] and self.row_scale is c[2] and self.bcsrRowPtr is c[3] and self.bcsrColIdx is c[4]:
            return
        device = self.codes.device if isinstance(self.codes, torch.Tensor) else None
        for name, t, dtype, least, most in (("codes", self.codes, torch.uint8, self.nnzb * 128, self.nnzb * 128),
                                            ("scales", self.scales, torch.uint8, self.nnzb * 16, self.nnzb * 16),
                                            ("row_scale", self.row_scale, torch.float32, self.M, self.M),
                                            ("bcsrRowPtr", self.bcsrRowPtr, torch.int32, self.M // 16 + 1, self.M // 16 + 1),
                                            ("bcsrColIdx", self.bcsrColIdx, torch.int32, self.nnzb, None)):
            if name == "row_scale" and t is None:
                continue
            if name == "row_scale" and self.fmt != "nvfp4":
                _refuse("row_scale: row scales go with nvfp4")
            if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.numel() < least or (most is not None and t.numel() > most):
                _refuse(f"{name}: {'at least ' if most is None else ''}{least} elements of {dtype} are expected")
            if not t.is_contiguous() or t.device != device:
                _refuse(f"{name}: it has to be contiguous and on {device}, like codes")
        self._checked = self._arrays()

    @classmethod
    def quantize(cls, A, fmt="nvfp4", check=False):
        """The blocks of a SparseMatrix in 4 bits; the structure is shared with it."""
        f = _format(fmt)
        v, rp, ci = A.bcsrVal, A.bcsrRowPtr, A.bcsrColIdx
        _on_current_device(v)
        if (v.numel() < A.nnzb * 256 or rp.numel() != A.M // 16 + 1 or ci.numel() < A.nnzb or rp.dtype != torch.int32 or ci.dtype != torch.int32
                or not (v.is_contiguous() and rp.is_contiguous() and ci.is_contiguous()) or not v.get_device() == rp.get_device() == ci.get_device()):
            _refuse(f"a SparseMatrix of {A.nnzb} blocks with int32 bcsrRowPtr of {A.M // 16 + 1} and bcsrColIdx, contiguous, on one device is expected")
        self = cls()
        n, dev = A.nnzb, v.device
        self.M, self.K, self.nnzb, self.fmt, self.bcsrRowPtr, self.bcsrColIdx = A.M, A.K, n, fmt, rp, ci
        self.codes = codes = torch.empty((n, 16, 8), dtype=torch.uint8, device=dev)
        self.scales = scales = torch.empty((n, 16), dtype=torch.uint8, device=dev)
        self.row_scale = row = torch.empty(A.M, dtype=torch.float32, device=dev) if f == 0 else None
        self._checked = (codes, scales, row, rp, ci)
        rc = (_LIB or _lib()).smat_fp4_quantize_blocks(v.data_ptr(), _dtype(v.dtype), rp.data_ptr(), ci.data_ptr(), A.M, n, f, codes.data_ptr(),
                                                       scales.data_ptr(), _ptr(row), api._stream())
        if rc:
            _check(rc)
        if check:
            _check(lib().smat_device_status(api._stream()))
        return self

    @classmethod
    def from_codes(cls, M, K, bcsr_rowptr, bcsr_colidx, codes, scales, fmt="nvfp4", row_scale=None, device="cuda"):
        """From arrays in 4 bits: codes uint8 [nnzb, 16, 8], scales 8-bit [nnzb, 16] (of mxfp4: equal for the two blocks of an
        aligned pair; products treat block-rows where they are not as empty and report it), row_scale one number or [M]; rowptr and element columns as in SparseMatrix."""
        _format(fmt)
        self = cls()
        self.M, self.K, self.nnzb, self.fmt = int(M), int(K), int(len(bcsr_colidx)), fmt
        rp = torch.as_tensor(bcsr_rowptr)
        dev = torch.empty(0, device=device).device
        if rp.numel() != self.M // 16 + 1:
            _refuse(f"bcsr_rowptr: {self.M // 16 + 1} numbers expected, not {rp.numel()}")
        self.bcsrRowPtr = rp.to(dev, torch.int32).contiguous()
        self.bcsrColIdx = torch.as_tensor(bcsr_colidx).to(dev, torch.int32).contiguous()
        self.codes = _bytes_like(torch.as_tensor(codes), (self.nnzb, 16, 8), "codes", dev)
        self.scales = _valid_scales(_bytes_like(torch.as_tensor(scales), (self.nnzb, 16), "scales", dev), fmt)
        self.row_scale = _row_scales(row_scale, fmt, self.M, dev)
        return self

    def dequantize(self, check=False):
        """A SparseMatrix of the values in fp16, rounded as by Fp4Matrix.dequantize; it shares the structure."""
        self._check_arrays()
        _on_current_device(self.codes)
        A = SparseMatrix()
        A.M, A.K, A.nnzb = self.M, self.K, self.nnzb
        A.bcsrRowPtr, A.bcsrColIdx = self.bcsrRowPtr, self.bcsrColIdx
        A.bcsrVal = torch.empty(max(self.nnzb, 1) * 256, dtype=torch.float16, device=self.codes.device)
        rc = _lib().smat_fp4_dequantize_blocks(self.codes.data_ptr(), self.scales.data_ptr(), _ptr(self.row_scale), _FORMATS[self.fmt],
                                               A.bcsrRowPtr.data_ptr(), A.M, A.nnzb, A.bcsrVal.data_ptr(), 0, api._stream())
        if rc:
            _check(rc)
        if check:
            _check(lib().smat_device_status(api._stream()))
        return A


class Fp4Plan:
    """Plan for products of block-rows [brow_begin, brow_end) of an Fp4SparseMatrix (smat_fp4_plan_*).  ``tiles=False``: only for
    products with 16-bit B (decoding), 148 bytes a block beside the matrix's own 144; those with B in 4 bits work but are slow.  With
    tiles a layer that stores a fifth of its blocks takes 720 bytes a block more.  Products do not change the plan and may run on several
    streams at a time."""

    def __init__(self, A, brow_begin=0, brow_end=None, tiles=True):
        self.A = A
        self.brow_begin = brow_begin
        self.brow_end = A.M // 16 if brow_end is None else brow_end
        self._h = None
        A._check_arrays()
        _on_current_device(A.bcsrRowPtr)
        h = C.c_void_p()
        L = _lib()
        _check(L.smat_fp4_plan_create(C.byref(h), A.codes.data_ptr(), A.scales.data_ptr(), _ptr(A.row_scale), _FORMATS[A.fmt],
                                      A.bcsrRowPtr.data_ptr(), A.bcsrColIdx.data_ptr(), A.M, A.K, A.nnzb, self.brow_begin,
                                      self.brow_end, int(tiles), api._stream()))
        self._h = h
        self._arrays = A._arrays()  # the plan has their addresses
        self._rows = (self.brow_end - self.brow_begin) * 16
        self._device = A.bcsrRowPtr.device

    def set_values(self):
        """After A's codes or scales changed in place (same structure)."""
        if self._h is None:
            _refuse("the plan is closed")
        if any(a is not b for a, b in zip(self._arrays, self.A._arrays())):
            _refuse("A has other arrays than when the plan was made: change them in place, or make a new plan")
        _check(_LIB.smat_fp4_plan_set_values(self._h, api._stream()))

    def spmm(self, B, Cout, check=False):
        """C = A x B.  B: Matrix / tensor [N, K] in fp16 or bf16 with C of the same type, or an Fp4Matrix of A's format with C in
        either; C: Matrix / tensor [rows, N], contiguous, fully overwritten.  16-bit B is meant for few tokens: from about 32 on
        ``Plan(A4.dequantize())`` is faster (fp16), for a prompt of thousands four times as fast, if the blocks may take 16 bits."""
        if self._h is None:
            _refuse("the plan is closed")
        Ct = Cout.data if isinstance(Cout, Matrix) else Cout
        four = isinstance(B, Fp4Matrix)
        if four:
            N, K, device = B.N, B.K, B.device
        else:
            Bt = B.data if isinstance(B, Matrix) else B
            if Bt.dim() != 2:
                _refuse(f"B [N, {self.A.K}] is expected, not shape {tuple(Bt.shape)}")
            N, K = Bt.shape
            device = Bt.device
            if Bt.dtype != Ct.dtype:
                _refuse(f"B is {Bt.dtype}, C is {Ct.dtype}: the same type is expected")
            if not Bt.is_contiguous():
                _refuse("B has to be contiguous")
        if K != self.A.K or tuple(Ct.shape) != (self._rows, N):
            _refuse(f"B [N, {self.A.K}] and C [{self._rows}, N] are expected, not [{N}, {K}] and {list(Ct.shape)}")
        if not Ct.is_contiguous():
            _refuse("C has to be contiguous")
        if device != self._device or Ct.device != self._device:
            _refuse(f"B and C have to be on {self._device}, like A")
        d = _dtype(Ct.dtype, most=1)
        if four:
            if B.fmt != self.A.fmt:
                _refuse(f"B is in {B.fmt}, A in {self.A.fmt}")
            codes, scales, row = B._at
            rc = _LIB.smat_fp4_plan_spmm_fp4(self._h, codes, scales, row, _FORMATS[B.fmt], Ct.data_ptr(), d, N, api._stream())
        else:
            rc = _LIB.smat_fp4_plan_spmm(self._h, Bt.data_ptr(), d, Ct.data_ptr(), N, api._stream())
        if rc:
            _check(rc)
        if check:
            _check(lib().smat_device_status(api._stream()))

    def __reduce__(self):  # by copy, deepcopy and pickle: a copy would free the handle a second time
        raise TypeError("a plan cannot be copied: make another one of the same Fp4SparseMatrix")

    def close(self):
        if self._h is not None:
            _lib().smat_fp4_plan_destroy(self._h)
            self._h = None
            self._arrays = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
