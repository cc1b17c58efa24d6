"""Linear layers with 4-bit weights over libdismoen_hip.so: the projections around the
port block's mixers, and the model's head.

Arrays are torch tensors on the block's device or numpy arrays, as in mixer.py.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from ._lib import DMH_F_DEVICE, DmhLinearRows, DmhLinearWeights, check
from .mixer import F32, _bad, _Operator, _packed, _strides, _type


class QuantLinear(_Operator):
    """y = W x + bias.  scales (fp16, [out_features * in_features / group_size]) and packed
    (uint8, [out_features * in_features / 2]) are a quant model's tensor as its file holds
    it; each weight is the bf16 value that dequant_kernel_simd gives.  The weights are
    copied; the arrays may be freed."""

    def __init__(self, blk, out_features: int, in_features: int, scales, packed,
                 group_size: int = 128, bias=None):
        super().__init__(blk)
        self._l = None
        host = isinstance(packed, np.ndarray)
        n, k = int(out_features), int(in_features)
        if min(n, k) < 1 or max(n, k) >= 1 << 31 or group_size not in (32, 64, 128, 256):
            raise _bad(f"out_features {n}, in_features {k}, group_size {group_size}")
        ptrs = []
        for a, size, kinds, what in (
                (scales, n * k // group_size, ("float16", "uint16"), "scales"),
                (packed, n * k // 2, ("uint8",), "packed"), (bias, n, ("float32",), "bias")):
            if a is None and what == "bias":
                ptrs.append(None)
                continue
            if isinstance(a, np.ndarray) is not host or str(a.dtype).split(".")[-1] not in kinds \
                    or int(np.prod(a.shape)) != size or not _packed(a.shape, _strides(a)):
                raise _bad(f"{what} must be {size} contiguous {kinds[0]} values on the side of"
                           " packed")
            if not host and (not a.is_cuda or a.get_device() != blk.device):
                raise _bad(f"{what} must be on the block's device, cuda:{blk.device}")
            ptrs.append(a.ctypes.data if host else a.data_ptr())
        self.out_features, self.in_features = n, k
        w = DmhLinearWeights(n, k, group_size, *ptrs)
        h = C.c_void_p()
        if not host:  # (what made the arrays, on any stream)
            import torch
            torch.cuda.synchronize(blk.device)
        check(blk._lib.dmh_upload_linear(blk.handle, C.addressof(w), 0 if host else DMH_F_DEVICE,
                                         C.byref(h), self._err, 2048), self._err)
        self._l = h.value
        self._c = DmhLinearRows()
        self._ref = C.addressof(self._c)

    @classmethod
    def from_quant_model(cls, blk, index, name: str, bias=None):
        """The layer of tensor `name` [out_features][in_features] of a quant model
        (formats.scan_quant_file)."""
        i = index.find(name)
        if i < 0:
            raise _bad(f"tensor {name} is not in the quant model")
        info = index.tensors[i]
        if len(info.shape) != 2:
            raise _bad(f"tensor {name} has {len(info.shape)} dimensions, not 2")
        scales, packed = index.read(i)
        return cls(blk, *info.shape, scales, packed, group_size=info.group_size, bias=bias)

    def close(self):
        if getattr(self, "_l", None) and self._blk.handle:
            self._blk._lib.dmh_free_linear(self._blk.handle, self._l)
        self._l = None

    def __del__(self):
        self.close()

    def __call__(self, x, out):
        """out [rows][out_features] for rows x [rows][in_features]; out has x's type or is
        float32."""
        c = self._c
        dev = None if isinstance(x, np.ndarray) else self._blk.device
        c.dtype, c.out_dtype = _type(x), _type(out)
        if c.out_dtype != c.dtype and c.out_dtype != F32:
            raise _bad("out must have x's type or be float32")
        n, c.x, c.x_stride = self._rows1(x, self.in_features, x.dtype, dev, "x")
        m, c.y, c.y_stride = self._rows1(out, self.out_features, out.dtype, dev, "out")
        if n != m or n >= 1 << 30:
            raise _bad("x and out differ in their rows, or have 2^30 or more")
        c.rows = n
        blk, e = self._blk, self._err
        rc = blk._lib.dmh_linear_forward(blk.handle, self._l, self._ref,
                                         0 if dev is None else DMH_F_DEVICE, e, 2048)
        if rc:
            check(rc, e)
        return out
