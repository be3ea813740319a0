"""Products with a matrix in 4 bits and a scale per group of a row.

``pack_int4_groups`` quantises a matrix as the corpus packer quantises tokens,
in groups of 32, 64 or 128 columns: ``s = bf16(max|w| / 7)`` and codes
``clip(rint(w / s), -7, 7)``.  ``Int4Linear`` holds it as the product reads it
and multiplies few rows with it (a token, a decoding batch): the matrix'
bytes are what such a product costs.
"""
from __future__ import annotations

import ctypes

from maxsim_amd import _native

GROUP_SIZES = (32, 64, 128)


def pack_int4_groups(weight, group_size: int = 128):
    """(codes u8 [n, k / 2], scales bfloat16 [n, k / group_size]) of a float
    matrix [n, k], on its device.  Codes are two's complement nibbles, the even
    column low; a group of zeros has the scale 1."""
    import torch

    if not torch.is_tensor(weight) or weight.ndim != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a float tensor of shape [out_features, in_features]")
    if group_size not in GROUP_SIZES:
        raise ValueError("group_size must be 32, 64 or 128")
    n, k = weight.shape
    if n < 1 or k < 1 or k % group_size:
        raise ValueError("in_features must be a positive multiple of group_size")
    w = weight.detach().to(torch.float32).reshape(n, k // group_size, group_size)
    if not bool(torch.isfinite(w).all()):
        raise ValueError("weight must contain only finite values")
    peak = w.abs().amax(-1)
    # Divided by a tensor: by a plain number it would be a product with 1 / 7.
    scales = (peak / torch.full_like(peak, 7.0)).to(torch.bfloat16)
    scales = torch.where(scales == 0, torch.ones_like(scales), scales)
    codes = torch.round(w / scales.float()[..., None]).clamp_(-7, 7).to(torch.int8).reshape(n, k).view(torch.uint8)
    return (codes[:, 0::2] & 15) | ((codes[:, 1::2] & 15) << 4), scales


class Int4Linear:
    """``y = x W^T + bias`` with W given by its codes and scales
    (``pack_int4_groups``), on the GPU.  The matrix is laid out once, here."""

    def __init__(self, codes, scales, bias=None):
        import torch

        if not torch.is_tensor(codes) or codes.ndim != 2 or codes.dtype != torch.uint8 or codes.device.type != "cuda":
            raise ValueError("codes must be a uint8 CUDA tensor of shape [out_features, in_features / 2]")
        n, k = codes.shape[0], codes.shape[1] * 2
        if not torch.is_tensor(scales) or scales.ndim != 2 or scales.dtype != torch.bfloat16 or \
                scales.device != codes.device or scales.shape[0] != n or scales.shape[1] < 1:
            raise ValueError("scales must be a bfloat16 tensor of shape [out_features, in_features / group_size] "
                             "on the device of codes")
        group = k // scales.shape[1]
        if group not in GROUP_SIZES or group * scales.shape[1] != k:
            raise ValueError("group_size must be 32, 64 or 128")
        if bias is not None and (not torch.is_tensor(bias) or bias.shape != (n,) or bias.device != codes.device
                                 or not bias.is_floating_point()):
            raise ValueError("bias must be a float tensor of shape [out_features] on the device of codes")
        self.out_features, self.in_features, self.group_size, self.device = n, k, group, codes.device
        self.bias = None if bias is None else bias.detach().to(torch.float32).contiguous()
        lib = _native.load()
        sizes = ctypes.c_uint64(0), ctypes.c_uint64(0)
        _native.check(lib.msim_linear4_layout_bytes(n, k, group, *map(ctypes.byref, sizes)))
        self._codes = torch.empty(sizes[0].value, dtype=torch.uint8, device=self.device)
        self._scales = torch.empty(sizes[1].value // 2, dtype=torch.bfloat16, device=self.device)
        codes, scales = codes.contiguous(), scales.contiguous()
        with torch.cuda.device(self.device):
            _native.check(lib.msim_linear4_layout_async(
                codes.data_ptr(), scales.data_ptr(), n, k, group, self._codes.data_ptr(), self._scales.data_ptr(),
                torch.cuda.current_stream().cuda_stream))
        self._calls = _native.tensor_calls()
        self._handle = self._calls.linear(self._codes, self._scales, self.bias, n, k, group)

    @classmethod
    def from_float(cls, weight, group_size: int = 128, bias=None) -> "Int4Linear":
        """Quantises a float CUDA matrix [out_features, in_features]."""
        return cls(*pack_int4_groups(weight, group_size), bias=bias)

    @property
    def resident_bytes(self) -> int:
        return self._codes.numel() + 2 * self._scales.numel() + (0 if self.bias is None else 4 * self.bias.numel())

    def __call__(self, x, out=None):
        """x [..., in_features] (float32, float16 or bfloat16) to [...,
        out_features] in x's dtype: sums in single precision, rounded once.
        ``out`` is contiguous and does not overlap x.
        Enqueued on the current stream; records no gradients.  Meant for few
        rows: the matrix is read once per 16 or 32 of them."""
        return self._calls.multiply(self._handle, x, out)
