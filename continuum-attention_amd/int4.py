"""Products with weights of four bits and a scale per group of columns.

``y[m, n] = sum_k x[m, k] scale[n, k / g] (code[n, k] - zero[n, k / g])``: a
linear layer's product for the few rows of a decoding step, bound by the bytes of
its weights, which are a quarter of their 16-bit ones.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _native
from .rotary import _DTYPES


def _check_group(group_size):
    if group_size not in (32, 64) and (group_size <= 0 or group_size % 128):
        raise ValueError(f"groups of {group_size} columns: 32, 64 or a multiple of 128")


def _aligned(t):
    t = t.detach().resolve_neg().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


# bits of a word's eight columns
_BITS = (0, 16, 4, 20, 8, 24, 12, 28)


class Int4Weight:
    """An ``[out, in]`` matrix of 4-bit codes as the kernel reads them.

    With the rows rounded up to a multiple of 16, ``codes`` is int32 ``[rows / 16,
    ceil(in / 128), 64, 4]``, tiles of 16 rows by 128 columns: word (16r + i, j) holds
    row i, columns c = 32j + 8r .. c + 7, column c + 2p in bits 4p and column c + 2p + 1
    in bits 16 + 4p.  ``scales`` and ``zeros`` (or None: 8) are ``[ceil(in / group), rows]``
    in the activations' dtype.  from_codes and quantize make them."""

    def __init__(self, codes, scales, zeros, out_features, in_features, group_size):
        _check_group(group_size)
        groups, rows = -(-in_features // group_size), -(-out_features // 16) * 16
        shape = (rows // 16, -(-in_features // 128), 64, 4)
        if min(out_features, in_features) < 1 or codes.dtype != torch.int32 or codes.shape != shape:
            raise ValueError(f"codes must be int32 {list(shape)}")
        if scales.dtype not in _DTYPES or scales.shape != (groups, rows):
            raise ValueError(f"scales must be fp32, bf16 or fp16 [{groups}, {rows}]")
        if zeros is not None and (zeros.dtype != scales.dtype or zeros.shape != scales.shape):
            raise ValueError("zeros must have the scales' dtype and shape")
        for t in (scales, zeros):
            if t is not None and t.device != codes.device:
                raise RuntimeError("codes, scales and zeros must be on one device")
        self.codes, self.scales = _aligned(codes), _aligned(scales)
        self.zeros = None if zeros is None else _aligned(zeros)
        self.in_features, self.out_features = int(in_features), int(out_features)
        self.group_size = int(group_size)

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, group_size=128):
        """From codes ``[out, in]`` (integers 0..15), scales ``[out, groups]`` and
        zero points ``[out, groups]`` (or None: 8)."""
        _check_group(group_size)
        if codes.dim() != 2 or codes.is_floating_point() or codes.shape[0] < 1 or codes.shape[1] < 1:
            raise ValueError("codes must be integers [out, in]")
        out, k = codes.shape
        shape = (out, -(-k // group_size))
        if scales.shape != shape or (zeros is not None and zeros.shape != shape):
            raise ValueError(f"scales and zeros must be {list(shape)}")
        pad = -out % 16
        c = nn.functional.pad(codes.to(torch.int32) & 15, (0, -k % 128, 0, pad))
        bits = torch.tensor(_BITS, dtype=torch.int32, device=codes.device)
        # disjoint bits (the last's sign wraps into place); [tile, i, block, j, r] to [tile, block, r, i, j]
        words = (c.view((out + pad) // 16, 16, -1, 4, 4, 8) << bits).sum(-1, dtype=torch.int32).permute(0, 2, 4, 1, 3)
        s, z = (None if t is None else nn.functional.pad(t.to(scales.dtype), (0, 0, 0, pad)).t().contiguous()
                for t in (scales, zeros))
        return cls(words.reshape(words.shape[0], -1, 64, 4), s, z, out, k, group_size)

    @classmethod
    def quantize(cls, weight, group_size=128, zero_points=False, dtype=None):
        """From a floating-point ``[out, in]`` weight: each group's values to the
        nearest of 15 codes around 8 (step: largest magnitude / 7) or, with
        ``zero_points``, of the 16 codes over the group's range with zero in it.
        Scales in ``dtype`` (default: the weight's)."""
        _check_group(group_size)
        dtype = weight.dtype if dtype is None else dtype
        if weight.dim() != 2 or dtype not in _DTYPES:
            raise ValueError("weight must be [out, in], scales fp32, bf16 or fp16")
        w = weight.detach().float()
        out, k = w.shape
        pad = -(-k // group_size) * group_size - k
        g = nn.functional.pad(w, (0, pad)).view(out, -1, group_size)
        if zero_points:
            lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
            scale = ((hi - lo) / 15).to(dtype).float()
            step = torch.where(scale > 0, scale, 1.0)
            zero = (-lo / step).round().clamp(0, 15)
        else:
            scale = (g.abs().amax(-1) / 7).to(dtype).float()
            step = torch.where(scale > 0, scale, 1.0)
            zero = torch.full_like(step, 8.0)
        codes = (g / step[..., None]).round().add_(zero[..., None]).clamp_(0, 15).to(torch.uint8)
        return cls.from_codes(codes.view(out, -1)[:, :k], scale.to(dtype), zero if zero_points else None, group_size)

    def dequantize(self):
        """The fp32 ``[out, in]`` matrix this stands for."""
        bits = torch.tensor(_BITS, dtype=torch.int32, device=self.codes.device)
        tiles, blocks = self.codes.shape[:2]
        c = (self.codes.view(tiles, blocks, 4, 16, 4).permute(0, 3, 1, 4, 2)[..., None] >> bits) & 15
        c = c.reshape(16 * tiles, -1)[:, :self.in_features].float()
        group = torch.arange(self.in_features, device=c.device) // self.group_size
        zero = 8.0 if self.zeros is None else self.zeros.float()[group].t()
        return ((c - zero) * self.scales.float()[group].t())[:self.out_features]


def int4_linear(x, weight: Int4Weight):
    """``x [..., in] @ weight^T`` in x's dtype (the scales': fp32, bf16, fp16),
    summed in fp32 and rounded once.

    Made for the few rows of a decoding step (any number works; the codes are
    read once per 16 or 32 rows).  No backward pass.  A row of x that holds an
    infinity gives NaN."""
    # the plain case runs in native code (csrc/ca_torch.cpp); what it does not take is checked here
    if x.is_cuda and not torch.compiler.is_compiling():
        y = _native.torch_ext().int4(x, weight.codes, weight.scales, weight.zeros, weight.out_features,
                                     weight.in_features, weight.group_size)
        if y is not None:
            return y
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("int4_linear has no backward pass; call it under torch.no_grad()")
    K, N = weight.in_features, weight.out_features
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1] if x.dim() else 0} columns, the weight {K}")
    if x.dtype != weight.scales.dtype:
        raise ValueError(f"x is {x.dtype}, the weight's scales are {weight.scales.dtype}")
    if x.device != weight.codes.device:
        raise RuntimeError("x and the weight must be on one device")
    rows = x.detach().resolve_neg().reshape(-1, K)
    M = rows.shape[0]
    if x.device.type == "cpu":
        return (rows.float() @ weight.dequantize().t()).to(x.dtype).view(*x.shape[:-1], N)
    if x.device.type != "cuda":
        raise RuntimeError(f"int4_linear runs on ROCm GPU and CPU tensors; got one on {x.device}")
    if rows.stride(1) != 1 and K > 1 or (M > 1 and rows.stride(0) < K):
        rows = rows.contiguous()
    y = torch.empty(M, N, device=x.device, dtype=x.dtype)
    with _native.on_device(x.device):
        _native.check(_native.load().ca_int4_linear(
            rows.data_ptr(), max(rows.stride(0), K), weight.codes.data_ptr(), weight.scales.data_ptr(),
            None if weight.zeros is None else weight.zeros.data_ptr(), y.data_ptr(), N, _DTYPES[x.dtype], M, N, K,
            weight.group_size, _native.stream_handle(x.device)))
    return y.view(*x.shape[:-1], N)


class Int4Linear(nn.Module):
    """A linear layer without bias over an Int4Weight, for inference; its input
    is cast to the scales' dtype.  ``from_linear`` quantizes an nn.Linear."""

    def __init__(self, weight: Int4Weight):
        super().__init__()
        self.in_features, self.out_features = weight.in_features, weight.out_features
        self.group_size = weight.group_size
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("zeros", weight.zeros)

    @classmethod
    def from_linear(cls, linear, group_size=128, zero_points=False, dtype=None):
        if linear.bias is not None:
            raise ValueError("Int4Linear has no bias")
        return cls(Int4Weight.quantize(linear.weight, group_size, zero_points, dtype))

    def forward(self, x):
        x = x.to(self.scales.dtype)
        if x.is_cuda and not torch.compiler.is_compiling():  # as in int4_linear
            y = _native.torch_ext().int4(x, self.codes, self.scales, self.zeros, self.out_features,
                                         self.in_features, self.group_size)
            if y is not None:
                return y
        w = Int4Weight(self.codes, self.scales, self.zeros, self.out_features, self.in_features, self.group_size)
        return int4_linear(x, w)


def quantize_linears(module, group_size=128, zero_points=False, dtype=None, skip=()):
    """Replaces every bias-free nn.Linear below ``module`` (but for those whose
    qualified names are in ``skip``) by its Int4Linear, in place; returns module."""
    for name, child in list(module.named_modules()):
        for key, linear in list(child.named_children()):
            full = f"{name}.{key}" if name else key
            if type(linear) is nn.Linear and linear.bias is None and full not in skip:
                setattr(child, key, Int4Linear.from_linear(linear, group_size, zero_points, dtype))
    return module
