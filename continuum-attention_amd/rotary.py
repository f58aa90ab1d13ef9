"""Rotary positions for any positions, layout and part of the head.

The decoder's training layer rotates inside its attention kernels, in one form
(``decoder.apply_rope``: whole heads, neighbouring pairs, positions 0..T-1, each
step rounded to the operands' type as the reference rounds it).  Here positions
are given per token, a head may turn in part, pairs may be neighbours or halves,
and frequencies may be scaled for contexts longer than the trained one; angles
are formed in 64 bits and the result rounded once.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native

_DTYPES = {torch.float32: _native.CA_DTYPE_F32, torch.bfloat16: _native.CA_DTYPE_BF16,
           torch.float16: _native.CA_DTYPE_F16}
_LAYOUTS = ("interleaved", "half")
_SCALINGS = (None, "linear", "ntk", "yarn")


class Rotary:
    """The frequencies of a rotary embedding, on a device.

    Pair i of a head's first ``rotary_dim`` dims (default: all) turns by
    position * f_i radians, f_i = theta^(-2i / rotary_dim); ``layout`` pairs dims
    (2i, 2i + 1) ("interleaved") or (i, i + rotary_dim / 2) ("half").  For contexts
    ``factor`` times the trained one, ``scaling``

    * "linear" divides every f_i by the factor (positions are interpolated);
    * "ntk" takes theta * factor^(rotary_dim / (rotary_dim - 2)), which leaves the
      fastest pair and divides the slowest by the factor;
    * "yarn" keeps the f_i that make at least ``beta_fast`` turns over
      ``original_length`` positions, divides those that make at most ``beta_slow``
      by the factor and goes linearly between (by the number of turns), and
      multiplies the rotated values by 0.1 ln(factor) + 1.

    ``frequencies`` (radians per position of each pair) and ``magnitude`` replace
    what theta and the scaling give."""

    def __init__(self, head_dim, theta=10000.0, rotary_dim=None, layout="interleaved", scaling=None,
                 factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0, frequencies=None,
                 magnitude=None, device=None):
        rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if head_dim <= 0 or head_dim % 2 or rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} of head dim {head_dim}: both must be positive and even")
        if layout not in _LAYOUTS:
            raise ValueError("layout must be one of " + ", ".join(_LAYOUTS))
        if scaling not in _SCALINGS:
            raise ValueError("scaling must be None, linear, ntk or yarn")
        if not theta > 0 or not factor >= 1:
            raise ValueError("theta must be positive and factor at least 1")
        if frequencies is None:
            if scaling == "ntk":
                if rotary_dim == 2:
                    raise ValueError("ntk scaling needs a rotary_dim above 2")
                theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
            f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
            if scaling == "linear":
                f = f / factor
            elif scaling == "yarn":
                if original_length is None or original_length <= 0:
                    raise ValueError("yarn scaling needs the original_length")
                if not beta_fast > beta_slow:
                    raise ValueError("beta_fast must be above beta_slow")
                turns = original_length * f / (2 * math.pi)
                keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
                f = f * keep + f / factor * (1 - keep)
        else:
            f = torch.as_tensor(frequencies, dtype=torch.float64).detach().cpu()
            if f.shape != (rotary_dim // 2,):
                raise ValueError(f"frequencies must be [{rotary_dim // 2}], got {tuple(f.shape)}")
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" and frequencies is None else 1.0
        self.head_dim, self.rotary_dim, self.layout = int(head_dim), rotary_dim, layout
        self.magnitude = float(magnitude)
        self.turns = (f / (2 * math.pi)).to(device if device is not None else "cpu")

    def to(self, device):
        """This embedding with its frequencies on ``device``."""
        device = torch.device(device)
        if self.turns.device == device:
            return self
        other = object.__new__(Rotary)
        other.__dict__.update(self.__dict__)
        other.turns = self.turns.to(device)
        return other


def _rows(name, x, rotary, like=None):
    """``x`` [..., H, D] as [N, H, D] rows the kernels read."""
    if not isinstance(x, torch.Tensor) or x.dim() < 3:
        raise ValueError(f"{name} must be [..., heads, head_dim]")
    if x.shape[-1] != rotary.head_dim:
        raise ValueError(f"{name} has head dim {x.shape[-1]}, the rotary embedding {rotary.head_dim}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: unsupported dtype {x.dtype}")
    if like is not None and (x.dtype != like.dtype or x.device != like.device or x.shape[:-2] != like.shape[:-2]):
        raise ValueError(f"q and {name} must share dtype, device and leading dims")
    x = x.detach().resolve_neg()
    if x.dim() != 3:
        x = x.reshape(-1, *x.shape[-2:])
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _positions(positions, lead, device):
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be a tensor of 32- or 64-bit integers")
    if positions.device != device:
        raise RuntimeError("positions must be on the device of q")
    if positions.shape != lead:
        try:
            positions = positions.expand(lead)
        except RuntimeError:
            raise ValueError(f"positions of shape {tuple(positions.shape)} do not fit tokens {tuple(lead)}") from None
    return positions.reshape(-1).contiguous()


def _argument(q, k, q_out, k_out, positions, rotary, inverse):
    r = _native.Rotary()
    if rotary.turns.device != q.device:
        raise RuntimeError("the rotary embedding is on another device (Rotary.to)")
    for t in (k, positions):  # saved-tensor hooks may have moved the positions
        if t is not None and t.device != q.device:
            raise RuntimeError("rotary_embedding: all tensors must be on the same GPU")
    r.q, r.q_out = q.data_ptr(), q_out.data_ptr()
    r.q_token_stride, r.q_head_stride, _ = q.stride()
    r.q_out_token_stride, r.q_out_head_stride, _ = q_out.stride()
    if k is not None:
        r.k = k.data_ptr()
        r.k_token_stride, r.k_head_stride, _ = k.stride()
        r.k_heads = k.shape[1]
        if k_out is not None:
            r.k_out = k_out.data_ptr()
            r.k_out_token_stride, r.k_out_head_stride, _ = k_out.stride()
    r.positions, r.positions64 = positions.data_ptr(), positions.dtype == torch.int64
    r.turns, r.magnitude = rotary.turns.data_ptr(), rotary.magnitude
    r.half, r.inverse = rotary.layout == "half", inverse
    r.dtype, r.tokens, r.q_heads = _DTYPES[q.dtype], q.shape[0], q.shape[1]
    r.head_dim, r.rotary_dim = rotary.head_dim, rotary.rotary_dim
    return r


def _turn_cpu(x, positions, rotary, inverse=False):
    """[N, H, D] rotated on the CPU."""
    R = rotary.rotary_dim
    t = positions.double()[:, None, None] * rotary.turns
    angle = (t - t.round()) * (2 * math.pi)
    cos, sin = (angle.cos() * rotary.magnitude).float(), (angle.sin() * rotary.magnitude).float()
    if inverse:
        sin = -sin
    xf = x.float()
    pairs = xf[..., :R].unflatten(-1, (-1, 2) if rotary.layout == "interleaved" else (2, -1))
    axis = -1 if rotary.layout == "interleaved" else -2
    a, b = pairs.unbind(axis)
    head = torch.stack((a * cos - b * sin, b * cos + a * sin), axis).flatten(-2)
    return torch.cat((head, xf[..., R:]), -1).to(x.dtype)


def _turn(q, k, positions, rotary, inverse):
    """Rotated q and k (None stays None); [N, H, D] rows in, contiguous out."""
    if q.device.type == "cpu":
        return (_turn_cpu(q, positions, rotary, inverse),
                None if k is None else _turn_cpu(k, positions, rotary, inverse))
    if q.device.type != "cuda":
        raise RuntimeError(f"rotary_embedding runs on ROCm GPU and CPU tensors; got one on {q.device}")
    q_out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=k.device, dtype=k.dtype)
    if q.numel() or (k is not None and k.numel()):
        r = _argument(q, k, q_out, k_out, positions, rotary, inverse)
        with _native.on_device(q.device):
            _native.check(_native.load().ca_rotary_embedding(ctypes.byref(r), _native.stream_handle(q.device)))
    return q_out, k_out


class _RotaryFn(torch.autograd.Function):
    """The rotation is linear and its transpose the rotation back, so nothing of
    q and k is kept and the backward is this function again, of any order."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        q3 = _rows("q", q, rotary)
        k3 = None if k is None else _rows("k", k, rotary, q)
        yq, yk = _turn(q3, k3, positions, rotary, inverse)
        yq = yq.view(q.shape)
        return yq if k is None else (yq, yk.view(k.shape))

    @staticmethod
    def backward(ctx, gq, gk=None):
        (positions,) = ctx.saved_tensors
        given = [g for g in (gq, gk) if g is not None]
        if not given:
            return None, None, None, None, None
        y = _RotaryFn.apply(given[0], given[1] if len(given) > 1 else None, positions, ctx.rotary,
                            not ctx.inverse)
        y = list(y) if len(given) > 1 else [y]
        return (y.pop(0) if gq is not None else None, y.pop(0) if gk is not None else None, None, None, None)


def rotary_embedding(q, k, positions, rotary):
    """``(q, k)`` with their heads turned to ``positions`` (``k`` may be None).

    q, k: ``[..., heads, head_dim]`` of one dtype (fp32, bf16 or fp16) and one
    leading shape, in any strides; positions: integers of the leading shape, or
    one that expands to it.  Differentiable in q and k.  On the GPU one kernel
    each way; the results are contiguous, in the inputs' dtype, rounded once."""
    # the plain case (see csrc/ca_torch.cpp) runs _RotaryFn's native counterpart
    if (isinstance(q, torch.Tensor) and q.is_cuda and q.dim() > 2 and q.shape[-1] == rotary.head_dim
            and not torch.compiler.is_compiling()):
        y = _native.torch_ext().rotary(q, k, positions, rotary.turns, rotary.magnitude, rotary.layout == "half",
                                       rotary.rotary_dim)
        if y is not None:
            return y
    _rows("q", q, rotary)
    if k is not None:
        _rows("k", k, rotary, q)
    p = _positions(positions, q.shape[:-2], q.device)
    y = _RotaryFn.apply(q, k, p, rotary, False)
    return (y, None) if k is None else y
