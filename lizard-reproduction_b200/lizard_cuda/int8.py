"""Matrix products in 8-bit integers with one scale a token and one a channel,
for serving (no counterpart in the reference).

  codes, scale = int8_quantize(w)          # once: a weight [N, K], or any rows
  y = int8_linear(x, codes, scale, bias)   # x [..., K] fp32 / bf16, quantised per row
  y = int8_matmul(a, a_scale, b, b_scale)  # both sides quantised already

scale = max|row| / 127 and code = rint(x * (127 / max|row|)) in fp32; the product
is an exact 32-bit integer sum times (token scale * channel scale), plus the
bias, rounded once to the output type. A row that holds an infinity or NaN gives
NaN throughout. int8_quantize lays rows of codes out on 16-byte boundaries, the
layout the tensor cores read in place; codes in other layouts are repacked on
every call. There is no backward.
"""
import struct

import torch
import torch.nn as nn

from . import _lib

_DT = {torch.float32: _lib.LZ_DTYPE_F32, torch.bfloat16: _lib.LZ_DTYPE_BF16}
_words = struct.Struct("16q").pack


def _rows(t):
    """t [..., K] as rows [M, K] with a contiguous last dimension (a view where it can be)."""
    if t.dim() != 2:
        t = t.unsqueeze(0) if t.dim() == 1 else t.flatten(0, -2)
    if t.is_contiguous():
        return t
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _no_grad(*tensors):
    if not torch.is_grad_enabled():
        return
    if any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("8-bit products have no backward; call them under torch.no_grad()")


def int8_quantize(x):
    """(codes int8 [..., K], scale fp32 [...]) of x [..., K] (fp32 or bf16; other
    float types are computed as fp32), one scale a row. The codes' rows start on
    16-byte boundaries."""
    _lib.require_cuda(x)
    _no_grad(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [..., K] with K >= 1, got {tuple(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    xr = _rows(x if x.dtype in _DT else x.float())
    M = xr.shape[0]
    codes = torch.empty(M, -(-K // 16) * 16, device=x.device, dtype=torch.int8)
    scale = torch.empty(M, device=x.device, dtype=torch.float32)
    if M:
        with _lib.on_device(x.device):
            rc = _lib.load().lz_int8_quantize(
                _lib.ptr(xr), _DT[xr.dtype], xr.stride(0), _lib.ptr(codes), codes.shape[1],
                _lib.ptr(scale), M, K, _lib.stream_of(x))
        _lib.check(rc, "int8 quantize")
    return codes.view(*lead, codes.shape[1])[..., :K], scale.view(lead)


def _check(K, N, b, b_scale, bias, dtype):
    if b.dim() != 2 or b.dtype is not torch.int8 or b.shape[1] != K or N < 1 or K < 1:
        raise ValueError(f"the weight codes must be int8 [N, {K}], got {b.dtype} {tuple(b.shape)}")
    if b_scale.dtype is not torch.float32 or b_scale.shape != (N,):
        raise ValueError(f"the weight's scale must be fp32 [{N}], got {b_scale.dtype} "
                         f"{tuple(b_scale.shape)}")
    if bias is not None and (bias.shape != (N,) or bias.dtype not in _DT):
        raise ValueError(f"bias must be fp32 or bf16 [{N}], got {bias.dtype} {tuple(bias.shape)}")
    if dtype not in _DT:
        raise ValueError(f"the output type must be float32 or bfloat16, got {dtype}")


def _aligned(t):
    return t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or t.stride(0) % 16 == 0)


def int8_matmul(a, a_scale, b, b_scale, bias=None, dtype=torch.bfloat16):
    """y [..., N] = (a b^T) * a_scale * b_scale + bias for codes a int8 [..., K],
    b int8 [N, K] and scales fp32 [...] and [N], in `dtype` (bf16 or fp32)."""
    index = a.get_device()
    if not (index == a_scale.get_device() == b.get_device() == b_scale.get_device()
            == (index if bias is None else bias.get_device()) >= 0):
        _lib.require_cuda(a, a_scale, b, b_scale, *(() if bias is None else (bias,)))
    _no_grad(a_scale, b_scale, bias)
    if a.dim() < 1 or a.dtype is not torch.int8:
        raise ValueError(f"a must be int8 [..., K], got {a.dtype} {tuple(a.shape)}")
    lead, K, N = a.shape[:-1], a.shape[-1], b.shape[0]
    if a_scale.dtype is not torch.float32 or a_scale.shape != lead:
        raise ValueError(f"a's scale must be fp32 {tuple(lead)}, got {a_scale.dtype} "
                         f"{tuple(a_scale.shape)}")
    _check(K, N, b, b_scale, bias, dtype)
    y = a.new_empty((*lead, N), dtype=dtype)
    ar = _rows(a)
    M = ar.shape[0]
    if M:
        br = _rows(b)
        sa, sb = a_scale.contiguous(), b_scale.contiguous()
        bias = None if bias is None else bias.contiguous()
        ws = None
        if not (_aligned(ar) and _aligned(br)):
            ws = a.new_empty(_lib.size_query("lz_int8_workspace_bytes", M, N, K))
        rc = _lib.call(index, _lib.CALL_INT8_MATMUL, _words(
            ar.data_ptr(), ar.stride(0), sa.data_ptr(), br.data_ptr(), br.stride(0),
            sb.data_ptr(), 0 if bias is None else bias.data_ptr(),
            0 if bias is None else _DT[bias.dtype], y.data_ptr(), _DT[dtype],
            0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), M, N, K,
            _lib.raw_stream(index)))
        if rc:
            _lib.check(rc, "int8 matmul")
    return y


def int8_linear(x, weight, weight_scale, bias=None, dtype=None):
    """y [..., N] = x W^T + bias with x [..., K] (fp32 or bf16) quantised row by
    row and the weight given as codes int8 [N, K] with a scale fp32 [N] for each
    channel (int8_quantize of an nn.Linear weight), in `dtype` (fp32 or bf16; x's by
    default). Other float types of x are computed as fp32, whose result is then
    rounded to x's type."""
    index = x.get_device()
    if not (index == weight.get_device() == weight_scale.get_device()
            == (index if bias is None else bias.get_device()) >= 0):
        _lib.require_cuda(x, weight, weight_scale, *(() if bias is None else (bias,)))
    _no_grad(x, weight_scale, bias)
    if x.dim() < 1:
        raise ValueError(f"x must be [..., K], got {tuple(x.shape)}")
    given = None  # the type of the result where the kernels do not write it
    if x.dtype not in _DT:
        if dtype is None and x.is_floating_point():
            given = x.dtype
        x = x.float()
    lead, K, N = x.shape[:-1], x.shape[-1], weight.shape[0]
    if dtype is None:
        dtype = x.dtype
    _check(K, N, weight, weight_scale, bias, dtype)
    y = x.new_empty((*lead, N), dtype=dtype)
    xr = _rows(x)
    M = xr.shape[0]
    if M:
        w, ws = _rows(weight), weight_scale.contiguous()
        bias = None if bias is None else bias.contiguous()
        size = (_lib.size_query("lz_int8_linear_workspace_bytes", M, N, K) if _aligned(w)
                else _lib.size_query("lz_int8_workspace_bytes", M, N, K))
        work = w.new_empty(size) if size else None
        rc = _lib.call(index, _lib.CALL_INT8_LINEAR, _words(
            xr.data_ptr(), _DT[xr.dtype], xr.stride(0), w.data_ptr(), w.stride(0), ws.data_ptr(),
            0 if bias is None else bias.data_ptr(), 0 if bias is None else _DT[bias.dtype],
            y.data_ptr(), _DT[dtype], work.data_ptr() if size else 0, size, M, N, K,
            _lib.raw_stream(index)))
        if rc:
            _lib.check(rc, "int8 linear")
    return y if given is None else y.to(given)


class Int8Linear(nn.Module):
    """nn.Linear for inference with the weight held as 8-bit codes and a scale for
    each output channel; inputs are quantised token by token. Build it from a
    linear layer on the GPU: Int8Linear(linear)."""

    def __init__(self, linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        with torch.no_grad():
            codes, scale = int8_quantize(linear.weight)
        # the padded rows are the buffer (a copy of a view would lose their alignment)
        self.register_buffer("codes", codes.as_strided(
            (codes.shape[0], codes.stride(0)), codes.stride()))
        self.register_buffer("scale", scale)
        bias = linear.bias
        if bias is not None:  # in a type that the product takes
            bias = bias.detach().clone() if bias.dtype in _DT else bias.detach().float()
        self.register_buffer("bias", bias)

    def _apply(self, fn, recurse=True):
        """Casts of the module (.half(), .to(dtype)) move the scales and do not round them;
        the bias is cast, to fp32 where the product does not take the type."""
        scale = self.scale
        super()._apply(fn, recurse)
        if self.scale.dtype is not torch.float32:
            self.scale = scale.to(self.scale.device)
        if self.bias is not None and self.bias.dtype not in _DT:
            self.bias = self.bias.float()
        return self

    def forward(self, x):
        return int8_linear(x, self.codes[:, :self.in_features], self.scale, self.bias)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, int8"
