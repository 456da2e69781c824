"""verify_drafts(...): drafted tokens against the target model's probabilities,
from given random numbers (no counterpart in the reference, which does not
decode). The tokens that come out follow the target's distribution exactly,
whatever the draft; see include/lizard_cuda.h (lz_verify_drafts) for the rule.
"""
import struct

import torch

from . import _lib

_DT = {torch.float32: _lib.LZ_DTYPE_F32, torch.bfloat16: _lib.LZ_DTYPE_BF16}
_words = struct.Struct("13qd9q").pack


def _logits(t, dtype):
    if t.dtype is not dtype:
        t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def verify_drafts(target_logits, draft_logits, draft_tokens, uniforms, noise, temperature=1.0,
                  lengths=None):
    """(tokens [B, K + 1], accepted int32 [B]) for K <= 64 drafted tokens a sequence.

    target_logits [B, K + 1, V]: the target's logits at the K drafted positions
    and the one after. draft_logits [B, K, V]: the logits the drafted tokens
    [B, K] (int64 or int32) were drawn from, at the same temperature. Logits of one
    type, bf16 or fp32, are read in place, others (and two types) as fp32. uniforms
    fp32 [B, K] in [0, 1) decide the acceptances, noise fp32 [B, V] from Exp(1)
    (torch.Tensor.exponential_) draws the token that follows. temperature: a
    number or fp32 [B]; below 1e-5 a sequence is greedy. lengths int32 [B]:
    drafted tokens of each sequence (0..K) when they differ. tokens holds the
    accepted tokens, the next one, and -1 beyond; the next one is -1 only where
    the target's row is masked (-inf or NaN) throughout."""
    index = target_logits.get_device()
    if not (index == draft_logits.get_device() == draft_tokens.get_device()
            == uniforms.get_device() == noise.get_device() >= 0):
        _lib.require_cuda(target_logits, draft_logits, draft_tokens, uniforms, noise)
    if target_logits.dim() != 3 or target_logits.shape[1] < 1:
        raise ValueError(f"target_logits must be [B, K + 1, V], got {tuple(target_logits.shape)}")
    B, K1, V = target_logits.shape
    K = K1 - 1
    if (draft_logits.shape != (B, K, V) or draft_tokens.shape != (B, K)
            or uniforms.shape != (B, K) or noise.shape != (B, V)):
        _wrong_shape(draft_logits=(draft_logits, (B, K, V)), draft_tokens=(draft_tokens, (B, K)),
                     uniforms=(uniforms, (B, K)), noise=(noise, (B, V)))
    if draft_tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"draft_tokens must be int64 or int32, got {draft_tokens.dtype}")
    temp, temp_all = None, 1.0
    if isinstance(temperature, torch.Tensor):
        _lib.require_cuda(target_logits, temperature)
        if temperature.shape != (B,):
            raise ValueError(f"temperature must be a number or [{B}], got "
                             f"{tuple(temperature.shape)}")
        temp = _lib.as_dtype(temperature, torch.float32)
    else:
        temp_all = float(temperature)
        if not 0 <= temp_all < float("inf"):
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if lengths is not None:
        _lib.require_cuda(target_logits, lengths)
        if lengths.dtype is not torch.int32 or lengths.shape != (B,):
            raise ValueError(f"lengths must be int32 [{B}], got {lengths.dtype} "
                             f"{tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    out = draft_tokens.new_empty((B, K1))
    accepted = draft_tokens.new_empty(B, dtype=torch.int32)
    if B == 0:
        return out, accepted
    xdt = target_logits.dtype
    if xdt not in _DT or K and draft_logits.dtype is not xdt:
        xdt = torch.float32  # holds both: rounded draft logits are not what the draft drew from
    t, d = _logits(target_logits, xdt), _logits(draft_logits, xdt)
    e = _logits(noise, torch.float32)
    tok, u = draft_tokens.contiguous(), _lib.as_dtype(uniforms, torch.float32)
    size = _lib.size_query("lz_verify_drafts_workspace_bytes", B, K, V)
    ws = noise.new_empty(size // 4, dtype=torch.float32)  # whole 16-byte records
    (tb, tr, _), (db, dr, _) = t.stride(), d.stride()
    rc = _lib.call(index, _lib.CALL_VERIFY_DRAFTS, _words(
        t.data_ptr(), tb, tr, d.data_ptr(), db, dr, _DT[xdt], tok.data_ptr(),
        tok.dtype is torch.int64, u.data_ptr(), e.data_ptr(), e.stride(0),
        0 if temp is None else temp.data_ptr(), temp_all,
        0 if lengths is None else lengths.data_ptr(), out.data_ptr(), accepted.data_ptr(),
        ws.data_ptr(), size, B, K, V, _lib.raw_stream(index)))
    if rc:
        _lib.check(rc, "verify drafts")
    return out, accepted


def _wrong_shape(**tensors):
    for name, (t, shape) in tensors.items():
        if t.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
