"""verify_drafts(...): drafted tokens against the target model's probabilities,
from given random numbers (no counterpart in the reference, which does not
decode). The tokens that come out follow the target's distribution exactly,
whatever the draft; see include/lizard_cuda.h (lz_verify_drafts) for the rule.
"""
import torch

from . import _lib

_DT = {torch.float32: _lib.LZ_DTYPE_F32, torch.bfloat16: _lib.LZ_DTYPE_BF16}


def _logits(t, dtype):
    t = t if t.dtype == dtype else t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def verify_drafts(target_logits, draft_logits, draft_tokens, uniforms, noise, temperature=1.0,
                  lengths=None):
    """(tokens [B, K + 1], accepted int32 [B]) for K <= 64 drafted tokens a sequence.

    target_logits [B, K + 1, V]: the target's logits at the K drafted positions
    and the one after. draft_logits [B, K, V]: the logits the drafted tokens
    [B, K] (int64 or int32) were drawn from, at the same temperature. uniforms
    fp32 [B, K] in [0, 1) decide the acceptances, noise fp32 [B, V] from Exp(1)
    (torch.Tensor.exponential_) draws the token that follows. temperature: a
    number or fp32 [B]; below 1e-5 a sequence is greedy. lengths int32 [B]:
    drafted tokens of each sequence (0..K) when they differ. tokens holds the
    accepted tokens, the next one, and -1 beyond; the next one is -1 only where
    the target's row is masked (-inf or NaN) throughout."""
    _lib.require_cuda(target_logits, draft_logits, draft_tokens, uniforms, noise)
    if target_logits.dim() != 3 or target_logits.shape[1] < 1:
        raise ValueError(f"target_logits must be [B, K + 1, V], got {tuple(target_logits.shape)}")
    B, K, V = target_logits.shape[0], target_logits.shape[1] - 1, target_logits.shape[2]
    want = {"draft_logits": (draft_logits, (B, K, V)), "draft_tokens": (draft_tokens, (B, K)),
            "uniforms": (uniforms, (B, K)), "noise": (noise, (B, V))}
    for name, (t, shape) in want.items():
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    if draft_tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"draft_tokens must be int64 or int32, got {draft_tokens.dtype}")
    temp, temp_all = None, 1.0
    if isinstance(temperature, torch.Tensor):
        _lib.require_cuda(target_logits, temperature)
        if tuple(temperature.shape) != (B,):
            raise ValueError(f"temperature must be a number or [{B}], got "
                             f"{tuple(temperature.shape)}")
        temp = temperature.float().contiguous()
    else:
        temp_all = float(temperature)
        if not 0 <= temp_all < float("inf"):
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    if lengths is not None:
        _lib.require_cuda(target_logits, lengths)
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,):
            raise ValueError(f"lengths must be int32 [{B}], got {lengths.dtype} "
                             f"{tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    dev = target_logits.device
    out = torch.empty(B, K + 1, device=dev, dtype=draft_tokens.dtype)
    accepted = torch.empty(B, device=dev, dtype=torch.int32)
    if B == 0:
        return out, accepted
    xdt = target_logits.dtype if target_logits.dtype in _DT else torch.float32
    t, d = _logits(target_logits, xdt), _logits(draft_logits, xdt)
    tok, u, e = draft_tokens.contiguous(), uniforms.float().contiguous(), _logits(noise, torch.float32)
    ws = torch.empty(_lib.size_query("lz_verify_drafts_workspace_bytes", B, K, V), device=dev,
                     dtype=torch.uint8)
    with _lib.on_device(dev):
        rc = _lib.load().lz_verify_drafts(
            _lib.ptr(t), t.stride(0), t.stride(1), _lib.ptr(d), d.stride(0), d.stride(1), _DT[xdt],
            _lib.ptr(tok), int(tok.dtype == torch.int64), _lib.ptr(u), _lib.ptr(e), e.stride(0),
            _lib.ptr(temp), temp_all, _lib.ptr(lengths), _lib.ptr(out), _lib.ptr(accepted),
            _lib.ptr(ws), ws.numel(), B, K, V, _lib.stream_of(t))
    _lib.check(rc, "verify drafts")
    return out, accepted
