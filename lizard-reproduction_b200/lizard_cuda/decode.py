"""Recurrent decode for the Lizard layer: O(1) work per new token.

The reference has no cache; its layer recomputes the whole sequence on every
call (src/lizard_attention.py:78-97). Both branches have a recurrent form
that gives the full-sequence output at the new position:
  * GLA: a running state S [F, D] and normaliser z [F] (fp32), decayed by the
    token's gate and extended by fk^T v, read out as fq S / (fq . z);
  * SWA: a ring of the last `window` rotated keys and values (fp32), attended
    with the sink logits.
gla_state / swa_ring build both from a prompt; gla_decode / swa_decode advance
them by one token on the GPU (lz_gla_decode, lz_swa_decode).

With a gate shared by the heads (log_gamma [B, L], the layer's case) and
grouped keys / values, the H / Hkv query heads of a group read the same state,
so the cache keeps Hkv states per batch row.
"""
import struct
from dataclasses import dataclass

import torch

from . import _lib

_DT = {torch.float32: _lib.LZ_DTYPE_F32, torch.bfloat16: _lib.LZ_DTYPE_BF16}


def gla_state(fk, v, log_gamma):
    """(S [B, Hs, F, D], z [B, Hs, F]) fp32 after the prompt, from a zero state.
    fk [B, Hs, L, F], v [B, Hs, L, D], log_gamma [B, L] or [B, Hs, L]."""
    _lib.require_cuda(fk, v, log_gamma)
    B, Hs, L, F = fk.shape
    D = v.shape[-1]
    if tuple(v.shape[:3]) != (B, Hs, L):
        raise ValueError(f"v must be [B, Hs, L, D] matching fk, got {tuple(v.shape)}")
    per_head = {(B, L): 0, (B, Hs, L): 1}.get(tuple(log_gamma.shape))
    if per_head is None:
        raise ValueError(f"log_gamma must be [B, L] or [B, Hs, L], got {tuple(log_gamma.shape)}")
    lib = _lib.load()
    fk16, v16 = fk.to(torch.bfloat16).contiguous(), v.to(torch.bfloat16).contiguous()
    lg = log_gamma.float().contiguous()
    ws = torch.empty(lib.lz_gla_seg_workspace_bytes(B, Hs, L, F, D), device=fk.device,
                     dtype=torch.uint8)
    summary = torch.empty(lib.lz_gla_seg_summary_floats(B, Hs, F, D), device=fk.device,
                          dtype=torch.float32)
    with _lib.on_device(fk.device):
        rc = lib.lz_gla_seg_fwd_begin(_lib.ptr(fk16), _lib.ptr(v16), _lib.ptr(lg), per_head,
                                      _lib.ptr(summary), _lib.ptr(ws), ws.numel(), B, Hs, L, F,
                                      D, _lib.stream_of(fk))
    _lib.check(rc, "gla state")
    nS, nZ = B * Hs * F * D, B * Hs * F
    return summary[:nS].view(B, Hs, F, D).clone(), summary[nS:nS + nZ].view(B, Hs, F).clone()


def gla_decode(fq, fk, v, log_gamma, state, zstate):
    """One token: fq [B, H, F], fk [B, Hkv, F], v [B, Hkv, D], log_gamma [B] or
    [B, H]; state [B, Hs, F, D] and zstate [B, Hs, F] (fp32, Hs = H or Hkv)
    advance in place. Returns y bf16 [B, H, D]."""
    _lib.require_cuda(fq, fk, v, log_gamma, state, zstate)
    B, H, F = fq.shape
    Hkv, D = fk.shape[1], v.shape[-1]
    Hs = state.shape[1]
    if state.dtype != torch.float32 or not state.is_contiguous() or not zstate.is_contiguous():
        raise ValueError("state and zstate must be contiguous fp32 tensors")
    if tuple(state.shape) != (B, Hs, F, D) or tuple(zstate.shape) != (B, Hs, F):
        raise ValueError(f"state must be [B, Hs, F, D] and zstate [B, Hs, F], got "
                         f"{tuple(state.shape)}, {tuple(zstate.shape)}")
    per_head = 1 if log_gamma.dim() == 2 else 0
    lib = _lib.load()
    fq16, fk16, v16 = (t.to(torch.bfloat16).contiguous() for t in (fq, fk, v))
    lg = log_gamma.float().contiguous()
    y = torch.empty(B, H, D, device=fq.device, dtype=torch.bfloat16)
    rc = lib.lz_gla_decode(_lib.ptr(fq16), _lib.ptr(fk16), _lib.ptr(v16), _lib.ptr(lg),
                           per_head, _lib.ptr(state), _lib.ptr(zstate), _lib.ptr(y), B, H, Hkv,
                           Hs, F, D, _lib.stream_of(fq))
    _lib.check(rc, "gla decode")
    return y


def rotate(x, cos, sin):
    """Llama rotate-half RoPE in fp32, as the reference's caller evaluates it
    (src/lizard_attention.py:87-88): x [B, Hx, L, D], cos / sin [B, L, D]."""
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def swa_ring(k, v, cos, sin, window):
    """Rings after a prompt: rotated keys and values of its last `window`
    tokens (fp32 [B, Hkv, window, D]), token t in slot t % window. k, v
    [B, Hkv, L, D] (k unrotated); cos, sin [B, L, D] or [1, L, D]."""
    B, Hkv, L, D = k.shape
    n = min(L, window)
    t = torch.arange(L - n, L, device=k.device)
    kr = rotate(k[:, :, L - n:], cos[:, L - n:].expand(B, n, D), sin[:, L - n:].expand(B, n, D))
    k_ring = torch.zeros(B, Hkv, window, D, device=k.device, dtype=torch.float32)
    v_ring = torch.zeros_like(k_ring)
    k_ring[:, :, t % window] = kr
    v_ring[:, :, t % window] = v[:, :, L - n:].float()
    return k_ring, v_ring


def swa_decode(q, k, v, cos, sin, meta, k_ring, v_ring, pos):
    """One token: q [B, H, D], k, v [B, Hkv, D] (q, k unrotated; strided views
    with a contiguous last dim are read in place), cos, sin [B, D] or [1, D]
    at the token's position, meta [n_meta], rings fp32 [B, Hkv, W, D] and pos
    int32 [B] (tokens before this one; the caller advances it). The new key
    and value go into slot pos % W. Returns y bf16 [B, H, D]."""
    _lib.require_cuda(q, k, v, cos, sin, k_ring, v_ring, pos)
    B, H, D = q.shape
    Hkv, W = k.shape[1], k_ring.shape[2]
    xdt = q.dtype if q.dtype in _DT else torch.float32
    q, k, v = (t if (t.dtype == xdt and t.stride(-1) == 1) else t.to(xdt).contiguous()
               for t in (q, k, v))
    if cos.dtype != sin.dtype or cos.dtype not in _DT:
        cos, sin = cos.float(), sin.float()
    cos, sin = cos.reshape(-1, D).contiguous(), sin.reshape(-1, D).contiguous()
    cs_sb = D if cos.shape[0] == B and B > 1 else 0
    if tuple(k_ring.shape) != (B, Hkv, W, D) or k_ring.dtype != torch.float32:
        raise ValueError(f"k_ring must be fp32 [B, Hkv, W, D], got {tuple(k_ring.shape)}")
    if pos.dtype != torch.int32 or pos.numel() != B:
        raise ValueError("pos must be int32 [B]")
    meta32 = meta.float().contiguous()
    lib = _lib.load()
    y = torch.empty(B, H, D, device=q.device, dtype=torch.bfloat16)
    rc = lib.lz_swa_decode(_lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _DT[xdt], q.stride(0),
                           q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                           _lib.ptr(cos), _lib.ptr(sin), _DT[cos.dtype], cs_sb,
                           _lib.ptr(k_ring), _lib.ptr(v_ring), _lib.ptr(pos),
                           _lib.ptr(meta32) if meta32.numel() else None, meta32.numel(),
                           _lib.ptr(y), B, H, Hkv, W, D, _lib.stream_of(q))
    _lib.check(rc, "swa decode")
    return y


def _pending_count(count, B, index):
    if count is None:
        return None
    if count.dtype is not torch.int32 or count.shape != (B,) or count.get_device() != index:
        raise ValueError(f"count must be int32 [{B}] on device {index}, got {count.dtype} "
                         f"{tuple(count.shape)} on {count.device}")
    return count.contiguous()


def gla_decode_block(fq, fk, v, log_gamma, state, zstate, pending=None):
    """A block of T <= 64 new tokens against the state, for drafted decoding:
    fq [B, H, T, F], fk [B, Hkv, T, F], v [B, Hkv, T, D], log_gamma [B, T] or
    [B, H, T]; returns y bf16 [B, H, T, D], the outputs T calls of gla_decode
    would give. The block is NOT folded into the state, since its tokens may be
    refused: pass it as `pending` = (fk, v, log_gamma, count) of the next call,
    which first advances state and zstate (fp32 [B, Hs, F, D] and [B, Hs, F], in
    place) by the first count[b] (int32 [B], None = all) of its tokens.
    T = 0 (empty fq, fk, v, log_gamma) only advances the state."""
    index = fq.get_device()
    if not (index == fk.get_device() == v.get_device() == log_gamma.get_device()
            == state.get_device() == zstate.get_device() >= 0):
        _lib.require_cuda(fq, fk, v, log_gamma, state, zstate)
    if fq.dim() != 4 or fk.dim() != 4 or v.dim() != 4 or state.dim() != 4:
        raise ValueError("fq, fk, v must be [B, heads, T, dim] and state [B, Hs, F, D]")
    B, H, T, F = fq.shape
    Hkv, D, Hs = fk.shape[1], v.shape[3], state.shape[1]
    if fk.shape != (B, Hkv, T, F) or v.shape != (B, Hkv, T, D):
        raise ValueError(f"fk and v must be [B, Hkv, T, F] and [B, Hkv, T, D] matching fq "
                         f"{tuple(fq.shape)}, got {tuple(fk.shape)}, {tuple(v.shape)}")
    if (state.dtype is not torch.float32 or zstate.dtype is not torch.float32
            or not state.is_contiguous() or not zstate.is_contiguous()):
        raise ValueError("state and zstate must be contiguous fp32 tensors")
    if state.shape != (B, Hs, F, D) or zstate.shape != (B, Hs, F):
        raise ValueError(f"state must be [B, Hs, F, D] and zstate [B, Hs, F], got "
                         f"{tuple(state.shape)}, {tuple(zstate.shape)}")
    per_head = 1 if log_gamma.dim() == 3 else 0
    if log_gamma.shape != ((B, H, T) if per_head else (B, T)):
        raise ValueError(f"log_gamma must be [B, T] or [B, H, T], got {tuple(log_gamma.shape)}")
    Tp = p_fk = p_v = p_lg = p_count = 0
    if pending is not None:
        fkp, vp, lgp, count = pending
        if not index == fkp.get_device() == vp.get_device() == lgp.get_device():
            _lib.require_cuda(fq, fkp, vp, lgp)
        Tp = fkp.shape[2]
        if fkp.shape != (B, Hkv, Tp, F) or vp.shape != (B, Hkv, Tp, D):
            raise ValueError(f"pending fk and v must be [B, Hkv, T, F] and [B, Hkv, T, D], got "
                             f"{tuple(fkp.shape)}, {tuple(vp.shape)}")
        if lgp.shape != ((B, H, Tp) if per_head else (B, Tp)):
            raise ValueError(f"pending log_gamma must have log_gamma's layout, got "
                             f"{tuple(lgp.shape)}")
        fkp, vp = _lib.as_dtype(fkp, torch.bfloat16), _lib.as_dtype(vp, torch.bfloat16)
        lgp = _lib.as_dtype(lgp, torch.float32)
        p_fk, p_v, p_lg = fkp.data_ptr(), vp.data_ptr(), lgp.data_ptr()
        if count is not None:
            count = _pending_count(count, B, index)
            p_count = count.data_ptr()
    y = fq.new_empty((B, H, T, D), dtype=torch.bfloat16)
    if B == 0 or T == 0 and Tp == 0:
        return y
    fq, fk = _lib.as_dtype(fq, torch.bfloat16), _lib.as_dtype(fk, torch.bfloat16)
    v, lg = _lib.as_dtype(v, torch.bfloat16), _lib.as_dtype(log_gamma, torch.float32)
    rc = _lib.call(index, _lib.CALL_GLA_DECODE_BLOCK, _gla_words(
        fq.data_ptr(), fk.data_ptr(), v.data_ptr(), lg.data_ptr(), per_head, p_fk, p_v, p_lg,
        p_count, state.data_ptr(), zstate.data_ptr(), y.data_ptr(), B, H, Hkv, Hs, T, Tp, F, D,
        _lib.raw_stream(index)))
    if rc:
        _lib.check(rc, "gla decode block")
    return y


def _tables(cos, sin, dtype, B, T, D):
    """cos / sin as contiguous [B or 1, T, D] of dtype, and the batch stride."""
    n = cos.shape[0]
    if cos.shape != (n, T, D) or sin.shape != (n, T, D) or n != B and n != 1:
        for t in (cos, sin):
            if t.dim() != 3 or t.shape[1:] != (T, D) or t.shape[0] not in (1, B):
                raise ValueError(f"cos and sin must be [{B} or 1, {T}, {D}], got {tuple(t.shape)}")
        cos, sin, n = cos.expand(B, T, D), sin.expand(B, T, D), B
    return _lib.as_dtype(cos, dtype), _lib.as_dtype(sin, dtype), T * D if n > 1 else 0


def _common(*tensors):
    """The tensors' type if they share one that the kernels read, else fp32 (which holds
    the values of all of them)."""
    dtype = tensors[0].dtype
    for t in tensors:
        if t.dtype is not dtype:
            return torch.float32
    return dtype if dtype in _DT else torch.float32


def _rows(t, dtype):
    """t in dtype with a contiguous last dimension, in place where it has one."""
    if t.dtype is not dtype:
        t = t.to(dtype)
    return t if t.stride(3) == 1 else t.contiguous()


_gla_words, _swa_words = struct.Struct("21q").pack, struct.Struct("52q").pack


_NO_STRIDES = (0,) * 8


def swa_decode_block(q, k, v, cos, sin, meta, k_ring, v_ring, pos, pending=None):
    """A block of T <= 64 new tokens against the rings, for drafted decoding:
    q [B, H, T, D], k, v [B, Hkv, T, D] (unrotated; strided views with a
    contiguous last dim are read in place), cos, sin [B, T, D] or [1, T, D] at
    the tokens' positions, meta [n_meta], rings fp32 [B, Hkv, W, D], pos int32
    [B]; returns y bf16 [B, H, T, D], the outputs T calls of swa_decode would
    give. The block does not enter the rings: pass it as `pending` = (k, v, cos,
    sin, count) of the next call, which first writes the first count[b] (int32
    [B], None = all) of its tokens to slots (pos[b] + t) % W. pos counts the
    tokens the rings hold before the call, without the pending ones; the caller
    then advances it by count. T = 0 only advances the rings. q, k, v and the
    pending ones are fp32 or bf16, the tables too; where types differ, or are
    others, all are read as fp32."""
    index = q.get_device()
    if not (index == k.get_device() == v.get_device() == cos.get_device() == sin.get_device()
            == meta.get_device() == k_ring.get_device() == v_ring.get_device()
            == pos.get_device() >= 0):
        _lib.require_cuda(q, k, v, cos, sin, meta, k_ring, v_ring, pos)
    if q.dim() != 4 or k.dim() != 4 or k_ring.dim() != 4:
        raise ValueError("q, k, v must be [B, heads, T, D] and the rings [B, Hkv, W, D]")
    B, H, T, D = q.shape
    Hkv, W = k.shape[1], k_ring.shape[2]
    if k.shape != (B, Hkv, T, D) or v.shape != k.shape:
        raise ValueError(f"k and v must be [B, Hkv, T, D] matching q {tuple(q.shape)}, got "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if (k_ring.shape != (B, Hkv, W, D) or v_ring.shape != k_ring.shape
            or k_ring.dtype is not torch.float32 or v_ring.dtype is not torch.float32
            or not k_ring.is_contiguous() or not v_ring.is_contiguous()):
        raise ValueError(f"the rings must be contiguous fp32 [B, Hkv, W, D], got {k_ring.dtype} "
                         f"{tuple(k_ring.shape)}, {v_ring.dtype} {tuple(v_ring.shape)}")
    if pos.dtype is not torch.int32 or pos.shape != (B,):
        raise ValueError("pos must be int32 [B]")
    if pending is None:
        xdt, cdt = _common(q, k, v), _common(cos, sin)
    Tp = cp_sb = p_k = p_v = p_c = p_s = p_count = 0
    strides_p = _NO_STRIDES
    if pending is not None:
        kp, vp, cp, sp, count = pending
        if not (index == kp.get_device() == vp.get_device() == cp.get_device()
                == sp.get_device()):
            _lib.require_cuda(q, kp, vp, cp, sp)
        Tp = kp.shape[2]
        if kp.shape != (B, Hkv, Tp, D) or vp.shape != kp.shape:
            raise ValueError(f"pending k and v must be [B, Hkv, T, D], got {tuple(kp.shape)}, "
                             f"{tuple(vp.shape)}")
        xdt, cdt = _common(q, k, v, kp, vp), _common(cos, sin, cp, sp)
        if Tp:
            cp, sp, cp_sb = _tables(cp, sp, cdt, B, Tp, D)
            kp, vp = _rows(kp, xdt), _rows(vp, xdt)
            strides_p = kp.stride() + vp.stride()
            p_k, p_v, p_c, p_s = kp.data_ptr(), vp.data_ptr(), cp.data_ptr(), sp.data_ptr()
        if count is not None:
            count = _pending_count(count, B, index)
            p_count = count.data_ptr()
    y = q.new_empty((B, H, T, D), dtype=torch.bfloat16)
    if B == 0 or T == 0 and Tp == 0:
        return y
    cos, sin, cs_sb = _tables(cos, sin, cdt, B, T, D)
    q, k, v = _rows(q, xdt), _rows(k, xdt), _rows(v, xdt)
    meta, pos = _lib.as_dtype(meta, torch.float32), pos.contiguous()
    size = _lib.size_query("lz_swa_decode_block_workspace_bytes", B, H, Hkv, T, D)
    ws = pos.new_empty((size + 3) // 4)
    # the strides follow the 32 arguments
    rc = _lib.call(index, _lib.CALL_SWA_DECODE_BLOCK, _swa_words(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _DT[xdt], 32, cos.data_ptr(), sin.data_ptr(),
        _DT[cdt], cs_sb, p_k, p_v, 44 if Tp else 0, p_c, p_s, cp_sb, p_count, k_ring.data_ptr(),
        v_ring.data_ptr(), pos.data_ptr(), meta.data_ptr(), meta.numel(), y.data_ptr(),
        ws.data_ptr(), size, B, H, Hkv, T, Tp, W, D, _lib.raw_stream(index), *q.stride(),
        *k.stride(), *v.stride(), *strides_p))
    if rc:
        _lib.check(rc, "swa decode block")
    return y


@dataclass
class LayerCache:
    """Decode state of one Lizard layer."""
    state: torch.Tensor   # fp32 [B, Hs, F, D]
    zstate: torch.Tensor  # fp32 [B, Hs, F]
    k_ring: torch.Tensor  # fp32 [B, Hkv, W, D], rotated keys
    v_ring: torch.Tensor  # fp32 [B, Hkv, W, D]
    pos: torch.Tensor     # int32 [B], tokens seen
    # the last block of drafted decoding, not folded in yet: (fk, v, log_gamma) of the
    # GLA branch and (k, v, cos, sin) of the SWA branch
    pending: tuple = None

    def _stand(self, accepted):
        """How many tokens of the pending block stand: accepted as the kernels clamp it."""
        if accepted is None:
            raise ValueError("a block is pending: accepted (int32 [B]) says how much of it "
                             "stands")
        return accepted.clamp(0, self.pending[0][0].shape[2])

    def block(self, fq, fk, v, log_gamma, q, k, cos, sin, meta, accepted):
        """Both branches' outputs for a block of new tokens, after the first
        accepted[b] tokens (int32 [B]) of the block before have been folded in; the
        block becomes the pending one. After an error the same call may be repeated:
        the ring's step comes first (once more, it writes the same slots), the
        state's, which must not happen twice, last."""
        gla_p = swa_p = None
        if self.pending is not None:
            stand = self._stand(accepted)
            gla_p, swa_p = ((*p, accepted) for p in self.pending)
        v16 = _lib.as_dtype(v, torch.bfloat16)
        y_swa = swa_decode_block(q, k, v, cos, sin, meta, self.k_ring, self.v_ring, self.pos,
                                 swa_p)
        y_gla = gla_decode_block(fq, fk, v16, log_gamma, self.state, self.zstate, gla_p)
        if self.pending is not None:
            self.pos += stand
        self.pending = (fk, v16, log_gamma), (k, v, cos, sin)
        return y_gla, y_swa

    def settle(self, accepted):
        """Fold the first accepted[b] tokens of the pending block in and forget the rest.
        May be repeated after an error, as block."""
        if self.pending is None:
            return
        stand = self._stand(accepted)
        (fk, v, lg), (k, v_, cos, sin) = self.pending
        H = lg.shape[1] if lg.dim() == 3 else fk.shape[1]
        fq, q = fk.new_empty(fk.shape[0], H, 0, fk.shape[3]), k[:, :, :0]
        swa_decode_block(q, q, v_[:, :, :0], cos[:, :0], sin[:, :0], cos.new_empty(0),
                         self.k_ring, self.v_ring, self.pos, (k, v_, cos, sin, accepted))
        gla_decode_block(fq, fk[:, :, :0], v[:, :, :0], lg[..., :0], self.state, self.zstate,
                         (fk, v, lg, accepted))
        self.pos += stand
        self.pending = None


class LizardCache(dict):
    """layer_idx -> LayerCache. Pass as `lizard_cache=` to a model whose
    attention layers are lizard_cuda LizardAttention: the first call with a
    layer's index missing runs the full forward over the prompt and stores the
    layer's state; later calls decode their tokens one at a time. Position ids
    of the new tokens must be given to the model (position_ids=).

    Drafted decoding: after draft(accepted) a call takes its tokens (up to 64) as
    one block that can be taken back. It first folds in the first accepted[b]
    tokens (int32 [B]) of the block before, and leaves its own to the next call,
    which needs a draft(accepted) of its own; settle(accepted) folds them in and
    returns to token-by-token decoding."""

    drafting = False
    accepted = None
    taken = frozenset()  # the layers that have run their block since draft()

    def draft(self, accepted=None):
        """The next call's tokens are a block; accepted tokens of the block before (all
        rows 0 when there is none to keep)."""
        self.drafting, self.accepted, self.taken = True, accepted, frozenset()
        return self

    def block_counts(self, layer_idx):
        """What draft was told, for a layer about to run its block."""
        if layer_idx in self.taken:
            raise RuntimeError(f"layer {layer_idx} has run its block since draft(accepted): the "
                               "next block needs a draft call that says how much of it stands")
        return self.accepted

    def settle(self, accepted):
        for layer in self.values():
            layer.settle(accepted)
        self.drafting, self.accepted, self.taken = False, None, frozenset()
