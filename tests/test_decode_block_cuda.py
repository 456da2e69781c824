"""Blocks of drafted tokens against the cached state (gla_decode_block,
swa_decode_block): a 64-bit token-by-token restatement at the sizes and masks
where they can go wrong, the single-token steps, and the refusals.

Tolerances, from the kernels' arithmetic:
  y     has to be the bf16 rounding of a number near the reference: operands split
        into bf16 hi + lo (2^-17 each) and fp32 sums, relative to the sums of
        magnitudes (the rounding itself is monotonic and takes no tolerance);
  state 2 roundings a token plus the decay's, relative to the undecayed
        magnitudes: (3 n + 8) 2^-24;
  rings bit for bit (each product and sum rounded once in both).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


def _rounds_to(y, ref, e):
    """y (bf16) lies between the bf16 roundings of ref - e and ref + e."""
    e = e + 2.0 ** -23 * ref.abs()  # 64 -> 32 bits on the way to bf16
    return ((y >= (ref - e).float().bfloat16()) & (y <= (ref + e).float().bfloat16())).all()


# ---------------------------------------------------------------- GLA

def _gla_inputs(B, H, Hkv, F, D, T, Tp, per_head, seed, gates=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    sp = torch.nn.functional.softplus
    Hs = H if per_head else Hkv

    def block(n):
        lg = torch.nn.functional.logsigmoid(
            gates + 1.5 * torch.randn(*((B, H, n) if per_head else (B, n)), generator=g, device=DEV))
        return ((sp(torch.randn(B, Hkv, n, F, generator=g, device=DEV)) / F ** 0.5).bfloat16(),
                torch.randn(B, Hkv, n, D, generator=g, device=DEV).bfloat16(), lg)

    fq = (sp(torch.randn(B, H, T, F, generator=g, device=DEV)) / F ** 0.5).bfloat16()
    z = 5 * torch.rand(B, Hs, F, generator=g, device=DEV)
    S = torch.randn(B, Hs, F, D, generator=g, device=DEV) * z[..., None]
    count = torch.randint(0, Tp + 1, (B,), generator=g, device=DEV).int()
    return fq, block(T), block(Tp), count, S, z


def _gla_walk(S, z, fk, v, lg, fq, count=None):
    """64-bit steps; returns y, |y| magnitudes, S, z and the undecayed magnitude of S."""
    Hs, Hkv = S.shape[1], fk.shape[1]
    mag, zmag, ys, yabs = S.abs(), z.abs(), [], []
    Sa = S.abs()
    for t in range(fk.shape[2]):
        k, x = (u[:, :, t].double().repeat_interleave(Hs // Hkv, 1) for u in (fk, v))
        g = torch.exp(lg[..., t].double()).reshape(S.shape[0], -1, 1)
        live = torch.ones(S.shape[0], dtype=torch.bool, device=S.device) if count is None \
            else t < count
        kv = k[..., None] * x[..., None, :]
        m4, m3 = live[:, None, None, None], live[:, None, None]
        S = torch.where(m4, g[..., None] * S + kv, S)
        Sa = torch.where(m4, g[..., None] * Sa + kv.abs(), Sa)
        z = torch.where(m3, g * z + k, z)
        mag = torch.where(m4, mag + kv.abs(), mag)
        zmag = torch.where(m3, zmag + k, zmag)
        if fq is not None:
            q = fq[:, :, t].double()
            rep = q.shape[1] // Hs
            Sq, Sqa, zq = (u.repeat_interleave(rep, 1) for u in (S, Sa, z))
            den = (q * zq).sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
            ys.append((q[..., None] * Sq).sum(-2) / den)
            yabs.append((q[..., None] * Sqa).sum(-2) / den)
    st = (lambda u: torch.stack(u, 2)) if ys else (lambda u: None)
    return st(ys), st(yabs), S, z, mag, zmag


def _check_gla(y, S, z, ref, n):
    ry, ra, rS, rz, mag, zmag = ref
    tol = (3 * n + 8) * 2.0 ** -24
    assert ((S.double() - rS).abs() <= tol * mag).all()
    assert ((z.double() - rz).abs() <= tol * zmag).all()
    if ry is not None:
        assert _rounds_to(y, ry, 2.0 ** -14 * ra)


@pytest.mark.parametrize("B,H,Hkv,F,D,T,Tp,per_head", [
    (2, 8, 2, 256, 64, 5, 5, False),     # the model's sizes, grouped queries
    (1, 1, 1, 1, 4, 1, 1, False),        # the smallest
    (3, 6, 3, 93, 84, 13, 7, True),      # odd features, per-head gates over grouped keys
    (2, 4, 4, 64, 32, 17, 3, False),     # one 32-column slice, rows past a 16-row tile
    (1, 4, 1, 200, 256, 64, 64, False),  # the longest blocks, four column slices
    (2, 3, 3, 130, 36, 9, 1, True),      # a second slice of four columns
    (2, 16, 1, 128, 128, 4, 2, False),   # 16 query heads on a state
    (5, 5, 5, 17, 68, 1, 64, False),     # one token after a long block
])
def test_gla_block_matches_single_steps_in_64_bits(B, H, Hkv, F, D, T, Tp, per_head):
    from lizard_cuda.decode import gla_decode_block
    fq, (fk, v, lg), (fkp, vp, lgp), count, S, z = _gla_inputs(B, H, Hkv, F, D, T, Tp, per_head,
                                                                T * 100 + F)
    adv = _gla_walk(S.double(), z.double(), fkp, vp, lgp, None, count)
    ref = _gla_walk(adv[2], adv[3], fk, v, lg, fq)
    y = gla_decode_block(fq, fk, v, lg, S, z, pending=(fkp, vp, lgp, count))
    _check_gla(y, S, z, (ref[0], ref[1]) + adv[2:], Tp)


def test_gla_block_without_pending_leaves_the_state():
    from lizard_cuda.decode import gla_decode_block
    fq, (fk, v, lg), _, _, S, z = _gla_inputs(2, 4, 2, 64, 64, 6, 1, False, 1)
    S0, z0 = S.clone(), z.clone()
    y = gla_decode_block(fq, fk, v, lg, S, z)
    assert torch.equal(S, S0) and torch.equal(z, z0)
    ref = _gla_walk(S.double(), z.double(), fk, v, lg, fq)
    _check_gla(y, S0, z0, (ref[0], ref[1], S.double(), z.double(), S.abs(), z.abs()), 0)
    # an empty prefix accepted is the same call
    y2 = gla_decode_block(fq, fk, v, lg, S, z,
                          pending=(fk, v, lg, torch.zeros(2, dtype=torch.int32, device=DEV)))
    assert torch.equal(y, y2) and torch.equal(S, S0) and torch.equal(z, z0)


def test_gla_block_without_tokens_only_advances():
    from lizard_cuda.decode import gla_decode_block
    fq, (fk, v, lg), pend, count, S, z = _gla_inputs(3, 4, 2, 70, 40, 0, 9, False, 2)
    ref = _gla_walk(S.double(), z.double(), *pend, None, None)
    y = gla_decode_block(fq, fk, v, lg, S, z, pending=(*pend, None))
    assert y.shape == (3, 4, 0, 40)
    _check_gla(None, S, z, (None, None) + ref[2:], 9)


def test_gla_block_with_closed_gates_and_an_empty_state():
    """lg = -inf forgets everything before the token (no inf - inf), also twice in a row."""
    from lizard_cuda.decode import gla_decode_block
    fq, (fk, v, lg), (fkp, vp, lgp), _, S, z = _gla_inputs(2, 4, 2, 64, 64, 6, 5, False, 3)
    lg[0, 2] = lg[0, 3] = lg[1, 0] = -math.inf
    lgp[0, 1] = lgp[1, 3] = lgp[1, 4] = -math.inf
    count = torch.tensor([5, 5], dtype=torch.int32, device=DEV)
    S.zero_(), z.zero_()
    adv = _gla_walk(S.double(), z.double(), fkp, vp, lgp, None, count)
    ref = _gla_walk(adv[2], adv[3], fk, v, lg, fq)
    y = gla_decode_block(fq, fk, v, lg, S, z, pending=(fkp, vp, lgp, count))
    assert torch.isfinite(y).all()
    _check_gla(y, S, z, (ref[0], ref[1]) + adv[2:], 5)
    # an all-zero key against an empty state: the clamped row sum, as the single step
    S.zero_(), z.zero_()
    y = gla_decode_block(fq, torch.zeros_like(fk), v, lg, S, z)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("F,D,T,per_head", [(256, 64, 5, False), (93, 84, 13, True),
                                            (32, 32, 40, False)])
def test_gla_block_tokens_that_are_not_numbers(F, D, T, per_head, bad):
    """A token with such a key or value leaves the tokens before it alone; pending ones
    that do not stand leave no trace."""
    from lizard_cuda.decode import gla_decode_block
    fq, (fk, v, lg), (fkp, vp, lgp), count, S, z = _gla_inputs(3, 6, 3, F, D, T, 4, per_head, F)
    count.fill_(2)
    fkp[:, :, 2], vp[:, :, 3], lgp[..., 2] = bad, bad, math.nan
    t = T // 2
    fk[0, :, t, F // 3] = bad
    v[1, :, t, :] = bad
    v[2, 1, T - 1, 7] = bad
    adv = _gla_walk(S.double(), z.double(), fkp, vp, lgp.nan_to_num(0), None, count)
    ref = _gla_walk(adv[2], adv[3], fk, v, lg, fq)
    y = gla_decode_block(fq, fk, v, lg, S, z, pending=(fkp, vp, lgp, count))
    # (the walk's magnitudes of the state count every pending token)
    assert S.isfinite().all() and z.isfinite().all()
    want = ref[0].isfinite()
    assert want[0, :, :t].all() and not want[0, :, t:].any() and not want[1, :, t:].any()
    assert torch.equal(want, y.isfinite())
    assert _rounds_to(y.masked_fill(~want, 0), ref[0].masked_fill(~want, 0),
                      2.0 ** -14 * ref[1].masked_fill(~want, 0))


def test_gla_block_agrees_with_gla_decode_and_repeats():
    from lizard_cuda.decode import gla_decode, gla_decode_block
    fq, (fk, v, lg), pend, count, S, z = _gla_inputs(2, 8, 2, 256, 64, 8, 8, False, 4)
    S1, z1 = S.clone(), z.clone()
    y = gla_decode_block(fq, fk, v, lg, S, z, pending=(*pend, None))
    for t in range(8):
        gla_decode(fq[:, :, t], pend[0][:, :, t], pend[1][:, :, t], pend[2][:, t], S1, z1)
    torch.testing.assert_close(S, S1, rtol=0, atol=float(S1.abs().max()) * 32 * 2.0 ** -24)
    steps = torch.stack([gla_decode(fq[:, :, t], fk[:, :, t], v[:, :, t], lg[:, t], S1, z1)
                         for t in range(8)], 2)
    assert (y.float() - steps.float()).abs().max() <= 2.0 ** -7 * steps.float().abs().max()
    S2, z2 = S.clone(), z.clone()
    again = [gla_decode_block(fq, fk, v, lg, S2, z2) for _ in range(2)]
    assert torch.equal(again[0], again[1])  # no order of threads in the sums


# ---------------------------------------------------------------- SWA

def _rot32(x, cos, sin):
    x, c, s = x.float(), cos.float()[:, None], sin.float()[:, None]
    half = x.shape[-1] // 2
    return x * c + torch.cat([-x[..., half:], x[..., :half]], -1) * s


def _tables(pos, T, D, dtype=torch.float32):
    inv = 5e5 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    a = (pos[:, None] + torch.arange(T, device=DEV))[..., None].double() * inv
    a = torch.cat([a, a], -1)
    return a.cos().to(dtype), a.sin().to(dtype)


def _swa_inputs(B, H, Hkv, W, D, T, Tp, dtype, pos, n_meta=4, seed=0, tables=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def heads(n, t):
        # as projections lie: [B, t, n * D] seen as heads, read in place
        return torch.randn(B, t, n * D, generator=g, device=DEV).to(dtype).view(B, t, n, D) \
            .transpose(1, 2)

    count = torch.randint(0, Tp + 1, (B,), generator=g, device=DEV).int()
    pos = torch.tensor(pos, dtype=torch.int32, device=DEV)
    # slots that hold no token yet must not be read: NaN there
    kr, vr = (torch.randn(B, Hkv, W, D, generator=g, device=DEV) for _ in range(2))
    empty = (torch.arange(W, device=DEV) >= pos[:, None])[:, None, :, None]
    kr, vr = kr.masked_fill(empty, math.nan), vr.masked_fill(empty, math.nan)
    blk = (heads(Hkv, T), heads(Hkv, T)) + _tables(pos + count, T, D, tables)
    pend = (heads(Hkv, Tp), heads(Hkv, Tp)) + _tables(pos, Tp, D, tables) + (count,)
    return heads(H, T), blk, pend, torch.randn(n_meta, generator=g, device=DEV), kr, vr, pos


def _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr):
    """64-bit reference: write the accepted tokens, then attend token by token. Where a
    value that the token sees is not a number, the output is not one either."""
    k, v, cos, sin = blk
    kp, vp, cp, sp, count = pend
    B, H, T, D = q.shape
    Hkv, W = kr0.shape[1:3]
    krp, kb, qb = _rot32(kp, cp, sp), _rot32(k, cos, sin).double(), _rot32(q, cos, sin).double()
    want_k, want_v = kr0.clone(), vr0.clone()
    for b in range(B):
        for t in range(int(count[b])):
            want_k[b, :, (int(pos[b]) + t) % W] = krp[b, :, t]
            want_v[b, :, (int(pos[b]) + t) % W] = vp[b, :, t].float()
    assert torch.equal(kr.nan_to_num(7), want_k.nan_to_num(7))
    assert torch.equal(vr.nan_to_num(7), want_v.nan_to_num(7))
    for b in range(B):
        base = int(pos[b]) + int(count[b])
        kk, vv = want_k[b].double(), want_v[b].double()
        for t in range(T):
            slot = (base + t) % W
            kk[:, slot], vv[:, slot] = kb[b, :, t], v[b, :, t].double()
            n = min(base + t + 1, W)
            keys, vals = (u[:, :n].repeat_interleave(H // Hkv, 0) for u in (kk, vv))
            x = torch.einsum("hnd,hd->hn", keys, qb[b, :, t]) / D ** 0.5
            mag = torch.einsum("hnd,hd->hn", keys.abs(), qb[b, :, t].abs()).amax(-1) / D ** 0.5
            p = torch.softmax(torch.cat([x, meta.double().expand(H, -1)], -1), -1)[:, :n]
            ref = torch.einsum("hn,hnd->hd", p, vals)
            assert torch.equal(ref.isfinite(), y[b, :, t].isfinite()), (b, t)
            ref, got = ref.nan_to_num(0, 0, 0), y[b, :, t].nan_to_num(0, 0, 0)
            top = vals.nan_to_num(0, 0, 0).abs().amax((1, 2))
            # split products miss 3 2^-18 of the score's magnitude, twice in a quotient
            tol = (top * (mag * 6 * 2.0 ** -18 + 2.0 ** -14))[:, None]
            assert _rounds_to(got, ref, tol), (b, t)


@pytest.mark.parametrize("B,H,Hkv,W,D,T,Tp,dtype,pos", [
    (3, 8, 2, 64, 64, 5, 5, torch.bfloat16, [200, 0, 61]),   # wrapped, empty, about to fill
    (2, 1, 1, 1, 2, 1, 1, torch.float32, [0, 3]),            # the smallest window and head
    (2, 6, 2, 37, 96, 11, 7, torch.float32, [30, 1000]),
    (2, 4, 4, 128, 64, 8, 8, torch.bfloat16, [128, 90]),
    (2, 4, 1, 5, 32, 13, 9, torch.float32, [2, 12]),         # blocks longer than the window
    (1, 2, 1, 130, 256, 3, 4, torch.bfloat16, [400]),        # the widest head
    (1, 8, 2, 1024, 64, 3, 2, torch.bfloat16, [5000]),       # the largest window
    (1, 4, 1, 64, 62, 64, 64, torch.float32, [77]),          # the longest blocks, D % 4 != 0
    (1, 16, 1, 40, 64, 1, 1, torch.bfloat16, [39]),
])
def test_swa_block_matches_single_steps_in_64_bits(B, H, Hkv, W, D, T, Tp, dtype, pos):
    from lizard_cuda.decode import swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(B, H, Hkv, W, D, T, Tp, dtype, pos, seed=W + T)
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos, pending=pend)
    assert torch.isfinite(y).all()
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("W,T,D", [(64, 5, 64), (8, 11, 32), (37, 20, 62)])
def test_swa_block_masked_values_that_are_not_numbers(W, T, D, bad):
    """Values at masked places: of later tokens of the block, and of ring tokens that have
    left the window of all or of some of the block's tokens."""
    from lizard_cuda.decode import swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(4, 4, 2, W, D, T, 2, torch.bfloat16,
                                                  [3 * W, 3 * W, W + 5, 2], seed=W)
    pend[4].zero_()
    blk[1][0, :, T - 1, 3] = bad               # the last token of the block
    blk[1][3, 1, T // 2] = bad
    vr[1, :, 0] = bad                          # the oldest: no token of the block sees it
    vr[2, 1, (5 + 2) % W, 5:9] = bad           # seen by the first two
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos, pending=pend)
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)


def test_swa_block_without_sinks_pending_or_own_tables():
    from lizard_cuda.decode import swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(2, 4, 2, 16, 64, 4, 1, torch.bfloat16, [9, 9],
                                                  n_meta=0, seed=5, tables=torch.bfloat16)
    pend[4].zero_()
    blk = blk[:2] + _tables(pos[:1], 4, 64, torch.bfloat16)  # one table for both rows
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos)
    full = blk[:2] + tuple(t.expand(2, 4, 64) for t in blk[2:])
    _check_swa(y, q, full, pend, meta, kr0, vr0, pos, kr, vr)
    # T = 0 writes the accepted tokens and nothing else
    e = q[:, :, :0]
    y0 = swa_decode_block(e, e[:, :2], e[:, :2], blk[2][:, :0], blk[3][:, :0], meta, kr, vr, pos,
                          pending=blk[:2] + full[2:] + (None,))
    assert y0.shape == (2, 4, 0, 64)
    slots = torch.arange(9, 13, device=DEV) % 16
    assert torch.equal(kr[:, :, slots], _rot32(blk[0], *full[2:]))
    assert torch.equal(vr[:, :, slots], blk[1].float())


def test_swa_block_agrees_with_swa_decode():
    from lizard_cuda.decode import swa_decode, swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(2, 8, 2, 64, 64, 6, 1, torch.bfloat16, [70, 64],
                                                  seed=6)
    pend[4].zero_()
    blk = blk[:2] + _tables(pos, 6, 64)
    y = swa_decode_block(q, *blk, meta, kr, vr, pos)
    p, steps = pos.clone(), []
    for t in range(6):
        steps.append(swa_decode(q[:, :, t], blk[0][:, :, t], blk[1][:, :, t], blk[2][:, t],
                                blk[3][:, t], meta, kr, vr, p))
        p += 1
    steps = torch.stack(steps, 2).float()
    assert (y.float() - steps).abs().max() <= 2.0 ** -7 * steps.abs().max()


# ---------------------------------------------------------------- refusals

def test_block_refusals():
    from lizard_cuda.decode import gla_decode_block, swa_decode_block
    fq, (fk, v, lg), pend, count, S, z = _gla_inputs(2, 4, 2, 64, 64, 3, 2, False, 7)
    with pytest.raises(ValueError, match="contiguous fp32"):
        gla_decode_block(fq, fk, v, lg, S.bfloat16(), z)
    with pytest.raises(ValueError, match="matching fq"):
        gla_decode_block(fq, fk[:, :, :2], v, lg, S, z)
    with pytest.raises(ValueError, match="log_gamma"):
        gla_decode_block(fq, fk, v, lg[:, :2], S, z)
    with pytest.raises(ValueError, match="count must be int32"):
        gla_decode_block(fq, fk, v, lg, S, z, pending=(*pend, count.long()))
    with pytest.raises(ValueError, match="pending"):
        gla_decode_block(fq, fk, v, lg, S, z, pending=(fk, v, pend[2], count))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gla_decode_block(fq.cpu(), fk, v, lg, S, z)
    big = [t.repeat_interleave(22, 2) for t in (fq, fk, v)]
    with pytest.raises(RuntimeError, match="at most 64"):
        gla_decode_block(*big, lg.repeat_interleave(22, 1), S, z)
    # state heads: a per-head gate needs a state per query head
    with pytest.raises(RuntimeError, match="state heads"):
        gla_decode_block(fq, fk, v, lg[:, None].expand(2, 4, 3), S, z)
    q, blk, spend, meta, kr, vr, pos = _swa_inputs(2, 4, 2, 16, 64, 3, 2, torch.bfloat16, [9, 9])
    with pytest.raises(ValueError, match="pos must be int32"):
        swa_decode_block(q, *blk, meta, kr, vr, pos.long())
    with pytest.raises(ValueError, match="rings"):
        swa_decode_block(q, *blk, meta, kr.bfloat16(), vr, pos)
    with pytest.raises(ValueError, match="rings"):
        swa_decode_block(q, *blk, meta, kr, vr[:, :, :8], pos)
    with pytest.raises(ValueError, match="cos and sin"):
        swa_decode_block(q, *blk[:2], blk[2][:, :2], blk[3], meta, kr, vr, pos)
    with pytest.raises(ValueError, match="pending k and v"):
        swa_decode_block(q, *blk, meta, kr, vr, pos, pending=(spend[0][..., :32],) + spend[1:])
    with pytest.raises(RuntimeError, match="n_meta"):
        swa_decode_block(q, *blk, torch.zeros(33, device=DEV), kr, vr, pos)
