"""The operators of drafted (speculative) decoding with a Lizard model, as measured cases.

  int8_linear       y = x W^T in 8-bit integers, one scale a token and one a channel
  verify_drafts     accepts drafted tokens against the target's probabilities and
                    draws the token that follows, from given random numbers
  gla_decode_block  a block of new tokens through the gated linear attention state
  swa_decode_block  a block of new tokens through the sliding-window ring

Sizes are those of the repository's full model (hidden 2048, 32 query heads and 8
key / value heads of 64, 256 features, MLP 8192, vocabulary 128256, window 64 or
128), with odd ones between them.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "lizard-reproduction_b200")
DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4}


def _api():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import lizard_cuda
    import lizard_cuda.decode
    return lizard_cuda


# ---------------------------------------------------------------------------- cases

def listed():
    return [
        # one new token through a q / o projection: latency, and 4 MB of weight codes
        dict(name="int8_token", op="int8", m=1, k=2048, n=2048, dtype="bf16", bias=False),
        # the language model head for a batch of 32 new tokens: 263 MB of weight codes
        dict(name="int8_head", op="int8", m=32, k=2048, n=128256, dtype="bf16", bias=False),
        # a short prompt through odd sizes, fp32 activations and outputs, with a bias
        dict(name="int8_odd", op="int8", m=333, k=1000, n=777, dtype="fp32", bias=True),
        # prefill of 8 prompts of 4096 tokens through the MLP's down projection
        dict(name="int8_prefill", op="int8", m=32768, k=8192, n=2048, dtype="bf16", bias=False),
        # one sequence, four drafted tokens: latency over nine rows of the vocabulary
        dict(name="verify_one", op="verify", b=1, k=4, v=128256, dtype="bf16", temp="one",
             ragged=False, masked=False),
        # small odd vocabulary, fp32 logits with tokens masked out, drafts of every
        # length from none, a temperature for each sequence (0, greedy, among them)
        dict(name="verify_odd", op="verify", b=37, k=5, v=32003, dtype="fp32", temp="mixed",
             ragged=True, masked=True),
        # a serving batch, seven drafted tokens each
        dict(name="verify_batch", op="verify", b=64, k=7, v=128256, dtype="bf16", temp="one",
             ragged=False, masked=False),
        # one sequence, a block of five tokens: latency
        dict(name="gla_one", op="gla", b=1, h=32, hkv=8, t=5, f=256, d=64, per_head=False),
        # a gate for each head, odd feature and value sizes, a longer block
        dict(name="gla_odd", op="gla", b=3, h=6, hkv=3, t=13, f=93, d=84, per_head=True),
        # a large serving batch: 134 MB of states
        dict(name="gla_batch", op="gla", b=256, h=32, hkv=8, t=8, f=256, d=64, per_head=False),
        # one sequence, a block of five tokens, window 64: latency
        dict(name="swa_one", op="swa", b=1, h=32, hkv=8, t=5, w=64, d=64, n_meta=4,
             dtype="bf16", young=False),
        # a serving batch at the training window of 128, some sequences shorter than it
        dict(name="swa_batch", op="swa", b=128, h=32, hkv=8, t=8, w=128, d=64, n_meta=4,
             dtype="bf16", young=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    op = rng.choice(["int8", "verify", "gla", "swa"])
    if op == "int8":
        return dict(op=op, m=_log_int(rng, 1, 32768), k=_log_int(rng, 64, 8192),
                    n=_log_int(rng, 64, 128256), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    bias=rng.random() < 0.5)
    if op == "verify":
        return dict(op=op, b=_log_int(rng, 1, 64), k=rng.randint(1, 7),
                    v=_log_int(rng, 1000, 128256), dtype=rng.choice(["bf16", "bf16", "fp32"]),
                    temp=rng.choice(["one", "mixed"]), ragged=rng.random() < 0.5,
                    masked=rng.random() < 0.5)
    hkv = rng.choice([1, 2, 3, 4, 8])
    h = hkv * rng.choice([1, 2, 4])
    if op == "gla":
        return dict(op=op, b=_log_int(rng, 1, 256), h=h, hkv=hkv, t=rng.randint(1, 16),
                    f=rng.choice([rng.randint(16, 256), 128, 256]),
                    d=rng.choice([4 * rng.randint(8, 32), 64, 128]), per_head=rng.random() < 0.3)
    return dict(op=op, b=_log_int(rng, 1, 128), h=h, hkv=hkv, t=rng.randint(1, 16),
                w=rng.choice([rng.randint(16, 128), 64, 128]), d=rng.choice([32, 64, 96, 128]),
                n_meta=rng.choice([0, 4]), dtype=rng.choice(["bf16", "fp32"]),
                young=rng.random() < 0.5)


def draw(rng):
    case = _drawn(rng)
    rows = "m" if case["op"] == "int8" else "b"
    top = [work(c) for c in listed() if c["op"] == case["op"]]
    # no more work than the largest listed case of the operator
    while case[rows] > 1 and any(work(case)[n] > max(w[n] for w in top) for n in top[0]):
        case[rows] = case[rows] * 3 // 4
    return case


# --------------------------------------------------------------------------- inputs

def _int8_inputs(c, g):
    m, k, n = c["m"], c["k"], c["n"]
    dt = _DT[c["dtype"]]
    # activations: normal, with a few channels an order larger, as after a norm
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= 1 + 12 * (torch.rand(k, generator=g, device=DEV) < 0.01)
    # rows of codes start on 16-byte boundaries, as a weight is laid out once
    codes = torch.zeros(n, -(-k // 16) * 16, device=DEV, dtype=torch.int8)[:, :k]
    for i in range(0, n, 16384):  # weights as codes: a normal row against its largest entry
        part = torch.randn(min(16384, n - i), k, generator=g, device=DEV) * (127 / 4.2)
        codes[i:i + 16384] = part.round().clamp(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand(n, generator=g, device=DEV)) * (4.2 / 127 / k ** 0.5)
    bias = torch.randn(n, generator=g, device=DEV).to(dt) if c["bias"] else None
    return dict(x=x.to(dt), w=codes, ws=scale, bias=bias)


def _verify_inputs(c, g):
    b, k, v = c["b"], c["k"], c["v"]
    dt = _DT[c["dtype"]]
    # a draft that agrees with the target in part: the same logits and its own error
    target = 2.5 * torch.randn(b, k + 1, v, generator=g, device=DEV)
    draft = target[:, :k] + 0.8 * torch.randn(b, k, v, generator=g, device=DEV)
    if c["masked"]:  # tokens that a grammar forbids, in both
        off = torch.rand(b, 1, v, generator=g, device=DEV) < 0.3
        target.masked_fill_(off, -math.inf)
        draft.masked_fill_(off, -math.inf)
    target, draft = target.to(dt), draft.to(dt)
    temp = 1.0
    if c["temp"] == "mixed":
        choice = torch.tensor([0.0, 0.6, 1.0, 1.3], device=DEV)
        temp = choice[torch.randint(0, 4, (b,), generator=g, device=DEV)]
    t = temp[:, None, None] if c["temp"] == "mixed" else 1.0
    # the drafter's own draw from its probabilities
    race = -torch.log(torch.rand(b, k, v, generator=g, device=DEV).clamp_min(1e-12))
    q = torch.exp(draft.float() - draft.float().amax(-1, keepdim=True))
    q = q ** (1 / torch.clamp(t, min=1e-3)) if c["temp"] == "mixed" else q
    tokens = (q / race).argmax(-1)
    del q, race
    # 24-bit uniforms in [0, 1) and exponentials
    u = torch.rand(b, k, generator=g, device=DEV)
    noise = -torch.log1p(-torch.rand(b, v, generator=g, device=DEV)).clamp_max(-1e-8)
    lengths = None
    if c["ragged"]:
        lengths = torch.randint(0, k + 1, (b,), generator=g, device=DEV).int()
    return dict(target=target, draft=draft, tokens=tokens, u=u, noise=noise, temp=temp,
                lengths=lengths)


def _gla_inputs(c, g):
    b, h, hkv, t, f, d = (c[n] for n in ("b", "h", "hkv", "t", "f", "d"))
    hs = h if c["per_head"] else hkv
    gate = (b, h, t) if c["per_head"] else (b, t)

    def feat(heads):
        x = torch.randn(b, heads, t, f, generator=g, device=DEV)
        return (torch.nn.functional.softplus(x) / f ** 0.5).bfloat16()

    def gates():
        return torch.nn.functional.logsigmoid(
            3 + 1.5 * torch.randn(gate, generator=g, device=DEV))

    def value():
        return torch.randn(b, hkv, t, d, generator=g, device=DEV).bfloat16()

    # a state as some ten tokens of memory leave it
    z = feat(hs)[:, :, 0].float() * 10
    s = torch.randn(b, hs, f, d, generator=g, device=DEV) * z[..., None] / 3
    count = torch.randint(0, t + 1, (b,), generator=g, device=DEV).int()
    return dict(fq=feat(h), fk=feat(hkv), v=value(), lg=gates(), state=s, zstate=z.clone(),
                pend=(feat(hkv), value(), gates(), count))


def _rotary(pos, d):
    inv = 5e5 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    a = pos[..., None].double() * inv
    a = torch.cat([a, a], -1)
    return a.cos().float(), a.sin().float()


def _swa_inputs(c, g):
    b, h, hkv, t, w, d = (c[n] for n in ("b", "h", "hkv", "t", "w", "d"))
    dt = _DT[c["dtype"]]

    def normal(heads):
        return torch.randn(b, heads, t, d, generator=g, device=DEV).to(dt)

    count = torch.randint(0, t + 1, (b,), generator=g, device=DEV).int()
    pos = torch.randint(0 if c["young"] else 4 * w, 8 * w, (b,), generator=g, device=DEV).int()
    if c["young"]:  # a part of the sequences does not fill the window yet
        pos = torch.where(torch.rand(b, generator=g, device=DEV) < 0.3, pos % w, pos)
    step = torch.arange(t, device=DEV)
    cos_p, sin_p = _rotary(pos[:, None] + step, d)
    cos, sin = _rotary((pos + count)[:, None] + step, d)
    return dict(q=normal(h), k=normal(hkv), v=normal(hkv), cos=cos, sin=sin,
                meta=torch.randn(c["n_meta"], generator=g, device=DEV),
                k_ring=torch.randn(b, hkv, w, d, generator=g, device=DEV),
                v_ring=torch.randn(b, hkv, w, d, generator=g, device=DEV), pos=pos,
                pend=(normal(hkv), normal(hkv), cos_p, sin_p, count))


_INPUTS = dict(int8=_int8_inputs, verify=_verify_inputs, gla=_gla_inputs, swa=_swa_inputs)


def _inputs(case, seed):
    return _INPUTS[case["op"]](case, torch.Generator(device=DEV).manual_seed(seed))


def prepare(case, seed):
    return dict(op=case["op"], **_inputs(case, seed))


# ---------------------------------------------------------------------- plain forms

def _int8_plain(s):
    x = s["x"].float()
    top = x.abs().amax(-1, keepdim=True)
    n = torch.full_like(top, 127)  # a true division, which number / tensor is not
    codes = torch.round(x * (n / top))
    y = codes @ s["w"].float().t()
    y = y * (top / n * s["ws"])
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _softmax(x, t):
    """exp((x - max) / t) over its sum; rows with nothing left give zeros."""
    m = x.amax(-1, keepdim=True)
    e = torch.where(x > -math.inf, torch.exp((x - m) * (1 / t)), torch.zeros_like(x))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-38)


def _first_argmax(score, valid):
    """Lowest index of the largest valid score of each row, -1 where none is valid."""
    n = score.shape[-1]
    score = torch.where(valid, score, torch.full_like(score, -math.inf))
    hit = valid & (score == score.amax(-1, keepdim=True))
    idx = torch.where(hit, torch.arange(n, device=score.device), n).amin(-1)
    return torch.where(idx < n, idx, -1)


def _verify_plain(s):
    tl, dl, tok, u = s["target"].float(), s["draft"].float(), s["tokens"], s["u"]
    b, k1, v = tl.shape
    k = k1 - 1
    t = torch.as_tensor(s["temp"], device=DEV, dtype=torch.float32).expand(b)
    n = s["lengths"].long() if s["lengths"] is not None else torch.full((b,), k, device=DEV)
    greedy = t == 0
    ts = torch.where(greedy, torch.ones_like(t), t)[:, None, None]
    best = _first_argmax(tl, tl > -math.inf)                       # [b, k + 1]
    p, q = _softmax(tl, ts), _softmax(dl, ts)
    px = p[:, :k].gather(-1, tok[..., None])[..., 0]
    qx = q.gather(-1, tok[..., None])[..., 0]
    ok = torch.where(greedy[:, None], tok == best[:, :k], u * qx < px)
    ok = ok & (torch.arange(k, device=DEV) < n[:, None])
    acc = ok.long().cumprod(-1).sum(-1)                            # [b]
    row = torch.arange(b, device=DEV)
    pr = p[row, acc]
    qr = torch.where((acc < n)[:, None], q[row, acc.clamp_max(k - 1)], torch.zeros_like(pr))
    r = (pr - qr).clamp_min(0)
    r = torch.where((r > 0).any(-1, keepdim=True), r, pr)
    nxt = torch.where(greedy, best[row, acc], _first_argmax(r / s["noise"], r > 0))
    out = torch.full((b, k1), -1, device=DEV, dtype=tok.dtype)
    out[:, :k] = torch.where(torch.arange(k, device=DEV) < acc[:, None], tok, -1)
    out[row, acc] = nxt
    return out, acc.int()


def _segment(lg):
    """exp of the sum of lg over (s, t] for every s <= t, zero above; lg [..., n]."""
    c = lg.cumsum(-1)
    n = lg.shape[-1]
    keep = torch.ones(n, n, device=lg.device, dtype=torch.bool).tril()
    diff = c[..., :, None] - c[..., None, :]
    return torch.where(keep, torch.exp(diff.clamp_max(0)), torch.zeros_like(diff))


def _gla_math(s, dt):
    """The block's outputs and the advanced state in dtype dt."""
    fq, fk, v, lg = (s[n].to(dt) for n in ("fq", "fk", "v", "lg"))
    S, z = s["state"].to(dt), s["zstate"].to(dt)
    kp, vp, lp = (x.to(dt) for x in s["pend"][:3])
    count = s["pend"][3]
    b, h, t, f = fq.shape
    hkv, hs = fk.shape[1], S.shape[1]
    if lg.dim() == 2:
        lg, lp = lg[:, None].expand(b, hs, t), lp[:, None].expand(b, hs, t)
    if hs != hkv:
        fk, v, kp, vp = (x.repeat_interleave(hs // hkv, 1) for x in (fk, v, kp, vp))
    live = torch.arange(t, device=fq.device) < count[:, None, None]
    lp = torch.where(live, lp, torch.zeros_like(lp))
    w = _segment(lp)[..., -1, :] * live                            # decay after each token
    S = S * torch.exp(lp.sum(-1))[..., None, None] + (kp * w[..., None]).transpose(-1, -2) @ vp
    z = z * torch.exp(lp.sum(-1))[..., None] + (kp * w[..., None]).sum(-2)
    qs = fq.view(b, hs, h // hs, t, f)
    M = _segment(lg)[:, :, None]
    a = (qs @ fk[:, :, None].transpose(-1, -2)) * M
    dec = torch.exp(lg.cumsum(-1))[:, :, None, :, None]
    num = dec * (qs @ S[:, :, None]) + a @ v[:, :, None]
    den = dec * (qs @ z[:, :, None, :, None]) + a.sum(-1, keepdim=True)
    return (num / den).view(b, h, t, -1), S, z


def _gla_plain(s):
    y, S, z = _gla_math(s, torch.float32)
    s["state"].copy_(S)
    s["zstate"].copy_(z)
    return y.bfloat16(), s["state"], s["zstate"]


def _rot(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * sin[:, None]


def _swa_math(s, dt):
    """The block's outputs and the rings with the accepted tokens, in dtype dt."""
    q, k, v, cos, sin, meta = (s[n].to(dt) for n in ("q", "k", "v", "cos", "sin", "meta"))
    kr, vr = s["k_ring"].to(dt), s["v_ring"].to(dt)
    kp, vp, cp, sp = (x.to(dt) for x in s["pend"][:4])
    pos, count = s["pos"].long(), s["pend"][4].long()
    b, h, t, d = q.shape
    hkv, w = kr.shape[1], kr.shape[2]
    base = pos + count
    # ring slot j after the update holds the last position below base with that remainder
    slot = torch.arange(w, device=q.device)
    at = base[:, None] - 1 - (base[:, None] - 1 - slot) % w        # [b, w]
    src = (at - pos[:, None])                                      # index into the pending tokens
    new = (src >= 0)[:, None, :, None]
    idx = src.clamp(0, t - 1)[:, None, :, None].expand(b, hkv, w, d)
    kr = torch.where(new, _rot(kp, cp, sp).gather(2, idx), kr)
    vr = torch.where(new, vp.gather(2, idx), vr)
    q, k = _rot(q, cos, sin), _rot(k, cos, sin)
    keys, vals = torch.cat([kr, k], 2), torch.cat([vr, v], 2)
    step = torch.arange(t, device=q.device)
    where = torch.cat([at, base[:, None] + step], 1)               # [b, w + t] positions
    mine = base[:, None] + step                                    # [b, t]
    see = ((where[:, None, :] >= 0) & (where[:, None, :] <= mine[..., None])
           & (where[:, None, :] > mine[..., None] - w))
    see[:, :, :w] &= (at < base[:, None])[:, None, :]
    x = (q.view(b, hkv, h // hkv, t, d) @ keys[:, :, None].transpose(-1, -2)) / d ** 0.5
    x = x.masked_fill(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if meta.numel():
        top = torch.maximum(top, meta.max())
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True) + torch.exp(meta - top).sum(-1, keepdim=True)
    return ((e @ vals[:, :, None]) / total).view(b, h, t, d), kr, vr


def _swa_plain(s):
    y, kr, vr = _swa_math(s, torch.float32)
    s["k_ring"].copy_(kr)
    s["v_ring"].copy_(vr)
    return y.bfloat16(), s["k_ring"], s["v_ring"]


_PLAIN = dict(int8=_int8_plain, verify=_verify_plain, gla=_gla_plain, swa=_swa_plain)


# ------------------------------------------------------------------ the framework's

def _own(s):
    lz = _api()
    if s["op"] == "int8":
        return lz.int8_linear(s["x"], s["w"], s["ws"], s["bias"])
    if s["op"] == "verify":
        return lz.verify_drafts(s["target"], s["draft"], s["tokens"], s["u"], s["noise"],
                                temperature=s["temp"], lengths=s["lengths"])
    if s["op"] == "gla":
        y = lz.decode.gla_decode_block(s["fq"], s["fk"], s["v"], s["lg"], s["state"],
                                       s["zstate"], pending=s["pend"])
        return y, s["state"], s["zstate"]
    y = lz.decode.swa_decode_block(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["meta"],
                                   s["k_ring"], s["v_ring"], s["pos"], pending=s["pend"])
    return y, s["k_ring"], s["v_ring"]


def run(state):
    with torch.no_grad():
        return _own(state) if own else _PLAIN[state["op"]](state)


# ------------------------------------------------------------------- work and exact

def work(c):
    if c["op"] == "int8":
        m, k, n, e = c["m"], c["k"], c["n"], _SIZE[c["dtype"]]
        return dict(bytes=m * k * e + n * k + 4 * n + m * n * e + (n * e if c["bias"] else 0),
                    flops=2 * m * k * n)
    if c["op"] == "verify":
        b, k, v, e = c["b"], c["k"], c["v"], _SIZE[c["dtype"]]
        return dict(bytes=b * ((2 * k + 1) * v * e + 4 * v + 24 * k + 12),
                    flops=4 * b * (2 * k + 1) * v)
    if c["op"] == "gla":
        b, h, hkv, t, f, d = (c[n] for n in ("b", "h", "hkv", "t", "f", "d"))
        hs = h if c["per_head"] else hkv
        gate = 4 * b * t * (h if c["per_head"] else 1)
        return dict(bytes=8 * b * hs * f * (d + 1) + 2 * (gate + 2 * b * hkv * t * (f + d))
                    + 2 * b * h * t * (f + d) + 4 * b,
                    flops=2 * b * t * (hs * f * d + h * f * d + h * (t + 1) // 2 * (f + d)))
    b, h, hkv, t, w, d = (c[n] for n in ("b", "h", "hkv", "t", "w", "d"))
    e = _SIZE[c["dtype"]]
    return dict(bytes=8 * b * hkv * (w + t // 2) * d + e * b * t * d * (h + 4 * hkv)
                + 2 * b * h * t * d + 16 * b * t * d + 8 * b,
                flops=4 * b * h * t * d * (w + t // 2))


def exact(case, seed):
    c = case
    if c["op"] == "verify":
        return None  # whole numbers
    s = _inputs(c, seed)
    if c["op"] == "gla":
        return _gla_exact(s)
    if c["op"] == "swa":
        return _swa_exact(s)
    # codes and scales are held in 32 and 8 bits by definition; all else in 64
    x = s["x"].double()
    top = x.abs().amax(-1, keepdim=True)
    n = torch.full_like(top, 127)
    inv = (n / top).float().double()
    codes = (x * inv).float().round().double()
    scale = (top / n).float().double()
    w, ws = s["w"], s["ws"].double()
    y = torch.empty(c["m"], c["n"], device=DEV, dtype=torch.float64)
    for i in range(0, c["n"], 8192):
        y[:, i:i + 8192] = (codes @ w[i:i + 8192].double().t()) * (scale * ws[i:i + 8192])
    if s["bias"] is not None:
        y += s["bias"].double()
    return y


def _gla_exact(s):
    """Token by token: S <- g S + k^T v, z <- g z + k, y = q S / q z."""
    S, z = s["state"].double(), s["zstate"].double()
    hs, hkv, h = S.shape[1], s["fk"].shape[1], s["fq"].shape[1]

    def step(S, z, k, v, lg):
        k, v = (x.double().repeat_interleave(hs // hkv, 1) for x in (k, v))
        g = torch.exp(lg.double()).reshape(lg.shape[0], -1, 1)
        return g[..., None] * S + k[..., None] * v[..., None, :], g * z + k

    kp, vp, lp, count = s["pend"]
    for t in range(kp.shape[2]):
        S2, z2 = step(S, z, kp[:, :, t], vp[:, :, t], lp[..., t])
        keep = (t < count)[:, None, None]
        S, z = torch.where(keep[..., None], S2, S), torch.where(keep, z2, z)
    S1, z1, ys = S, z, []
    for t in range(s["fq"].shape[2]):
        S1, z1 = step(S1, z1, s["fk"][:, :, t], s["v"][:, :, t], s["lg"][..., t])
        q = s["fq"][:, :, t].double()
        Sq, zq = (x.repeat_interleave(h // hs, 1) for x in (S1, z1))
        ys.append((q[..., None] * Sq).sum(-2) / (q * zq).sum(-1, keepdim=True))
    return torch.stack(ys, 2), S, z


def _swa_exact(s):
    """Token by token: rotate, write slot position % window, attend the whole ring."""
    b, h, t, d = s["q"].shape
    hkv, w = s["k_ring"].shape[1:3]
    half = d // 2

    def rotate(x, c, n):
        x, c, n = x.double(), c.double()[:, None], n.double()[:, None]
        return torch.cat([x[..., :half] * c[..., :half] - x[..., half:] * n[..., :half],
                          x[..., half:] * c[..., half:] + x[..., :half] * n[..., half:]], -1)

    kr, vr = s["k_ring"].double(), s["v_ring"].double()
    kp, vp, cp, sp, count = s["pend"]
    row = torch.arange(b, device=DEV)
    pos = s["pos"].long()
    for i in range(t):
        live = (i < count)[:, None, None]
        slot = (pos + i) % w
        kr[row, :, slot] = torch.where(live, rotate(kp[:, :, i], cp[:, i], sp[:, i]),
                                       kr[row, :, slot])
        vr[row, :, slot] = torch.where(live, vp[:, :, i].double(), vr[row, :, slot])
    pos = pos + count.long()
    k1, v1, ys = kr.clone(), vr.clone(), []
    for i in range(t):
        slot = (pos + i) % w
        k1[row, :, slot] = rotate(s["k"][:, :, i], s["cos"][:, i], s["sin"][:, i])
        v1[row, :, slot] = s["v"][:, :, i].double()
        q = rotate(s["q"][:, :, i], s["cos"][:, i], s["sin"][:, i])
        keys, vals = (x.repeat_interleave(h // hkv, 1) for x in (k1, v1))
        x = (keys @ q[..., None])[..., 0] / d ** 0.5
        seen = torch.arange(w, device=DEV) < (pos + i + 1)[:, None]
        x = x.masked_fill(~seen[:, None], -math.inf)
        x = torch.cat([x, s["meta"].double().expand(b, h, -1)], -1)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        ys.append((p[..., None, :w] @ vals)[..., 0, :])
    return torch.stack(ys, 2), kr, vr
