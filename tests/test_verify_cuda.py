"""verify_drafts against a 64-bit restatement of its rule, token for token, at
the masks, sizes and layouts where it can go wrong; the law of its tokens; its
refusals. The random inputs are fixed by their seeds; a decision of theirs
closer than fp32 resolves would show as a mismatch (none is)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


def _softmax(x, t):
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    live = x > -math.inf
    if not live.any():
        return torch.zeros_like(x)
    e = torch.where(live, torch.exp((x - x[live].max()) / t), 0.0)
    return e / e.sum()


def _first_max(score, valid):
    if not valid.any():
        return -1
    return int((valid & (score == score[valid].max())).nonzero()[0])


def reference(target, draft, tokens, u, noise, temperature=1.0, lengths=None):
    B, K1, V = target.shape
    out = torch.full((B, K1), -1, dtype=torch.int64)
    acc = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        t = float(temperature[b]) if isinstance(temperature, torch.Tensor) else temperature
        n = K1 - 1 if lengths is None else max(0, min(int(lengths[b]), K1 - 1))
        tg, e = target[b].double().cpu(), noise[b].double().cpu()
        dr = draft[b].double().cpu()
        a, greedy = 0, not t >= 1e-5
        while a < n:
            x = int(tokens[b, a])
            if greedy:
                row = torch.where(torch.isnan(tg[a]), -math.inf, tg[a])
                ok = x == _first_max(row, row > -math.inf)
            else:
                ok = 0 <= x < V and float(u[b, a]) * _softmax(dr[a], t)[x] < _softmax(tg[a], t)[x]
            if not ok:
                break
            out[b, a] = x
            a += 1
        if greedy:
            row = torch.where(torch.isnan(tg[a]), -math.inf, tg[a])
            nxt = _first_max(row, row > -math.inf)
        else:
            p = _softmax(tg[a], t)
            r = (p - _softmax(dr[a], t)).clamp_min(0) if a < n else p
            nxt = _first_max(r / e, (r > 0) & (e > 0))
            if nxt < 0:
                nxt = _first_max(p / e, (p > 0) & (e > 0))
        out[b, a], acc[b] = nxt, a
    return out, acc


def inputs(B, K, V, dtype, seed, temp=1.0, spread=2.0, own=0.8, masked=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    target = spread * torch.randn(B, K + 1, V, generator=g, device=DEV)
    draft = target[:, :K] + own * torch.randn(B, K, V, generator=g, device=DEV)
    if masked:
        off = torch.rand(B, 1, V, generator=g, device=DEV) < masked
        target.masked_fill_(off, -math.inf)
        draft.masked_fill_(off, -math.inf)
    target, draft = target.to(dtype), draft.to(dtype)
    race = -torch.log1p(-torch.rand(B, K, V, generator=g, device=DEV)) + 1e-9
    q = torch.softmax(draft.float() / temp, -1).nan_to_num(0)
    tokens = (q / race).argmax(-1)
    u = torch.rand(B, K, generator=g, device=DEV)
    noise = -torch.log1p(-torch.rand(B, V, generator=g, device=DEV)) + 1e-9
    return target, draft, tokens, u, noise


def check(args, **kw):
    from lizard_cuda import verify_drafts
    out, acc = verify_drafts(*args, **kw)
    want, wacc = reference(*args, **kw)
    assert out.dtype == args[2].dtype and acc.dtype == torch.int32
    assert torch.equal(acc.cpu(), wacc), (acc, wacc)
    assert torch.equal(out.cpu().long(), want), (out, want)
    return out, acc


@pytest.mark.parametrize("B,K,V,dtype", [
    (1, 1, 1, torch.float32),           # one token to choose from
    (2, 3, 5, torch.bfloat16),
    (1, 4, 128256, torch.bfloat16),     # the model's vocabulary
    (3, 2, 128256, torch.float32),
    (7, 5, 4099, torch.bfloat16),       # rows on every alignment
    (5, 7, 32003, torch.float32),
    (2, 64, 257, torch.float32),        # the longest draft
    (300, 2, 33, torch.bfloat16),
])
@pytest.mark.parametrize("masked", [0.0, 0.4])
def test_verify_matches_the_rule(B, K, V, dtype, masked):
    args = inputs(B, K, V, dtype, B + K + V, masked=masked)
    out, acc = check(args)
    if B * K >= 20 and V > 100:
        assert 0 < int(acc.sum()) < B * K  # both outcomes occur


def test_temperatures_lengths_and_types():
    B, K, V = 40, 4, 1003
    args = list(inputs(B, K, V, torch.float32, 5))
    temp = torch.tensor([0.0, 0.5, 1.0, 1.7, 1e-7], device=DEV).repeat(8)
    lengths = torch.arange(B, device=DEV).int() % 7 - 1  # -1 .. 5, clamped to 0 .. 4
    check(args, temperature=temp, lengths=lengths)
    check(args, temperature=0.7)
    args[2] = args[2].int()
    check(args, temperature=temp)
    out, acc = check(args, temperature=0.0)
    args[2][:, :] = out[:, :1]
    check(args, temperature=0)


def test_greedy_takes_the_lowest_of_equal_logits():
    args = list(inputs(6, 3, 5000, torch.bfloat16, 6))
    for j in (4999, 8, 3001):
        args[0][..., j] = 50.0
    args[2][:, 0], args[2][:, 1] = 8, 8
    args[2][::2, 1] = 4999
    out, acc = check(args, temperature=0.0)
    assert acc.tolist() == [1, 2] * 3 and (out[:, 0] == 8).all()
    args[0].neg_()  # negative logits order as well
    check(args, temperature=0.0)


def test_no_drafts_is_sampling():
    args = inputs(9, 0, 777, torch.float32, 7)
    out, acc = check(args)
    assert out.shape == (9, 1) and not acc.any()


def test_masks_that_leave_nothing():
    for temp in (1.0, 0.0):
        args = list(inputs(6, 2, 300, torch.float32, 8))
        args[0][0] = -math.inf            # nothing is allowed: refused, and no next token
        args[0][1] = math.nan
        args[0][2, 1, 7] = math.nan       # a NaN is a masked token
        args[0][3, 0, 5] = math.inf       # an infinity takes all the probability
        args[1][4] = -math.inf            # a draft without probabilities: its token has q = 0
        args[0][5, 0, args[2][5, 0]] = -math.inf  # a drafted token that the target forbids
        out, acc = check(args, temperature=temp)
        assert out[0, 0] == -1 and out[1, 0] == -1 and acc[5] == 0
        assert out[3, int(acc[3])] == 5 or acc[3] > 0
        # u = 0 does not accept a token of probability 0
        args[3].zero_()
        out, acc = check(args, temperature=temp)
        assert acc[5] == 0


@pytest.mark.parametrize("nothing", [-math.inf, math.nan])
@pytest.mark.parametrize("V", [97, 300, 1000])
def test_a_draft_without_probabilities_stays_inside_the_vocabulary(V, nothing):
    """Draft rows masked throughout, in rows that go on past the vocabulary with large
    logits and small noise: nothing past the end is looked at."""
    from lizard_cuda import verify_drafts
    B, K = 16, 2
    args = list(inputs(B, K, V, torch.float32, 18))
    args[1][:] = nothing
    args[2][:] = -1
    wide = [torch.full((B, n, V + 300), 60.0, device=DEV) for n in (K + 1, K)]
    noise = torch.full((B, V + 300), 1e-9, device=DEV)
    for w, a in zip(wide, args):
        w[..., :V] = a
    noise[:, :V] = args[4]
    want, wacc = reference(*args)
    out, acc = verify_drafts(wide[0][..., :V], wide[1][..., :V], *args[2:4], noise[:, :V])
    assert not wacc.any() and torch.equal(acc.cpu(), wacc)
    assert torch.equal(out.cpu(), want)


def test_an_infinite_temperature_is_uniform_over_what_is_allowed():
    args = list(inputs(6, 2, 9001, torch.float32, 19, masked=0.3))
    args[0][:, :, 2000:7000] = -math.inf  # pieces of a row with nothing in them
    args[1][:, :, 2000:7000] = -math.inf
    check(args, temperature=torch.full((6,), math.inf, device=DEV))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masks_of_the_types_lowest_value(dtype):
    """Forbidden tokens at finfo.min rather than -inf; a piece of the row, and a whole
    row, of nothing else."""
    low = torch.finfo(dtype).min
    args = list(inputs(5, 2, 40000, dtype, 17))
    args[0][:, :, 100:30000] = low
    args[1][:, :, 100:30000] = low
    args[0][3, 0] = low  # uniform over the vocabulary, as softmax has it
    check(args)
    check(args, temperature=0.3)


def test_tokens_outside_the_vocabulary_are_refused():
    args = list(inputs(4, 3, 100, torch.float32, 9))
    args[3].zero_()  # accepts whatever has a probability
    args[2][0, 1], args[2][1, 0], args[2][2, 2] = -1, 100, 1 << 40
    out, acc = check(args)
    assert acc.tolist() == [1, 0, 2, 3]


def test_an_empty_residual_draws_from_the_target():
    args = list(inputs(5, 2, 2000, torch.float32, 10, own=0.0))
    args[3].fill_(1.0)  # refuses although p = q
    out, acc = check(args)
    assert not acc.any() and (out[:, 0] >= 0).all()


def test_strides_and_padding_of_the_vocabulary():
    from lizard_cuda import verify_drafts
    args = list(inputs(4, 3, 1000, torch.bfloat16, 11))
    want = verify_drafts(*args)
    pad = [torch.full((4, n, 1033), 60.0, device=DEV, dtype=torch.bfloat16) for n in (4, 3)]
    for p, a in zip(pad, args):
        p[..., 16:1016] = a
    noise = torch.full((4, 2111), 1e-6, device=DEV)
    noise[:, 3:1003] = args[4]
    got = verify_drafts(pad[0][..., 16:1016], pad[1][..., 16:1016], *args[2:4], noise[:, 3:1003])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a broadcast row of noise, transposed logits
    t = args[0].transpose(0, 1).contiguous().transpose(0, 1)
    one = args[4][:1].expand(4, 1000)
    want = verify_drafts(*args[:4], one.contiguous())
    got = verify_drafts(t, *args[1:4], one)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_noise_that_is_not_positive_is_never_chosen():
    args = list(inputs(3, 1, 64, torch.float32, 12))
    args[4][:, ::2] = 0
    args[4][:, 1::4] = math.nan
    check(args)
    args[4].fill_(math.nan)
    out, acc = check(args)
    assert all(int(out[b, int(acc[b])]) == -1 for b in range(3))


def test_the_first_token_follows_the_target():
    """Whatever the draft, the first emitted token has the target's law: chi-square
    over 8 tokens from 8192 sequences, 7 degrees of freedom; 45 has probability 1e-7."""
    from lizard_cuda import verify_drafts
    g = torch.Generator(device=DEV).manual_seed(13)
    B, K, V = 8192, 2, 8
    target = torch.randn(1, K + 1, V, generator=g, device=DEV).expand(B, K + 1, V)
    draft = torch.randn(1, K, V, generator=g, device=DEV).expand(B, K, V)
    q = torch.softmax(draft, -1)
    tokens = (q / torch.empty(B, K, V, device=DEV).exponential_(generator=g)).argmax(-1)
    u = torch.rand(B, K, generator=g, device=DEV)
    noise = torch.empty(B, V, device=DEV).exponential_(generator=g)
    out, acc = verify_drafts(target, draft, tokens, u, noise)
    assert 0.2 < float((acc > 0).float().mean()) < 0.95
    p = torch.softmax(target[0, 0].double(), -1)
    n = torch.bincount(out[:, 0], minlength=V).double()
    assert float(((n - B * p) ** 2 / (B * p)).sum()) < 45


def test_verify_refusals():
    from lizard_cuda import verify_drafts
    args = list(inputs(2, 2, 10, torch.float32, 14))
    with pytest.raises(ValueError, match="draft_logits"):
        verify_drafts(args[0], args[1][:, :1], *args[2:])
    with pytest.raises(ValueError, match="noise"):
        verify_drafts(*args[:4], args[4][:, :9])
    with pytest.raises(ValueError, match="int64 or int32"):
        verify_drafts(*args[:2], args[2].float(), *args[3:])
    with pytest.raises(ValueError, match="temperature"):
        verify_drafts(*args, temperature=-1.0)
    with pytest.raises(ValueError, match="temperature"):
        verify_drafts(*args, temperature=torch.ones(3, device=DEV))
    with pytest.raises(ValueError, match="lengths"):
        verify_drafts(*args, lengths=torch.ones(2, device=DEV))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        verify_drafts(args[0].cpu(), *args[1:])
    with pytest.raises(RuntimeError, match="at most 64"):
        verify_drafts(*inputs(1, 65, 10, torch.float32, 15))
    empty = inputs(1, 2, 10, torch.float32, 16)
    out, acc = verify_drafts(*(t[:0] for t in empty))
    assert out.shape == (0, 3) and acc.shape == (0,)
