"""Drafted decoding end to end: the layer's block step against its full forward and
its token-by-token decode, with prefixes kept and refused; the 8-bit model; and
speculative_generate against the model's own full forwards."""
import copy
from types import SimpleNamespace

import pytest
import torch

import lizard_oracle as orc
from parity import assert_output

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layer_blocks_match_full_forward(dtype):
    """Blocks of which only a prefix stands (different for each row): every block's
    outputs are the full forward's at its positions."""
    from lizard_cuda.decode import LizardCache
    from lizard_cuda.layer import LizardAttention
    cfg = SimpleNamespace(hidden_size=256, num_attention_heads=4, num_key_value_heads=2)
    torch.manual_seed(0)
    layer = LizardAttention(cfg, 0, window=16, num_meta=4, feature_dim=32)
    with torch.no_grad():
        for p in layer.parameters():
            p.normal_(0, 0.3)
    layer = layer.to(DEV).to(dtype)
    B, L0, T = 3, 30, 5
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(B, L0, 256, generator=g, device=DEV).to(dtype)
    cos, sin = (t.to(DEV) for t in orc.rotary_tables(128, 64, 5e5))
    cos, sin = cos.view(1, 128, 64), sin.view(1, 128, 64)

    def tables(pos):  # [B, T] positions
        return cos[0][pos], sin[0][pos]

    with torch.no_grad():
        cache = LizardCache()
        layer(x, (cos[:, :L0].expand(B, L0, 64), sin[:, :L0].expand(B, L0, 64)),
              lizard_cache=cache)
        rows = [list(x[b]) for b in range(B)]  # the tokens that stand
        stand = None
        for counts in ([5, 1, 3], [1, 4, 2], [5, 5, 0], [2, 3, 5]):
            blk = torch.randn(B, T, 256, generator=g, device=DEV).to(dtype)
            pos = torch.tensor([[len(r) + t for t in range(T)] for r in rows], device=DEV)
            y = layer(blk, tables(pos), lizard_cache=cache.draft(stand))[0]
            for b in range(B):
                seq = torch.stack(rows[b] + list(blk[b]))[None]
                n = seq.shape[1]
                full = layer(seq, (cos[:, :n], sin[:, :n]))[0][0, -T:]
                assert_output(y[b], full, f"block of row {b}", layer=True)
                rows[b] += list(blk[b, :counts[b]])
            stand = torch.tensor(counts, dtype=torch.int32, device=DEV)
        cache.settle(stand)
        assert cache[0].pos.tolist() == [len(r) for r in rows] and cache[0].pending is None
        # token by token from there
        new = torch.randn(B, 1, 256, generator=g, device=DEV).to(dtype)
        pos = torch.tensor([[len(r)] for r in rows], device=DEV)
        y = layer(new, tables(pos), lizard_cache=cache)[0]
        for b in range(B):
            seq = torch.stack(rows[b] + [new[b, 0]])[None]
            n = seq.shape[1]
            full = layer(seq, (cos[:, :n], sin[:, :n]))[0][0, -1:]
            assert_output(y[b], full, f"decode after settling, row {b}", layer=True)


def _model(seed=1):
    from test_model import tiny_llama
    from lizard_cuda.model import to_lizard
    model = to_lizard(tiny_llama(layers=2), window=16, num_meta=4, feature_dim=16)
    torch.manual_seed(seed)
    with torch.no_grad():
        for block in model.model.layers:
            for n, p in block.self_attn.named_parameters():
                if not n.endswith("proj.weight"):
                    p.normal_(0, 0.3)
    return model.to(DEV).eval()


def test_to_int8_swaps_the_large_layers_and_stays_close():
    from lizard_cuda import Int8Linear
    from lizard_cuda.model import to_int8
    model = _model()
    ids = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(2)).to(DEV)
    with torch.no_grad():
        ref = model(ids, use_cache=False).logits
        quick = to_int8(copy.deepcopy(model))
        got = quick(ids, use_cache=False).logits
    kinds = [type(m).__name__ for m in quick.modules()]
    assert kinds.count("Int8Linear") == 2 * 7 + 1
    assert isinstance(quick.lm_head, Int8Linear)
    assert not isinstance(quick.model.layers[0].self_attn.phi_q, Int8Linear)
    # a hundredth of the range a layer, over some ten layers in a row
    assert float((got - ref).norm() / ref.norm()) < 0.1


@pytest.mark.parametrize("same", [True, False])
def test_speculative_greedy_is_the_models_own(same):
    from lizard_cuda.model import speculative_generate, to_int8
    model = _model()
    draft = copy.deepcopy(model) if same else to_int8(copy.deepcopy(model))
    B, L, steps = 3, 20, 24
    ids = torch.randint(0, 97, (B, L), generator=torch.Generator().manual_seed(3)).to(DEV)
    toks, cache, rounds = speculative_generate(model, draft, ids, steps, draft_len=4)
    assert toks.shape == (B, steps) and -(-(steps - 1) // 5) <= rounds < steps
    with torch.no_grad():
        full = model(torch.cat([ids, toks], 1), use_cache=False).logits[:, L - 1:-1].float()
    # each token is the argmax of the full forward, up to its bf16 branch outputs
    got = full.gather(-1, toks[..., None])[..., 0]
    assert (full.amax(-1) - got <= 2e-2 * full.abs().amax()).all()
    if same:  # a draft that is the model itself is hardly ever refused
        assert rounds <= 8
    assert cache[0].pending is None and (cache[0].pos >= L + steps - 1).all()


def test_speculative_sampling_follows_the_model():
    """The second token's law, over many copies of one prompt, against the model's own
    probabilities: chi-square over the 8 likeliest tokens and the rest."""
    from lizard_cuda.model import speculative_generate, to_int8
    model = _model(4)
    with torch.no_grad():
        model.lm_head.weight.mul_(6)  # a peaked distribution
    draft = to_int8(copy.deepcopy(model))
    with torch.no_grad():
        for p in draft.model.layers[1].self_attn.parameters():
            p.mul_(0.5)  # and a draft that is wrong
    B = 2048
    ids = torch.randint(0, 97, (1, 12), generator=torch.Generator().manual_seed(5)).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(6)
    toks, _, rounds = speculative_generate(model, draft, ids.expand(B, 12), 3, draft_len=2,
                                           temperature=0.8, generator=g)
    first = int(torch.bincount(toks[:, 0]).argmax())
    rows = toks[toks[:, 0] == first]
    with torch.no_grad():
        seq = torch.cat([ids, torch.tensor([[first]], device=DEV)], 1)
        p = torch.softmax(model(seq, use_cache=False).logits[0, -1].double() / 0.8, -1)
    n = torch.bincount(rows[:, 1], minlength=97).double()
    top = p.topk(8).indices
    obs = torch.cat([n[top], (n.sum() - n[top].sum())[None]])
    want = torch.cat([p[top], (1 - p[top].sum())[None]]) * n.sum()
    chi = float(((obs - want) ** 2 / want.clamp_min(1e-9)).sum())
    # 8 degrees of freedom: 45 has probability 4e-7
    assert rows.shape[0] > 100 and chi < 45, chi


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_speculative_with_a_draft_of_nan(temperature):
    """A draft whose logits are NaN proposes nothing that stands: every round gives the
    model's own token."""
    from lizard_cuda.model import speculative_generate
    model = _model()
    draft = copy.deepcopy(model)
    with torch.no_grad():
        draft.lm_head.weight.fill_(float("nan"))
    ids = torch.randint(0, 97, (2, 20), generator=torch.Generator().manual_seed(3)).to(DEV)
    steps = 6
    toks, cache, rounds = speculative_generate(
        model, draft, ids, steps, draft_len=3, temperature=temperature,
        generator=torch.Generator(device=DEV).manual_seed(7))
    assert rounds == steps - 1 and int(toks.min()) >= 0
    assert (cache[0].pos == 20 + steps - 1).all()
    if temperature == 0:
        with torch.no_grad():
            full = model(torch.cat([ids, toks], 1), use_cache=False).logits[:, 19:-1].float()
        got = full.gather(-1, toks[..., None])[..., 0]
        assert (full.amax(-1) - got <= 2e-2 * full.abs().amax()).all()


def test_speculative_refusals():
    from lizard_cuda.model import speculative_generate
    model = _model()
    ids = torch.zeros(1, 4, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="draft_len"):
        speculative_generate(model, model, ids, 4, draft_len=64)
