"""The cache of drafted decoding when a call fails, is forgotten or says too much. The two
kernels' calls are replaced by recorders: no GPU needed."""
import types

import pytest
import torch


@pytest.fixture
def cache(monkeypatch):
    """A LayerCache with a pending block of 3 tokens for 2 rows, whose steps record
    (name, count) in .calls and raise when their name is in .failing."""
    from lizard_cuda import decode
    B, H, T, F, D, W = 2, 2, 3, 4, 8, 16
    c = decode.LayerCache(torch.zeros(B, H, F, D), torch.zeros(B, H, F), torch.zeros(B, H, W, D),
                          torch.zeros(B, H, W, D), torch.tensor([20, 30], dtype=torch.int32))
    c.calls, c.failing = [], set()

    def step(name):
        def run(*args, **kw):
            if name in c.failing:
                raise ValueError(f"{name} refuses")
            pending = kw.get("pending", args[-1])
            c.calls.append((name, None if pending is None else pending[-1].tolist()))
            return torch.zeros(B, H, T, D)
        return run

    monkeypatch.setattr(decode, "gla_decode_block", step("gla"))
    monkeypatch.setattr(decode, "swa_decode_block", step("swa"))

    def block(accepted=None):
        x, f = torch.zeros(B, H, T, D), torch.zeros(B, H, T, F)
        return c.block(f, f, x, torch.zeros(B, T), x, x, torch.zeros(1, T, D), torch.zeros(1, T, D),
                       torch.zeros(0), accepted)

    c.next = block
    block()
    del c.calls[:]
    return c


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("settle", [False, True])
def test_a_refused_step_leaves_nothing_folded_in_twice(cache, settle):
    """The ring's step (which may be repeated: it writes the same slots) comes before the
    state's (which may not); where one refuses, pos and the pending block stay."""
    act = cache.settle if settle else cache.next
    before = cache.pending
    cache.failing = {"swa"}
    with pytest.raises(ValueError, match="swa refuses"):
        act(_i32(1, 2))
    assert not [n for n, _ in cache.calls if n == "gla"]
    cache.failing = {"gla"}
    with pytest.raises(ValueError, match="gla refuses"):
        act(_i32(1, 2))
    assert cache.pending is before and cache.pos.tolist() == [20, 30]
    cache.failing = set()
    act(_i32(1, 2))
    assert [n for n, _ in cache.calls].count("gla") == 1 and cache.pos.tolist() == [21, 32]
    assert (cache.pending is None) == settle


@pytest.mark.parametrize("settle", [False, True])
def test_pos_advances_by_what_the_kernels_fold_in(cache, settle):
    """The kernels take counts as 0 .. the block's length; so does pos."""
    (cache.settle if settle else cache.next)(_i32(-4, 9))
    assert cache.pos.tolist() == [20, 33] and cache.pos.dtype == torch.int32


def _layer(monkeypatch):
    """A layer whose forms of decoding record which of them ran."""
    from lizard_cuda.layer import LizardAttention
    cfg = types.SimpleNamespace(hidden_size=32, num_attention_heads=4, num_key_value_heads=2)
    layer = LizardAttention(cfg, 0, window=8, num_meta=2, feature_dim=4)
    ran = []
    monkeypatch.setattr(layer, "decode_block",
                        lambda x, pe, c, accepted: ran.append(accepted) or x)
    monkeypatch.setattr(layer, "decode", lambda x, pe, c: ran.append("token") or x)
    return layer, ran


def test_a_cache_may_be_a_plain_dict(cache, monkeypatch):
    layer, ran = _layer(monkeypatch)
    cache.pending = None
    x = torch.zeros(2, 1, 32)
    layer(x, None, lizard_cache={0: cache})
    assert ran == ["token"]


def test_every_block_needs_a_draft_call_of_its_own(cache, monkeypatch):
    """A second call would fold the newer block in with the older one's counts."""
    from lizard_cuda.decode import LizardCache
    layer, ran = _layer(monkeypatch)
    x, c = torch.zeros(2, 3, 32), LizardCache({0: cache})
    for n in (_i32(1, 2), _i32(3, 0)):
        layer(x, None, lizard_cache=c.draft(n))
        assert ran[-1] is n
        with pytest.raises(RuntimeError, match="draft"):
            layer(x, None, lizard_cache=c)
    assert len(ran) == 2


def test_a_block_that_failed_may_be_repeated(cache, monkeypatch):
    from lizard_cuda.decode import LizardCache
    layer, ran = _layer(monkeypatch)
    x, c = torch.zeros(2, 3, 32), LizardCache({0: cache})

    def refuse(*args):
        raise ValueError("refused")

    with monkeypatch.context() as m:
        m.setattr(layer, "decode_block", refuse)
        with pytest.raises(ValueError, match="refused"):
            layer(x, None, lizard_cache=c.draft(_i32(1, 2)))
    layer(x, None, lizard_cache=c)
    assert ran[0].tolist() == [1, 2]


@pytest.mark.parametrize("whole", [True, False])
def test_a_pending_block_is_not_passed_over(cache, whole):
    """Token by token with a block pending: refused, whichever way the layer is called."""
    from lizard_cuda.decode import LizardCache
    from lizard_cuda.layer import LizardAttention
    cfg = types.SimpleNamespace(hidden_size=32, num_attention_heads=4, num_key_value_heads=2)
    layer = LizardAttention(cfg, 0, window=8, num_meta=2, feature_dim=4)
    x = torch.zeros(2, 1, 32)
    with pytest.raises(ValueError, match="settle"):
        if whole:
            layer(x, (x, x), lizard_cache=LizardCache({0: cache}))
        else:
            layer.decode(x, (x, x), cache)


def test_a_cache_of_ones_own_needs_no_pending_field(cache):
    """Token by token, the layer reads the state, the rings and pos; without a GPU it gets
    as far as the kernels."""
    from lizard_cuda.layer import LizardAttention
    cfg = types.SimpleNamespace(hidden_size=32, num_attention_heads=4, num_key_value_heads=2)
    layer = LizardAttention(cfg, 0, window=8, num_meta=2, feature_dim=4)
    own = types.SimpleNamespace(state=cache.state, zstate=cache.zstate, k_ring=cache.k_ring,
                                v_ring=cache.v_ring, pos=cache.pos)
    x = torch.zeros(2, 1, 32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer(x, (x, x), lizard_cache={0: own})
