"""The layer cache of drafted decoding on the GPU: what a refused step leaves behind."""
import pytest
import torch

from test_decode_block_cuda import _gla_inputs, _swa_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


def _cache_and_blocks(T=4):
    """A cache and the arguments of two blocks (without meta and accepted)."""
    from lizard_cuda.decode import LayerCache
    fq, blk_a, blk_b, _, S, z = _gla_inputs(2, 4, 2, 32, 64, T, T, False, 41)
    q, swa_a, swa_b, meta, kr, vr, pos = _swa_inputs(2, 4, 2, 16, 64, T, T, torch.bfloat16,
                                                     [40, 90], seed=42)
    cache = LayerCache(S, z, kr, vr, pos)

    def args(gla, swa):
        (fk, _, lg), (k, v, cos, sin) = gla, swa[:4]
        return fq, fk, v, lg, q, k, cos, sin

    return cache, args(blk_a, swa_a), args(blk_b, swa_b), meta


def _copy(cache):
    from lizard_cuda.decode import LayerCache
    return LayerCache(*(t.clone() for t in (cache.state, cache.zstate, cache.k_ring, cache.v_ring,
                                            cache.pos)))


def _same(a, b):
    return all(torch.equal(getattr(a, n), getattr(b, n))
               for n in ("state", "zstate", "k_ring", "v_ring", "pos"))


@pytest.mark.parametrize("what", ["sinks", "tables", "queries"])
def test_a_call_that_was_refused_can_be_repeated(what):
    """One call of the two branches' is refused (by the library, or before it); the call,
    put right, then gives what it would have given at once."""
    cache, first, second, meta = _cache_and_blocks()
    clean = _copy(cache)
    n = torch.tensor([3, 1], dtype=torch.int32, device=DEV)
    for c in (cache, clean):
        c.block(*first, meta, None)
    want = clean.block(*second, meta, n)
    bad, bad_meta = list(second), meta
    if what == "sinks":
        bad_meta = torch.zeros(33, device=DEV)
    elif what == "tables":
        bad[6] = bad[6][:, :2]
    else:
        bad[0] = bad[0][:, :, :2]  # the state's step refuses
    for _ in range(2):
        with pytest.raises((ValueError, RuntimeError)):
            cache.block(*bad, bad_meta, n)
    got = cache.block(*second, meta, n)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and _same(cache, clean)
    for c in (cache, clean):
        c.settle(n)
    assert _same(cache, clean) and cache.pending is None


def test_counts_outside_the_block_are_clamped_throughout():
    cache, first, second, meta = _cache_and_blocks()
    clean = _copy(cache)
    over = torch.tensor([-3, 9], dtype=torch.int32, device=DEV)
    for c, n in ((cache, over), (clean, over.clamp(0, 4))):
        c.block(*first, meta, None)
        c.block(*second, meta, n)
        c.settle(n)
    assert _same(cache, clean)
