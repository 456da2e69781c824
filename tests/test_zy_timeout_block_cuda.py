"""The bounded waits of the block steps, exercised without a GPU fault: a test switch leaves
out one load of the state (or of the ring's first part), so that nothing ever completes its
barrier and the wait runs out after about 2 s. The call then returns with the wait's site
in the flag and has written no output and no state; after clearing the flag the same call
is right. No copy is in flight when the kernels leave. Collected after the other GPU
tests, which check that no wait ever timed out."""
import ctypes

import pytest
import torch

from test_decode_block_cuda import (_check_gla, _check_swa, _gla_inputs, _gla_walk, _swa_inputs)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _in_vain(lib, _lib, call, site):
    """Runs call with the load withheld; the flag has to name the site."""
    assert _lib.device_timeout_flag() == 0
    lib.lz_test_withhold_block_load(1)
    try:
        call()
        torch.cuda.synchronize()
        flag = _lib.device_timeout_flag()
    finally:
        lib.lz_test_withhold_block_load(0)
        _lib.clear_device_timeout_flag()
    assert flag == 0x80000000 | site
    assert _lib.device_timeout_flag() == 0


@pytest.mark.parametrize("F,D,T", [(64, 64, 5), (200, 200, 40), (93, 84, 0)])
def test_a_state_that_does_not_come(built_lib, F, D, T):
    from lizard_cuda import _lib
    lib, p = _lib.load(), _lib.ptr
    B, H, Hkv, Tp = 2, 4, 2, 6
    fq, (fk, v, lg), (fkp, vp, lgp), count, S, z = _gla_inputs(B, H, Hkv, F, D, T, Tp, False, F)
    y = torch.full((B, H, T, D), 7.0, device=DEV, dtype=torch.bfloat16)
    S0, z0 = S.clone(), z.clone()

    def call():
        _lib.check(lib.lz_gla_decode_block(
            p(fq), p(fk), p(v), p(lg), 0, p(fkp), p(vp), p(lgp), p(count), p(S), p(z), p(y), B, H,
            Hkv, Hkv, T, Tp, F, D, _lib.stream_of(S)), "gla decode block")

    _in_vain(lib, _lib, call, 95)
    assert (y == 7).all() and torch.equal(S, S0) and torch.equal(z, z0)
    call()
    adv = _gla_walk(S0.double(), z0.double(), fkp, vp, lgp, None, count)
    ref = _gla_walk(adv[2], adv[3], fk, v, lg, fq)
    _check_gla(y, S, z, (ref[0], ref[1]) + adv[2:], Tp)
    assert _lib.device_timeout_flag() == 0


@pytest.mark.parametrize("W,D,T,rep", [(64, 64, 5, 4), (600, 64, 20, 2), (100, 256, 9, 4)])
def test_a_ring_that_does_not_come(built_lib, W, D, T, rep):
    """Rings in one part and in several: the later parts are not waited for in vain, either."""
    from lizard_cuda import _lib
    lib, p = _lib.load(), _lib.ptr
    B, Hkv, Tp = 2, 2, 3
    H = rep * Hkv
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(B, H, Hkv, W, D, T, Tp, torch.bfloat16,
                                                  [3 * W, 5], seed=W)
    kr0, vr0 = kr.clone(), vr.clone()
    y = torch.full((B, H, T, D), 7.0, device=DEV, dtype=torch.bfloat16)
    n = lib.lz_swa_decode_block_workspace_bytes(B, H, Hkv, T, D)
    ws = torch.empty(n, device=DEV, dtype=torch.uint8)
    strides = (ctypes.c_longlong * 12)(*q.stride(), *blk[0].stride(), *blk[1].stride())
    strides_p = (ctypes.c_longlong * 8)(*pend[0].stride(), *pend[1].stride())

    def call():
        _lib.check(lib.lz_swa_decode_block(
            p(q), p(blk[0]), p(blk[1]), 1, ctypes.cast(strides, ctypes.c_void_p), p(blk[2]),
            p(blk[3]), 0, T * D, p(pend[0]), p(pend[1]), ctypes.cast(strides_p, ctypes.c_void_p),
            p(pend[2]), p(pend[3]), Tp * D, p(pend[4]), p(kr), p(vr), p(pos), p(meta),
            meta.numel(), p(y), p(ws), n, B, H, Hkv, T, Tp, W, D, _lib.stream_of(q)),
            "swa decode block")

    _in_vain(lib, _lib, call, 96)
    assert (y == 7).all()
    call()  # the accepted tokens are in the ring already: writing them again changes nothing
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)
    assert _lib.device_timeout_flag() == 0
