"""The SWA block step where its sizes, sinks and types leave the usual. Reference and
tolerances are those of test_decode_block_cuda.py."""
import math

import pytest
import torch

from test_decode_block_cuda import _check_swa, _swa_inputs, _tables

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


@pytest.mark.parametrize("B,H,Hkv,W,D,T,Tp,dtype,pos", [
    (2, 8, 2, 64, 256, 5, 5, torch.bfloat16, [200, 9]),     # 20 query rows a group
    (1, 4, 4, 130, 256, 64, 64, torch.float32, [77]),       # the longest block, a ring part cut short
    (2, 2, 1, 37, 130, 49, 3, torch.float32, [20, 500]),    # the shortest block of that kind
    (1, 2, 1, 40, 130, 48, 2, torch.bfloat16, [100]),       # and the longest of the other
    (1, 1, 1, 16, 200, 17, 1, torch.float32, [3]),
    (1, 4, 1, 1024, 256, 16, 4, torch.bfloat16, [4000]),    # 64 rows, the largest window
])
def test_heads_above_128_with_many_query_rows(B, H, Hkv, W, D, T, Tp, dtype, pos):
    from lizard_cuda.decode import swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(B, H, Hkv, W, D, T, Tp, dtype, pos, seed=D + T)
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos, pending=pend)
    assert torch.isfinite(y).all()
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_sinks_of_weight_zero_beside_masked_values(bad):
    """Sinks of -inf weigh nothing, also where an output is computed by itself because a
    value that its token does not see is not a number."""
    from lizard_cuda.decode import swa_decode_block
    q, blk, pend, meta, kr, vr, pos = _swa_inputs(2, 4, 2, 16, 64, 5, 2, torch.bfloat16, [50, 3],
                                                  seed=21)
    meta.fill_(-math.inf)
    blk[1][:, :, 4] = bad  # the last token: the four before do not see it
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos, pending=pend)
    assert torch.isfinite(y[:, :, :4]).all()
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)


@pytest.mark.parametrize("now,before", [(torch.bfloat16, torch.float32),
                                        (torch.float32, torch.bfloat16)])
def test_each_block_keeps_its_own_precision(now, before):
    """The pending block and its tables may be of another type than the block: every value
    is read as it was given."""
    from lizard_cuda.decode import swa_decode_block
    q, blk, _, meta, kr, vr, pos = _swa_inputs(2, 4, 2, 16, 64, 3, 1, now, [40, 5], seed=22,
                                               tables=now)
    pend = _swa_inputs(2, 4, 2, 16, 64, 1, 4, before, [40, 5], seed=23, tables=before)[2]
    blk = blk[:2] + _tables(pos + pend[4], 3, 64, now)
    kr0, vr0 = kr.clone(), vr.clone()
    y = swa_decode_block(q, *blk, meta, kr, vr, pos, pending=pend)
    _check_swa(y, q, blk, pend, meta, kr0, vr0, pos, kr, vr)
    # and within a block
    kr, vr = kr0.clone(), vr0.clone()
    y = swa_decode_block(q, blk[0].to(before), blk[1], blk[2].to(before), blk[3], meta, kr, vr, pos,
                         pending=pend)
    _check_swa(y, q, (blk[0].to(before), blk[1], blk[2].to(before), blk[3]), pend, meta, kr0, vr0,
               pos, kr, vr)
