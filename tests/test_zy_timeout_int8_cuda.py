"""The bounded waits of the 8-bit products, exercised without a GPU fault: a test switch
leaves one load of a CTA's first stage out, so that nothing ever completes that stage's barrier
and every wait behind it runs out after about 2 s. The call then returns, has written
nothing, and names a wait of these kernels; after clearing the flag the next call is right.

The kernels leave with none of their copies or products in flight and their tensor memory
freed. The file is collected after the other GPU tests, which check that no wait ever
timed out."""
import pytest
import torch

from test_int8_cuda import _codes, _product, _quantize, _same

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("M,K,N,path,fused", [
    (2, 2048, 300, 0, True),      # quantised by the product, K split over clusters
    (16, 2048, 300, 1, False),    # K split over clusters
    (40, 300, 640, 1, False),     # a CTA a tile, y by TMA
    (40, 300, 641, 1, False),     # y by plain stores
    (20, 640, 128 * 300, 1, False),  # more tiles than CTAs
    (300, 1024, 520, 2, False),   # CTA pairs, y by TMA
    (300, 1024, 521, 2, False),   # y by plain stores
])
def test_a_product_that_waits_in_vain_writes_nothing(built_lib, M, K, N, path, fused):
    from lizard_cuda import _lib
    lib, p = _lib.load(), _lib.ptr
    g = torch.Generator(device=DEV).manual_seed(M + N)
    b, sb = _codes(N, K, g), torch.rand(N, generator=g, device=DEV) + 0.01
    x = torch.randn(M, K, generator=g, device=DEV)
    a, sa = _quantize(x)
    want = _product(a, sa, b, sb, None, torch.float32)
    y = torch.full((M, N), 7.0, device=DEV)
    wide = torch.zeros(M, -(-K // 16) * 16, dtype=torch.int8, device=DEV)
    wide[:, :K] = a

    def call():
        if fused:
            rc = lib.lz_int8_linear(p(x), 0, K, p(b), b.stride(0), p(sb), None, 0, p(y), 0, None, 0,
                                    M, N, K, _lib.stream_of(x))
        else:
            rc = lib.lz_int8_matmul(p(wide), wide.stride(0), p(sa), p(b), b.stride(0), p(sb), None,
                                    0, p(y), 0, None, 0, M, N, K, _lib.stream_of(x))
        _lib.check(rc, "8-bit product")
        torch.cuda.synchronize()

    assert _lib.device_timeout_flag() == 0
    old = lib.lz_int8_set_path(path)
    lib.lz_test_withhold_int8_load(1)
    try:
        call()
        flag = _lib.device_timeout_flag()
    finally:
        lib.lz_test_withhold_int8_load(0)
        _lib.clear_device_timeout_flag()
        lib.lz_int8_set_path(old)
    assert flag & 0x80000000 and 120 <= flag & 0x7fffffff <= 134
    assert (y == 7).all()
    assert _lib.device_timeout_flag() == 0
    lib.lz_int8_set_path(path)
    try:
        call()
    finally:
        lib.lz_int8_set_path(old)
    assert _same(y, want) and _lib.device_timeout_flag() == 0
