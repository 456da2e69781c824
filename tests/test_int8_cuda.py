"""8-bit products against the same arithmetic in plain torch. The integer sum is
exact (float64 holds it) and every later step rounds once in a fixed order, so
outputs have to agree bit for bit; the codes and scales too."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


def _quantize(x):
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    n = torch.full_like(top, 127)  # tensor by tensor: torch takes number / tensor by a reciprocal
    codes = torch.round(x * (n / top))
    zero = top < 4e-37
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    codes = torch.where(zero | bad, torch.zeros_like(codes), codes)
    scale = torch.where(bad, torch.full_like(top, math.nan),
                        torch.where(zero, torch.zeros_like(top), top / n))
    return codes.to(torch.int8), scale[..., 0]


def _product(a, sa, b, sb, bias, dtype):
    acc = (a.double() @ b.double().t()).to(torch.int64)
    y = acc.float() * (sa[:, None] * sb)
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype)


def _same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(
        a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))


def _codes(rows, k, g, aligned=True):
    pad = -(-k // 16) * 16 if aligned else k
    return torch.randint(-128, 128, (rows, pad), generator=g, device=DEV,
                         dtype=torch.int8)[:, :k]


@pytest.mark.parametrize("M,K,dtype", [
    (1, 1, torch.float32), (3, 7, torch.bfloat16), (5, 16, torch.bfloat16),
    (2, 1000, torch.float32), (4, 2048, torch.bfloat16), (3, 8193, torch.bfloat16),
    (2, 20000, torch.float32), (300, 129, torch.bfloat16),
])
def test_quantize_bit_for_bit(M, K, dtype):
    from lizard_cuda import int8_quantize
    g = torch.Generator(device=DEV).manual_seed(M * K)
    x = (torch.randn(M, K, generator=g, device=DEV) * 3).to(dtype)
    codes, scale = int8_quantize(x)
    want, wscale = _quantize(x)
    assert torch.equal(codes, want) and torch.equal(scale, wscale)
    assert codes.stride(0) % 16 == 0
    # a view with strides, and leading dimensions
    wide = torch.zeros(2, M, K + 5, device=DEV, dtype=dtype)
    wide[..., 3:3 + K] = x
    codes, scale = int8_quantize(wide[..., 3:3 + K])
    assert codes.shape == (2, M, K) and scale.shape == (2, M)
    assert torch.equal(codes[1], want) and torch.equal(scale[0], wscale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 5, 8, 31, 255, 1023, 2047, 2055, 4133, 9001])
def test_quantize_rows_that_start_anywhere(K, dtype):
    """Rows at every offset from 16 bytes (an odd row length runs through them), short
    rows and such that a warp, and a block, keeps in part only; padding codes are zero."""
    from lizard_cuda import int8_quantize
    g = torch.Generator(device=DEV).manual_seed(K)
    for off in (0, 1, 6):
        flat = torch.randn(off + 19 * (K + 2 - K % 2 + 1), generator=g, device=DEV).to(dtype)
        x = flat[off:].view(19, -1)[:, :K]
        codes, scale = int8_quantize(x)
        want, wscale = _quantize(x)
        assert torch.equal(codes, want) and torch.equal(scale, wscale)
        whole = codes.as_strided((19, codes.stride(0)), codes.stride())
        assert not whole[:, K:].any()


def test_quantize_rows_without_a_scale():
    from lizard_cuda import int8_linear, int8_quantize
    x = torch.randn(8, 100, device=DEV)
    x[0] = 0
    x[1] = 1e-38
    x[2] *= 1e37
    x[3, 50] = math.inf
    x[4, 99] = math.nan
    x[5, 0] = -math.inf
    x[6] = 0
    x[6, 3] = -3e38
    for dtype in (torch.float32, torch.bfloat16):
        codes, scale = int8_quantize(x.to(dtype))
        want, wscale = _quantize(x.to(dtype))
        assert torch.equal(codes, want) and _same(scale, wscale)
        y = int8_linear(x.to(dtype), want[:4], torch.ones(4, device=DEV))
        assert torch.isnan(y[3:6]).all() and not y[:2].any()


SIZES = [
    (1, 1, 1), (1, 2048, 2048), (2, 129, 300), (16, 2048, 128), (17, 100, 129), (32, 4096, 512),
    (33, 1000, 777), (64, 127, 1000), (65, 512, 257), (128, 2048, 96), (200, 1040, 384),
    (512, 128, 640), (513, 129, 255), (700, 1000, 513), (1030, 2048, 520), (2500, 384, 1032),
    (600, 16, 3), (1, 64, 20000),
]


@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_matmul_bit_for_bit(M, K, N, dtype):
    from lizard_cuda import int8_matmul
    g = torch.Generator(device=DEV).manual_seed(M + K + N)
    a, b = _codes(M, K, g), _codes(N, K, g)
    sa, sb = (torch.rand(n, generator=g, device=DEV) + 0.01 for n in (M, N))
    bias = torch.randn(N, generator=g, device=DEV).to(dtype)
    for bi in (None, bias, bias.float()):
        y = int8_matmul(a, sa, b, sb, bi, dtype=dtype)
        assert _same(y, _product(a, sa, b, sb, bi, dtype)), (M, K, N)


@pytest.mark.parametrize("path", [1, 2])
@pytest.mark.parametrize("M,K,N", [(1, 200, 300), (20, 16, 1), (100, 700, 2000), (300, 129, 257),
                                   (1000, 4096, 136), (260, 384, 5000), (3000, 65, 700),
                                   (129, 300, 40000), (290, 73, 4097), (65, 140, 323),
                                   (257, 100, 130)])
def test_both_kernels_at_any_size(M, K, N, path):
    """Few and many tokens, tiles more and fewer than the machine holds, K in one step
    or split, y that TMA can and cannot write: both kernels give the same bits."""
    from lizard_cuda import _lib, int8_matmul
    g = torch.Generator(device=DEV).manual_seed(M + K + N)
    a, b = _codes(M, K, g), _codes(N, K, g)
    sa, sb = (torch.rand(n, generator=g, device=DEV) + 0.01 for n in (M, N))
    bias = torch.randn(N, generator=g, device=DEV)
    old = _lib.load().lz_int8_set_path(path)
    try:
        for dtype in (torch.bfloat16, torch.float32):
            y = int8_matmul(a, sa, b, sb, bias, dtype=dtype)
            assert _same(y, _product(a, sa, b, sb, bias, dtype))
    finally:
        assert _lib.load().lz_int8_set_path(old) == path


@pytest.mark.parametrize("M,K,N", [(1, 130, 77), (40, 1001, 300), (800, 250, 301),
                                   # quantised by the product itself, and just not
                                   (1, 4096, 2048), (4, 4096, 140), (5, 2048, 300),
                                   (4, 999, 129), (3, 64, 20000), (2, 4097, 64), (2, 2500, 64)])
def test_linear_bit_for_bit_and_in_any_layout(M, K, N):
    from lizard_cuda import int8_linear, int8_matmul, int8_quantize
    g = torch.Generator(device=DEV).manual_seed(M + K)
    w = torch.randn(N, K, generator=g, device=DEV)
    codes, scale = int8_quantize(w)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
        xq, xs = _quantize(x)
        bias = torch.randn(N, generator=g, device=DEV)
        want = _product(xq, xs, codes, scale, bias, dtype)
        assert _same(int8_linear(x, codes, scale, bias), want)
        packed = codes.contiguous()  # rows that do not start on 16 bytes
        assert _same(int8_linear(x, packed, scale, bias), want)
        assert _same(int8_matmul(xq, xs, packed, scale, bias, dtype), want)
        assert _same(int8_linear(x.t().contiguous().t(), codes, scale, bias), want)
        other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
        assert _same(int8_linear(x, codes, scale, bias, dtype=other),
                     _product(xq, xs, codes, scale, bias, other))
    x3 = torch.randn(3, 2, K, generator=g, device=DEV)
    assert _same(int8_linear(x3, codes, scale).view(6, N),
                 int8_linear(x3.view(6, K), codes, scale))
    assert int8_linear(x3[:0], codes, scale).shape == (0, 2, N)


@pytest.mark.parametrize("M,K,N,dtype", [(4100, 2048, 1500, torch.bfloat16),
                                         (5000, 2056, 1289, torch.bfloat16),
                                         (4096, 2052, 1300, torch.float32),
                                         (20000, 4096, 256, torch.bfloat16)])
def test_many_long_rows(M, K, N, dtype):
    from lizard_cuda import int8_linear, int8_quantize
    g = torch.Generator(device=DEV).manual_seed(M)
    codes, scale = int8_quantize(torch.randn(N, K, generator=g, device=DEV))
    wide = torch.randn(M, K + 32, generator=g, device=DEV).to(dtype)
    x = wide[:, :K]  # rows further apart than they are long
    x[7] = 0
    x[M - 1, 3] = math.nan
    xq, xs = _quantize(x)
    want = _product(xq, xs, codes, scale, None, dtype)
    for _ in range(3):
        assert _same(int8_linear(x, codes, scale), want)
    assert _same(int8_linear(x.contiguous(), codes, scale), want)


@pytest.mark.parametrize("M", [3, 600])
def test_the_largest_sums_stay_exact(M):
    from lizard_cuda import int8_matmul
    K = 131071
    pad = -(-K // 16) * 16
    a = torch.full((M, pad), -128, device=DEV, dtype=torch.int8)[:, :K]
    b = torch.full((130, pad), -128, device=DEV, dtype=torch.int8)[:, :K]
    b[1::2] = 127
    one = torch.ones(M, device=DEV), torch.ones(130, device=DEV)
    y = int8_matmul(a, one[0], b, one[1], dtype=torch.float32)
    want = torch.tensor([128.0 * 128 * K, -128.0 * 127 * K], device=DEV).float().repeat(65)
    assert torch.equal(y, want.expand(M, 130))


def test_on_another_stream_and_in_a_graph():
    from lizard_cuda import int8_linear, int8_quantize
    g = torch.Generator(device=DEV).manual_seed(3)
    codes, scale = int8_quantize(torch.randn(512, 256, generator=g, device=DEV))
    x = torch.randn(4, 256, generator=g, device=DEV)
    want = int8_linear(x, codes, scale)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = int8_linear(x, codes, scale)
    s.synchronize()
    assert torch.equal(y, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int8_linear(x, codes, scale)
    x.mul_(2)  # codes stay, scales double: exactly twice the output
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, 2 * want)


def test_module_holds_codes_and_computes_as_the_function():
    from lizard_cuda import Int8Linear, int8_linear, int8_quantize
    torch.manual_seed(0)
    lin = torch.nn.Linear(100, 60).to(DEV)
    m = Int8Linear(lin)
    x = torch.randn(2, 5, 100, device=DEV)
    with torch.no_grad():
        codes, scale = int8_quantize(lin.weight)
        assert torch.equal(m(x), int8_linear(x, codes, scale, lin.bias))
        ref = lin(x)
        assert float((m(x) - ref).abs().max()) < 0.05 * float(ref.abs().max())
    assert not list(m.parameters()) and "codes" in m.state_dict()


def test_int8_refusals():
    from lizard_cuda import int8_linear, int8_matmul, int8_quantize
    x = torch.randn(4, 32, device=DEV)
    codes, scale = int8_quantize(torch.randn(8, 32, device=DEV))
    with pytest.raises(ValueError, match="weight codes"):
        int8_linear(x[:, :16], codes, scale)
    with pytest.raises(ValueError, match="scale must be fp32"):
        int8_linear(x, codes, scale[:4])
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, codes, scale, torch.zeros(7, device=DEV))
    with pytest.raises(ValueError, match="output type"):
        int8_linear(x, codes, scale, dtype=torch.float16)
    with pytest.raises(ValueError, match="a must be int8"):
        int8_matmul(x, scale, codes, scale)
    with pytest.raises(RuntimeError, match="no backward"):
        int8_linear(x.requires_grad_(), codes, scale)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        int8_quantize(torch.randn(2, 2))
    big = torch.zeros(1, 131072, device=DEV, dtype=torch.int8)
    with pytest.raises(RuntimeError, match="131071"):
        int8_matmul(big, torch.ones(1, device=DEV), big, torch.ones(1, device=DEV))
