"""8-bit products for activations and modules of other types than fp32 and bf16."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("M", [1, 40])
def test_the_output_has_the_type_of_x(dtype, M):
    """Computed in fp32, given back in x's type; an asked-for type stays the one asked for."""
    from lizard_cuda import int8_linear, int8_quantize
    g = torch.Generator(device=DEV).manual_seed(M)
    codes, scale = int8_quantize(torch.randn(72, 100, generator=g, device=DEV))
    x = torch.randn(M, 100, generator=g, device=DEV).to(dtype)
    want = int8_linear(x.float(), codes, scale)
    y = int8_linear(x, codes, scale)
    assert y.dtype == dtype and torch.equal(y, want.to(dtype))
    for other in (torch.float32, torch.bfloat16):
        y = int8_linear(x, codes, scale, dtype=other)
        assert torch.equal(y, int8_linear(x.float(), codes, scale, dtype=other))
    assert int8_linear(x[:0], codes, scale).dtype == dtype


@pytest.mark.parametrize("bias", [True, False])
def test_a_module_made_of_a_half_layer(bias):
    from lizard_cuda import Int8Linear, int8_linear, int8_quantize
    torch.manual_seed(1)
    lin = torch.nn.Linear(100, 60, bias=bias).to(DEV).half()
    m = Int8Linear(lin)
    x = torch.randn(2, 5, 100, device=DEV).half()
    with torch.no_grad():
        codes, scale = int8_quantize(lin.weight)
        want = int8_linear(x.float(), codes, scale, lin.bias.float() if bias else None).half()
        y = m(x)
    assert y.dtype == torch.float16 and torch.equal(y, want)
