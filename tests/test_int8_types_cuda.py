"""8-bit products for activations and modules of other types than fp32 and bf16."""
import copy

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


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.bfloat16), lambda m: m.half(),
                                  lambda m: m.double(), lambda m: m.bfloat16().float(),
                                  lambda m: m.to(DEV, torch.bfloat16), copy.deepcopy])
def test_the_scale_of_a_module_survives_casts(cast):
    from lizard_cuda import Int8Linear
    torch.manual_seed(2)
    m = Int8Linear(torch.nn.Linear(100, 60, bias=False).to(DEV))
    scale = m.scale.clone()
    x = torch.randn(7, 100, device=DEV)
    want = m(x)
    m = cast(torch.nn.Sequential(m))[0]
    assert m.scale.dtype == torch.float32 and torch.equal(m.scale, scale)
    assert torch.equal(m(x), want)
    assert m.state_dict()["scale"].data_ptr() == m.scale.data_ptr()


def test_the_bias_of_a_module_keeps_a_type_that_the_product_takes():
    from lizard_cuda import Int8Linear, int8_linear
    torch.manual_seed(3)
    lin = torch.nn.Linear(100, 60).to(DEV)
    x = torch.randn(7, 100, device=DEV)
    m = Int8Linear(lin).half()
    bias = lin.bias.detach().half().float()  # the cast rounds it, as it would a linear layer's
    assert torch.equal(m(x), int8_linear(x, m.codes[:, :100], m.scale, bias))
    assert m(x.half()).dtype == torch.float16
    m = Int8Linear(lin).bfloat16()
    assert m.bias.dtype == torch.bfloat16 and m(x.bfloat16()).dtype == torch.bfloat16
