"""verify_drafts with target and draft logits of two types: each side's probabilities are
those of its logits as given, so the result is that of the same logits in fp32."""
import pytest
import torch

from test_verify_cuda import check, inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib(built_lib):
    import lizard_cuda
    lizard_cuda.load()


@pytest.mark.parametrize("target,draft", [(torch.bfloat16, torch.float32),
                                          (torch.float32, torch.bfloat16),
                                          (torch.bfloat16, torch.float16),
                                          (torch.float16, torch.bfloat16),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_two_types_of_logits(target, draft, temperature):
    from lizard_cuda import verify_drafts
    args = list(inputs(4096, 3, 50, torch.float32, 31, spread=2.5, own=0.3))
    args[0], args[1] = (args[0] + 8).to(target), (args[1] + 8).to(draft)
    tokens, accepted = verify_drafts(*args, temperature=temperature)
    want, wacc = verify_drafts(args[0].float(), args[1].float(), *args[2:], temperature=temperature)
    assert torch.equal(tokens, want) and torch.equal(accepted, wacc)
    check([a[:64] for a in args], temperature=temperature)


def test_a_draft_without_tokens_has_no_type():
    """K = 0: the empty draft's type changes nothing."""
    from lizard_cuda import verify_drafts
    args = list(inputs(9, 0, 777, torch.bfloat16, 32))
    want = verify_drafts(*args)[0]
    args[1] = args[1].float()
    assert torch.equal(verify_drafts(*args)[0], want)
