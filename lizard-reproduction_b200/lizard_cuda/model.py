"""Model-level integration of the cuda backend.

to_lizard(model, ...) replaces every decoder block's self-attention of a
Hugging Face Llama model by LizardAttention with the `cuda` backend, copying
the q / k / v / o projections, as the reference's training script does
(src/train.py:35-39 with from_llama, src/lizard_attention.py:100-107). The
Lizard parameters (phi_q, phi_k, W_gamma, meta_tokens, alpha_blend) start from
the layer's own init, as in the reference.

check_kernels(api, cfg) is the reference's pre-flight check
(src/check.py:39-45) with a branch for the `cuda` backend: it loads
liblizard_cuda.so (which verifies its ABI revision) and checks that the GPU
is a compute capability 10.0 part, the one the library is built for.

greedy_generate(model, input_ids, steps) decodes with the recurrent cache
(lizard_cuda.decode): one full forward over the prompt, then one token per
step at O(1) cost per layer (the reference has no cache and would recompute
the whole sequence for every new token); GraphedDecoder replays a captured
decode step as one CUDA graph launch.

speculative_generate(model, draft, input_ids, steps) gets several tokens out of a
pass over the model's weights: a cheaper draft model proposes tokens, the model
runs them as one block against its cache and keeps the prefix that its own
probabilities accept. to_int8(model) makes such a draft of a copy of the model.
"""
import torch
import torch.nn as nn

from .decode import LizardCache
from .int8 import Int8Linear
from .layer import LizardAttention, from_llama  # noqa: F401
from .verify import verify_drafts
from . import _lib

OPTIONS = ("window", "num_meta", "feature_dim", "backend")


def to_lizard(model, window=128, num_meta=4, feature_dim=128, backend="cuda"):
    """Swap model.model.layers[i].self_attn for LizardAttention in place and
    return the model (src/train.py:35-39). The keyword arguments are the
    reference config's `lizard` section (src/config.py:10-15)."""
    options = dict(window=window, num_meta=num_meta, feature_dim=feature_dim, backend=backend)
    for block in model.model.layers:
        block.self_attn = from_llama(block.self_attn, model.config, **options)
    return model


def check_kernels(api, cfg):
    """Pre-flight check of the kernel backend named by cfg.lizard.backend.
    Returns a one-line status; raises RuntimeError when the backend cannot run
    here (the reference's check runner reports any exception as a failed check,
    src/check.py:39-45, where the triton branch asserts instead; a raised error
    also survives python -O)."""
    backend = cfg.lizard.backend
    if backend != "cuda":
        return f"skipped, backend {backend}"
    if not torch.cuda.is_available():
        raise RuntimeError("the cuda backend needs a CUDA GPU")
    lib = _lib.load()
    major, minor = torch.cuda.get_device_capability()
    if (major, minor) != (10, 0):
        raise RuntimeError(
            f"liblizard_cuda.so is built for sm_100a; this GPU is sm_{major}{minor}")
    return f"lizard_cuda ABI {lib.lz_abi_version()} on {torch.cuda.get_device_name()}"


class GraphedDecoder:
    """One greedy decode step of the whole model for a fixed batch, captured
    as a CUDA graph: a step is one graph launch instead of several hundred
    kernel launches from Python. The step reads the token and position
    buffers, advances every layer's cache in place (the cache tensors are the
    graph's static buffers) and writes the next token and position back.

    Construction runs one eager step (which also prepares every kernel's
    launch attributes) and then captures the next; `tokens` / `position`
    ([B, 1], the last token and its position) are copied into the static
    buffers. step() replays the graph and returns the new tokens [B, 1]."""

    def __init__(self, model, cache, tokens, position):
        self.model, self.cache = model, cache
        self.tok = tokens.clone()
        self.pos = position.clone()
        self._step()  # eager: the kernels' one-time setup happens outside the capture
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self._step()

    def _step(self):
        logits = self.model(self.tok, position_ids=self.pos, lizard_cache=self.cache,
                            use_cache=False).logits
        self.tok.copy_(logits[:, -1].argmax(-1, keepdim=True))
        self.pos.add_(1)

    def step(self):
        self.graph.replay()
        return self.tok


@torch.no_grad()
def greedy_generate(model, input_ids, steps, graph=False):
    """Greedy continuation of input_ids [B, L] by `steps` tokens with a
    LizardCache: the prompt runs through the full forward (which stores every
    layer's state), each new token through the layers' decode path, eagerly or
    (graph=True) as replays of a GraphedDecoder. Returns the new token ids
    [B, steps] and the cache."""
    cache = LizardCache()
    B, L = input_ids.shape
    logits = model(input_ids, lizard_cache=cache, use_cache=False, logits_to_keep=1).logits
    tokens = [logits[:, -1].argmax(-1, keepdim=True)]
    pos = torch.full((B, 1), L, dtype=torch.long, device=input_ids.device)
    if graph and steps > 2:
        dec = GraphedDecoder(model, cache, tokens[-1], pos)  # runs step 2 eagerly
        tokens.append(dec.tok.clone())
        for _ in range(2, steps):
            tokens.append(dec.step().clone())
        return torch.cat(tokens, 1), cache
    for _ in range(1, steps):
        logits = model(tokens[-1], position_ids=pos, lizard_cache=cache, use_cache=False).logits
        tokens.append(logits[:, -1].argmax(-1, keepdim=True))
        pos = pos + 1
    return torch.cat(tokens, 1), cache


INT8_LAYERS = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj",
               "lm_head")


@torch.no_grad()
def to_int8(model, names=INT8_LAYERS):
    """Replace the model's linear layers of these names by Int8Linear in place
    (weights as 8-bit codes with a scale a channel, inputs quantised token by token)
    and return the model: half the weight bytes of bf16, for inference on the GPU.
    The small layers (feature maps, gate) keep their weights."""
    for module in model.modules():
        for name, child in module.named_children():
            if name in names and isinstance(child, nn.Linear):
                setattr(module, name, Int8Linear(child))
    return model


def _draw(logits, temperature, generator):
    """One token a row of logits [B, V]: argmax at temperature 0, else by their probabilities."""
    B, V = logits.shape
    noise = torch.empty(B, V, device=logits.device).exponential_(generator=generator)
    none = logits.new_empty(B, 0, V)
    return verify_drafts(logits[:, None], none, torch.empty(B, 0, device=logits.device,
                                                            dtype=torch.long),
                         noise[:, :0], noise, temperature)[0]


@torch.no_grad()
def speculative_generate(model, draft, input_ids, steps, draft_len=4, temperature=0.0,
                         generator=None):
    """Continuation of input_ids [B, L] by `steps` tokens with drafted decoding: the
    draft model proposes draft_len tokens a round, the model checks them in one
    block and adds one of its own. At temperature 0 the tokens are the model's greedy
    ones (up to near ties: the logits of a block and of single steps differ by bf16
    roundings); otherwise they follow the model's probabilities at that temperature,
    whatever the draft. Both models are Lizard models with the same vocabulary.
    Returns the tokens [B, steps], the model's cache, settled on the tokens before
    the last one it emitted (a row may run a few tokens past `steps`), and how many
    rounds it took. A row whose logits are NaN or masked throughout gets the token -1
    there and goes on as after token 0."""
    dev, (B, L) = input_ids.device, input_ids.shape
    K = draft_len
    if not 1 <= K <= 63:
        raise ValueError(f"draft_len must be 1 .. 63, got {draft_len}")
    cache, draft_cache = LizardCache(), LizardCache()
    logits = model(input_ids, lizard_cache=cache, use_cache=False, logits_to_keep=1).logits
    draft(input_ids, lizard_cache=draft_cache, use_cache=False, logits_to_keep=1)
    last = _draw(logits[:, -1], temperature, generator)
    out = torch.zeros(B, steps + K + 1, device=dev, dtype=torch.long)
    out[:, :1] = last
    have = torch.ones(B, 1, device=dev, dtype=torch.long)
    pos = torch.full((B, 1), L, device=dev, dtype=torch.long)  # of `last`
    none = torch.zeros(B, device=dev, dtype=torch.int32)
    stand, step, rounds = none, torch.arange(K + 1, device=dev), 0
    while int(have.min()) < steps:
        block, proposals = last, []
        for i in range(K):
            proposals.append(draft(block.clamp_min(0), position_ids=pos + step[:i + 1], use_cache=False,
                                   lizard_cache=draft_cache.draft(stand if i == 0 else none),
                                   logits_to_keep=1).logits[:, -1].to(logits.dtype))
            block = torch.cat([block, _draw(proposals[-1], temperature, generator)], 1)
        # the draft's own pass over the whole block, so that its cache can keep any prefix
        fed = block.clamp_min(0)
        draft(fed, position_ids=pos + step, lizard_cache=draft_cache.draft(none),
              use_cache=False, logits_to_keep=1)
        logits = model(fed, position_ids=pos + step, lizard_cache=cache.draft(stand),
                       use_cache=False).logits
        uniforms = torch.rand(B, K, device=dev, generator=generator)
        noise = torch.empty(B, logits.shape[-1], device=dev).exponential_(generator=generator)
        tokens, accepted = verify_drafts(logits, torch.stack(proposals, 1), block[:, 1:], uniforms,
                                         noise, temperature)
        # rows that are done write their further tokens into the spare columns
        at = torch.minimum(have + step, torch.full_like(have, steps + K))
        new = step <= accepted[:, None]
        out.scatter_(1, at, torch.where(new, tokens, out.gather(1, at)))
        last = tokens.gather(1, accepted[:, None].long())
        stand = accepted + 1  # the block's first token stands in any case
        have, pos, rounds = have + stand[:, None], pos + stand[:, None], rounds + 1
    cache.settle(stand)
    return out[:, :steps], cache, rounds
