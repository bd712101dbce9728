"""GPU: a small random-init model whose attention caps its scores (Gemma 2's form: caps, sliding windows in every other layer) over `kvquant.PagedCache`, against the same
model with plain attention over a dense cache that holds what the paged one is defined to hold."""
import pytest
import torch

import paged_rows as plain
from test_gpu_press_llama import DEV, LOGIT_ATOL, _ids

pytestmark = pytest.mark.gpu


def _model(implementation, cap=2.0):
    from transformers import Gemma2Config, Gemma2ForCausalLM
    torch.manual_seed(5)
    cfg = Gemma2Config(hidden_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=1024, vocab_size=1000,
                       max_position_embeddings=1024, query_pre_attn_scalar=128, attn_logit_softcapping=cap, sliding_window=96, attn_implementation=implementation)
    model = Gemma2ForCausalLM(cfg)
    with torch.no_grad():                                    # (scores of a few units, which the cap bears on: 2.0 changes logits by 2 and more)
        for layer in model.model.layers:
            for proj, by in (("q_proj", 3), ("k_proj", 3), ("v_proj", 2), ("o_proj", 2)):
                getattr(layer.self_attn, proj).weight.mul_(by)
    return model.to(device=DEV, dtype=torch.float16).eval()


def _dense(config):
    """A `DynamicCache` that hands out, from the prompt on, what the paged cache holds."""
    from transformers import DynamicCache
    from transformers.cache_utils import DynamicLayer

    class Layer(DynamicLayer):
        def update(self, key_states, value_states, *args, **kwargs):
            return tuple(plain.to_type(torch.stack([plain.held(row, "int8") for row in x.cpu()]), x.dtype).to(DEV)
                         for x in super().update(key_states, value_states, *args, **kwargs))

    cache = DynamicCache()
    cache.layers = [Layer() for _ in range(config.num_hidden_layers)]
    return cache


@torch.inference_mode()
def test_a_capped_model_is_capped_from_the_prompt_on():
    from kvquant import PagedCache
    ids, forced = _ids(150, 5), _ids(45, 6)[0]
    got = {}
    for name, cap in (("sdpa", 2.0), ("eager", 2.0), ("eager", None)):
        model = _model(name, cap)
        cache = PagedCache(model.config) if name == "sdpa" else _dense(model.config)
        out = [model(input_ids=ids, past_key_values=cache).logits[0]]
        out += [model(input_ids=t.view(1, 1), past_key_values=cache).logits[0] for t in forced[:16]]
        out += [model(input_ids=forced[None, 16:], past_key_values=cache).logits[0]]
        got[name, cap] = torch.cat(out).float()
    off = (got["sdpa", 2.0] - got["eager", 2.0]).abs()
    assert off.max().item() < LOGIT_ATOL, (off[:150].max().item(), off[150:].max().item())
    assert (got["eager", 2.0] - got["eager", None]).abs().max().item() > 10 * LOGIT_ATOL        # (the cap is something that would be missed)


@torch.inference_mode()
def test_a_capped_model_with_padding_in_front():
    from kvquant import PagedCache
    ids = torch.cat([_ids(130, 7), _ids(130, 8)])
    keep = torch.ones(2, 130, dtype=torch.long, device=DEV)
    keep[1, :71] = 0
    got = {}
    for name in ("sdpa", "eager"):
        model = _model(name)
        cache, mask = PagedCache(model.config) if name == "sdpa" else _dense(model.config), keep
        out = [model(input_ids=ids, attention_mask=mask, past_key_values=cache).logits]
        for n in (1, 5, 1):
            mask = torch.cat([mask, torch.ones(2, n, dtype=torch.long, device=DEV)], dim=1)
            out.append(model(input_ids=_ids(n, 20 + n).expand(2, n), attention_mask=mask, past_key_values=cache).logits)
        got[name] = torch.cat(out, dim=1).float()
    off = (got["sdpa"] - got["eager"]).abs()
    assert off[0].max().item() < LOGIT_ATOL and off[1, 71:].max().item() < LOGIT_ATOL


@torch.inference_mode()
def test_a_cap_that_only_the_call_names():
    """The prompt of a call with `softcap`, whatever the model's configuration says, goes to the pages' attention."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    from test_gpu_press_llama import _model as _llama
    from kvquant import PagedCache
    model = _llama(14, layers=1)
    cache = PagedCache(model.config)
    g = torch.Generator().manual_seed(3)
    k, v, q = (torch.randn(1, h, 140, 128, generator=g).half() for h in (2, 2, 4))
    keys, values = cache.update(k.to(DEV), v.to(DEV), 0)
    out, _ = ALL_ATTENTION_FUNCTIONS["sdpa"](model.model.layers[0].self_attn, q.to(DEV), keys, values, None, softcap=1.0, scaling=0.3)
    want, _, tol, _ = plain.attend(q[0], plain.held(k[0], "int8"), plain.held(v[0], "int8"), cap=1.0, scaling=0.3)
    assert ((out[0].cpu().double() - want).abs() <= tol + 2.0 ** -11 * (want.abs() + tol)).all()
