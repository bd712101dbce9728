"""GPU: a small random-init Llama over `kvquant.PagedCache`, against the same model over a dense cache that holds what the paged one is defined to hold
(tests/paged_rows.py): greedy steps, questions, rewinds, beams, padded batches, soft caps and sliding windows."""
import pytest
import torch

import paged_rows as plain
from test_gpu_press_llama import DEV, LOGIT_ATOL, _ids, _model

pytestmark = pytest.mark.gpu


def _dense_cache(config, kind):
    """A `DynamicCache` whose layers keep the model's keys and values and hand out, behind the prompt, what the paged cache holds of them."""
    from transformers import DynamicCache
    from transformers.cache_utils import DynamicLayer

    class Layer(DynamicLayer):
        def update(self, key_states, value_states, *args, **kwargs):
            first = self.get_seq_length() == 0
            keys, values = super().update(key_states, value_states, *args, **kwargs)
            if first:
                return keys, values
            return tuple(plain.to_type(torch.stack([plain.held(row, kind) for row in x.cpu()]), x.dtype).to(DEV) for x in (keys, values))

        def crop(self, tokens_to_remove):
            n = self.get_seq_length() - abs(tokens_to_remove)
            self.keys, self.values = (torch.stack([plain.cut(row, n, kind) for row in x.cpu()]).to(DEV) for x in (self.keys, self.values))

    cache = DynamicCache(config=config)
    cache.layers = [Layer() for _ in cache.layers]
    return cache


def _paged(config, kind="int8", **kw):
    from kvquant import PagedCache
    return PagedCache(config, kind=kind, **kw)


@pytest.mark.parametrize("kind,dtype", [("int8", torch.float16), ("e4m3", torch.float16), ("int8", torch.bfloat16)])
@torch.inference_mode()
def test_steps_question_and_rewind(kind, dtype):
    from kvquant import attention_patch
    model = _model(3).to(dtype)
    ids = _ids(300, 5)
    forced = _ids(40, 6)[0]
    logits = {}
    for name in ("paged", "dense"):
        cache = _paged(model.config, kind) if name == "paged" else _dense_cache(model.config, kind)
        before = attention_patch.paged_counts["paged"]
        got = [model(input_ids=ids, past_key_values=cache).logits[0, -1]]
        got += [model(input_ids=t.view(1, 1), past_key_values=cache).logits[0, -1] for t in forced[:25]]
        got += list(model(input_ids=forced[None, :29], past_key_values=cache).logits[0])             # a question: 300 + 25 + 29 tokens
        assert cache.get_seq_length() == 354
        cache.crop(-34)                                                                           # back to 320, a block's end, and to 310 inside it
        cache.crop(-10)
        assert cache.get_seq_length() == 310
        got += [model(input_ids=t.view(1, 1), past_key_values=cache).logits[0, -1] for t in forced[25:]]
        logits[name] = torch.stack(got).float()
        if name == "paged":
            assert attention_patch.paged_counts["paged"] - before == 2 * (25 + 1 + 15)
    assert torch.isfinite(logits["paged"]).all()
    assert (logits["paged"] - logits["dense"]).abs().max().item() < LOGIT_ATOL * (8 if dtype == torch.bfloat16 else 1)
    # the first logits are the prompt's own: the same attention on the same numbers
    assert torch.equal(logits["paged"][0], logits["dense"][0])


@torch.inference_mode()
def test_beams_are_forked_rows():
    """Beams that change places at every step, some dropped and some doubled, across the ends of blocks."""
    model = _model(7)
    ids = torch.cat([_ids(120, 8), _ids(120, 9)]).repeat_interleave(3, dim=0)
    logits = []
    for cache in (_paged(model.config), _dense_cache(model.config, "int8")):
        model(input_ids=ids, past_key_values=cache)
        g = torch.Generator().manual_seed(1)
        got = []
        for step in range(20):
            parents = torch.cat([torch.randint(0, 3, (3,), generator=g), 3 + torch.randint(0, 3, (3,), generator=g)])
            cache.reorder_cache(parents.to(DEV))
            tokens = torch.randint(1, 1000, (6, 1), generator=g).to(DEV)
            got.append(model(input_ids=tokens, past_key_values=cache).logits[:, -1].float())
        logits.append(torch.stack(got))
    assert (logits[0] - logits[1]).abs().max().item() < LOGIT_ATOL


@torch.inference_mode()
def test_beam_search():
    """`generate` over the paged cache: the scores that it returns are those of its sequences, attended from scratch."""
    model = _model(7)
    model.generation_config.pad_token_id = 0
    ids = torch.cat([_ids(150, 8), _ids(150, 9)])
    cache = _paged(model.config)
    run = model.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=cache, num_beams=3, do_sample=False, max_new_tokens=70, min_new_tokens=70,
                         length_penalty=1.0, return_dict_in_generate=True, output_scores=True)
    assert run.sequences.shape == (2, 220)
    logp = model(input_ids=run.sequences).logits[:, 149:-1].float().log_softmax(-1)
    want = logp.gather(-1, run.sequences[:, 150:, None])[..., 0].sum(-1) / 70
    assert (run.sequences_scores - want).abs().max().item() < LOGIT_ATOL
    # beams share the blocks that they have in common: two prompts of two full blocks, and what three beams added
    assert cache.pool.batch == 6 and int((cache.pool.refs > 0).sum()) <= 2 * 2 + 6 * 2 and int(cache.pool.refs.max()) <= 3


@torch.inference_mode()
def test_padded_batch():
    """Rows padded in front: the mask becomes where each row starts."""
    model = _model(9)
    ids = torch.cat([_ids(200, 10), _ids(200, 11), _ids(200, 12)])
    attend = torch.ones(3, 200, dtype=torch.long, device=DEV)
    attend[0, :77] = 0
    attend[2, :130] = 0
    logits = []
    for cache in (_paged(model.config), _dense_cache(model.config, "int8")):
        got, mask = [], attend
        model(input_ids=ids, attention_mask=mask, past_key_values=cache)
        for step, n in enumerate((1, 1, 6, 1)):
            mask = torch.cat([mask, torch.ones(3, n, dtype=torch.long, device=DEV)], dim=1)
            got.append(model(input_ids=_ids(n, 20 + step).expand(3, n), attention_mask=mask, past_key_values=cache).logits.float())
        logits.append(torch.cat(got, dim=1))
    assert (logits[0] - logits[1]).abs().max().item() < LOGIT_ATOL


@torch.inference_mode()
def test_rows_are_repeated_selected_and_reset():
    model = _model(11)
    ids = torch.cat([_ids(140, 13), _ids(140, 14)])
    logits = []
    for cache in (_paged(model.config), _dense_cache(model.config, "int8")):
        model(input_ids=ids, past_key_values=cache)
        cache.batch_repeat_interleave(3)
        got = [model(input_ids=_ids(6, 15).view(6, 1), past_key_values=cache).logits[:, -1]]
        cache.batch_select_indices(torch.tensor([4, 0, 5], device=DEV))
        got += [model(input_ids=_ids(3 * 60, 16).view(3, 60), past_key_values=cache).logits.reshape(-1, 1000)]
        cache.reorder_cache(torch.tensor([2, 2, 0], device=DEV))
        got += [model(input_ids=_ids(3, 17).view(3, 1), past_key_values=cache).logits[:, -1]]
        logits.append(torch.cat(got).float())
    assert (logits[0] - logits[1]).abs().max().item() < LOGIT_ATOL
    cache = _paged(model.config)
    first = model(input_ids=ids, past_key_values=cache).logits
    cache.reset()
    assert cache.get_seq_length() == 0
    assert torch.equal(model(input_ids=ids[:1].expand(4, -1), past_key_values=cache).logits[0], model(input_ids=ids[:1].expand(4, -1)).logits[0])
    assert cache.pool.batch == 4 and first.shape[0] == 2


@torch.inference_mode()
def test_the_pool_grows_with_the_rows():
    model = _model(13, layers=1)
    cache = _paged(model.config)
    model(input_ids=_ids(70, 18), past_key_values=cache)
    pages = cache.pool.pages
    for n in range(6):
        model(input_ids=_ids(200, 30 + n), past_key_values=cache)
    assert cache.pool.pages > pages and cache.get_seq_length() == 1270 == cache.pool.refresh()[0]
    assert int((cache.pool.refs > 0).sum()) == 1270 // 64
    with pytest.raises(ValueError, match="max_tokens"):
        model(input_ids=_ids(3000, 1), past_key_values=cache)


@torch.inference_mode()
def test_soft_cap_and_sliding_window_of_the_model():
    """What a model's attention passes on: the patched function is called as its layers call it."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    model = _model(14, layers=1)
    cache = _paged(model.config)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, 2, 200, 128, generator=g).half() for _ in range(2))
    cache.update(k[:, :, :190].to(DEV), v[:, :, :190].to(DEV), 0)
    q = (3 * torch.randn(1, 4, 10, 128, generator=g)).half()
    keys, values = cache.update(k[:, :, 190:].to(DEV), v[:, :, 190:].to(DEV), 0)
    attention = ALL_ATTENTION_FUNCTIONS["sdpa"]
    module = model.model.layers[0].self_attn
    i, j = torch.arange(190, 200)[:, None], torch.arange(200)
    held = [plain.held(x[0], "int8") for x in (k, v)]
    for mask, kw, how in ((None, {}, {}), (None, dict(softcap=20.0), dict(cap=20.0)), (None, dict(sliding_window=50, scaling=0.2), dict(window=50, scaling=0.2)),
                          ((j <= i)[None, None], {}, {}), (((j <= i) & (j > i - 50))[None, None], dict(sliding_window=50), dict(window=50)),
                          (torch.where((j <= i) & (j >= 30), 0.0, torch.finfo(torch.float16).min).half()[None, None], {}, dict(starts=torch.tensor(30)))):
        out, _ = attention(module, q.to(DEV), keys, values, None if mask is None else mask.to(DEV), **kw)
        want, _, tol, _ = plain.attend(q[0], *held, **how)
        assert ((out[0].cpu().double() - want).abs() <= tol + 2.0 ** -11 * (want.abs() + tol)).all()
    holes = (j <= i)[None, None].clone()
    holes[..., 60] = False
    for mask, kw in ((holes, {}), ((j < 200).expand(10, 200)[None, None], {}), (None, dict(dropout=0.1)), (None, dict(s_aux=torch.zeros(4)))):
        with pytest.raises(RuntimeError, match="paged cache"):
            attention(module, q.to(DEV), keys, values, None if mask is None else mask.to(DEV), **kw)


def test_refusals():
    from transformers import LlamaConfig
    from kvquant import PagedCache
    base = dict(hidden_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128)
    for change, how in ((dict(head_dim=64), {}), ({}, dict(kind="int4")), (dict(attn_implementation="eager"), {})):
        with pytest.raises(ValueError):
            PagedCache(LlamaConfig(**dict(dict(base, attn_implementation="sdpa"), **change)), **how)
    cache = PagedCache(LlamaConfig(**base, attn_implementation="sdpa"))
    with pytest.raises(NotImplementedError):
        cache.layers[0].crop(-1)
