"""GPU: packed prompts that are turned, stored and attended, samples that go on from them over common blocks, and a model that is served this way: every call's result
against its definition in 64 bits, over what the calls before it gave."""
import pytest
import torch

import paged_rows as plain
import prompt_rows
from test_gpu_paged_cache import _check_attend
from test_gpu_paged_llama import _dense_cache, _paged
from test_gpu_paged_rotate import _tables, _turned
from test_gpu_press_llama import DEV, LOGIT_ATOL, _ids, _model

pytestmark = pytest.mark.gpu


class _Shared:
    def __init__(self, cache):
        self.cache = cache

    def attend(self, *args, **kw):
        return self.cache.attend(*args, shared=True, **kw)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kind,dtype,interleaved", [("int8", torch.bfloat16, False), ("e4m3", torch.float16, True)])
@torch.no_grad()
def test_prompts_and_samples(kind, dtype, interleaved, captured):
    """Three packed prompts, of them seven samples, which move on by single tokens over a block's end and change places on the way; the steps eager or as replays of one graph."""
    from kvquant import PagedKVCache, prompt_attention
    lengths, parents, H, Hq, layers, steps = [130, 61, 320], [0, 2, 2, 1, 2, 0, 2], 2, 8, 2, 6
    N, B = sum(lengths), len(parents)
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(layers, 1, h, N, 128, generator=g).to(dtype) for h in (Hq, H, H))
    cos, sin = _tables(400, 128)
    offsets = [0, 130, 191, 511]
    first = PagedKVCache(3, H, 400, layers=layers, kind=kind, dtype=dtype)
    first.extend(lengths)
    rows = []
    for layer in range(layers):
        at = torch.tensor(offsets, dtype=torch.int32, device=DEV)
        turned, keys = first.write_rotated(layer, q[layer].to(DEV), k[layer].to(DEV), v[layer].to(DEV), cos.to(DEV), sin.to(DEV), offsets=at, interleaved=interleaved, return_keys=True)
        out, lse = prompt_attention(turned, keys, v[layer].to(DEV), offsets=at, return_lse=True)
        rows.append([])
        for s, (lo, hi) in enumerate(zip(offsets, offsets[1:])):
            n = hi - lo
            want_q = _turned(q[layer, 0, :, lo:hi], cos[:n], sin[:n], interleaved)
            want_k = _turned(k[layer, 0, :, lo:hi], cos[:n], sin[:n], interleaved, key=True)
            assert torch.equal(turned[0, :, lo:hi].cpu(), want_q) and torch.equal(keys[0, :, lo:hi].cpu(), want_k)
            want = prompt_rows.attend(want_q, want_k, v[layer, 0, :, lo:hi])
            prompt_rows.check(out[0, lo:hi].cpu(), lse[0, :, lo:hi].cpu(), *want)
            rows[layer].append((want_k, v[layer, 0, :, lo:hi]))
    batch = first.select(parents)
    first.release()
    rows = [[rows[layer][p] for p in parents] for layer in range(layers)]
    order = torch.zeros(B, dtype=torch.int64, device=DEV)
    q1, k1, v1 = (torch.zeros(layers, B, h, 1, 128, dtype=dtype, device=DEV) for h in (Hq, H, H))
    outs = []

    def step():
        batch.reorder(order)
        batch.extend(1)
        outs[:] = []
        for layer in range(layers):
            turned = batch.write_rotated(layer, q1[layer], k1[layer], v1[layer], cos_d, sin_d, interleaved=interleaved)
            outs.append((turned, batch.attend(layer, turned, shared=True)))

    cos_d, sin_d = cos.to(DEV), sin.to(DEV)
    graph = None
    places = [[0, 1, 2, 3, 4, 5, 6], [1, 1, 2, 3, 4, 0, 6], [6, 5, 4, 3, 2, 1, 0], [0, 0, 0, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5, 6], [3, 3, 2, 1, 1, 6, 5]]
    for n in range(steps):
        fresh = [torch.randn(layers, B, h, 1, 128, generator=g).to(dtype) for h in (Hq, H, H)]
        for to, x in zip((q1, k1, v1), fresh):
            to.copy_(x)
        order.copy_(torch.tensor(places[n]))
        if graph is not None:
            graph.replay()
            batch.refresh()
        else:
            step()
        at = [rows[0][p][0].shape[1] for p in places[n]]
        for layer in range(layers):
            moved = []
            for b, p in enumerate(places[n]):
                c, s = cos[at[b]:at[b] + 1], sin[at[b]:at[b] + 1]
                key = _turned(fresh[1][layer, b], c, s, interleaved, key=True)
                moved.append(tuple(torch.cat(x, dim=1) for x in ((rows[layer][p][0], key), (rows[layer][p][1], fresh[2][layer, b]))))
                assert torch.equal(outs[layer][0][b].cpu(), _turned(fresh[0][layer, b], c, s, interleaved))
            rows[layer] = moved
            turned, out = outs[layer]
            for b in range(B):
                held = [plain.held(x, kind) for x in rows[layer][b]]
                want, _, tol, _ = plain.attend(turned[b].cpu(), *held)
                tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)
                assert bool(((out[b].cpu().double() - want).abs() <= tol).all()), (n, layer, b)
        if captured and n == 1:                                         # (a record moves nothing: the next step is its first replay)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
    _check_attend(_Shared(batch), rows[0], kind, turned.cpu())
    assert batch.length.tolist() == [x.shape[1] for x, _ in rows[0]]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@torch.inference_mode()
def test_a_model_s_samples_and_beams(kind):
    """The cache's own switches: prompts by the kernel, steps over common blocks; samples of two prompts, then beams that change places."""
    from kvquant import attention_patch
    model = _model(21)
    ids = torch.cat([_ids(150, 40), _ids(150, 41)])
    logits = []
    for cache in (_paged(model.config, kind, shared=True, native_prompt=True), _dense_cache(model.config, kind)):
        before = dict(attention_patch.paged_counts)
        got = [model(input_ids=ids, past_key_values=cache).logits.float()]
        cache.batch_repeat_interleave(4)
        g = torch.Generator().manual_seed(2)
        for step in range(30):                                          # over a block's end
            if step % 3 == 2:
                cache.reorder_cache(torch.cat([torch.randint(0, 4, (4,), generator=g), 4 + torch.randint(0, 4, (4,), generator=g)]).to(DEV))
            got.append(model(input_ids=torch.randint(1, 1000, (8, 1), generator=g).to(DEV), past_key_values=cache).logits.float())
        got.append(model(input_ids=_ids(8 * 20, 42).view(8, 20), past_key_values=cache).logits.float())            # (too many queries for common blocks)
        logits.append(got)
        if hasattr(cache, "pool"):
            assert cache.pool.shares and cache.pool._plan is not None
            assert attention_patch.paged_counts["prompt"] - before["prompt"] == 2 and attention_patch.paged_counts["paged"] - before["paged"] == 2 * 31
    for a, b in zip(*logits):
        assert (a - b).abs().max().item() < LOGIT_ATOL


@torch.inference_mode()
def test_a_padded_prompt_and_a_pool_that_grows():
    model = _model(22)
    ids = torch.cat([_ids(200, 43), _ids(200, 44), _ids(200, 45)])
    attend = torch.ones(3, 200, dtype=torch.long, device=DEV)
    attend[0, :77] = 0
    attend[2, :130] = 0
    logits = []
    for cache in (_paged(model.config, shared=True, native_prompt=True), _dense_cache(model.config, "int8")):
        mask = attend
        got = [model(input_ids=ids, attention_mask=mask, past_key_values=cache).logits.float()[attend.bool()]]
        pages = getattr(getattr(cache, "pool", None), "pages", None)
        for step, n in enumerate((1, 400, 1)):
            mask = torch.cat([mask, torch.ones(3, n, dtype=torch.long, device=DEV)], dim=1)
            got.append(model(input_ids=_ids(n, 50 + step).expand(3, n), attention_mask=mask, past_key_values=cache).logits.float().reshape(-1, 1000))
        logits.append(torch.cat(got))
        if pages is not None:
            assert cache.pool.pages > pages and cache.pool.shares
    assert (logits[0] - logits[1]).abs().max().item() < LOGIT_ATOL


@torch.inference_mode()
def test_capped_windowed_and_padded_prompts_of_a_model():
    """The patched function as a model's layers call it, with a prompt that the cache holds: in 16 bits, under the cap as well."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS
    model = _model(23, layers=1)
    module, attention = model.model.layers[0].self_attn, ALL_ATTENTION_FUNCTIONS["sdpa"]
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, 2, 150, 128, generator=g).half() for _ in range(2))
    q = (3 * torch.randn(1, 4, 150, 128, generator=g)).half()
    i, j = torch.arange(150)[:, None], torch.arange(150)
    for mask, kw, how in ((None, {}, {}), (None, dict(softcap=20.0), dict(cap=20.0)), ((j <= i) & (j > i - 50), dict(sliding_window=50, scaling=0.2), dict(window=50, scaling=0.2)),
                          ((j <= i) & (j >= 30), dict(softcap=5.0), dict(cap=5.0, start=30))):
        cache = _paged(model.config, native_prompt=True)
        keys, values = cache.update(k.to(DEV), v.to(DEV), 0)
        out, _ = attention(module, q.to(DEV), keys, values, None if mask is None else mask[None, None].to(DEV), **kw)
        want, _, tol, _ = prompt_rows.attend(q[0], k[0], v[0], **how)
        assert bool(((out[0].cpu().double() - want).abs() <= tol).all())
        with pytest.raises(RuntimeError, match="paged cache"):
            attention(module, q.to(DEV), keys, values, None, dropout=0.1)
        with pytest.raises(RuntimeError, match="newest tokens alone"):
            keys + 1


@torch.no_grad()
def test_offsets_that_pass_32_bits():
    """Tensors of more than 2^32 bytes and 2^31 elements: their last tokens, a prompt's and a step's."""
    from kvquant import PagedKVCache, prompt_attention
    N, Hq, dtype = 540001, 32, torch.bfloat16
    q = torch.zeros(1, N, Hq, 128, dtype=dtype, device=DEV).transpose(1, 2)
    k, v = (torch.zeros(1, N, 1, 128, dtype=dtype, device=DEV).transpose(1, 2) for _ in range(2))
    g = torch.Generator().manual_seed(9)
    ends = [torch.randn(1, h, 300, 128, generator=g).to(dtype) for h in (Hq, 1, 1)]
    for t, x in zip((q, k, v), ends):
        t[:, :, -300:] = x.to(DEV)
    cos, sin = torch.zeros(N, 64), torch.zeros(N, 64)
    angles = torch.arange(N - 300, N, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    cos[-300:], sin[-300:] = angles.cos().float(), angles.sin().float()
    cache = PagedKVCache(1, 1, N + 1, dtype=dtype)
    cache.extend(N)
    turned, keys = cache.write_rotated(0, q, k, v, cos.to(DEV), sin.to(DEV), offsets=torch.tensor([0, N], dtype=torch.int32, device=DEV), return_keys=True)
    want_q, want_k = _turned(ends[0][0], cos[-300:], sin[-300:], False), _turned(ends[1][0], cos[-300:], sin[-300:], False, key=True)
    assert torch.equal(turned[0, :, -300:].cpu(), want_q) and torch.equal(keys[0, :, -300:].cpu(), want_k)
    out, lse = prompt_attention(turned, keys, v, window=64, return_lse=True)
    prompt_rows.check(out[0, -200:].cpu(), lse[0, :, -200:].cpu(), *prompt_rows.attend(want_q[:, -200:], want_k, ends[2][0], window=64))
    del q, k, v, turned, keys, out, lse, cache
    # pages of the last of many layers
    cache = PagedKVCache(1, 8, 700, layers=10, pages=9000, kind="int8", dtype=dtype)
    assert cache.k_codes.numel() > 2 ** 32
    k, v = (torch.randn(1, 8, 600, 128, generator=g).to(dtype) for _ in range(2))
    q = torch.randn(4, 16, 1, 128, generator=g).to(dtype)
    cache.extend(600)
    cache.write(9, k.to(DEV), v.to(DEV))
    samples = cache.select([0, 0, 0, 0])
    out = samples.attend(9, q.to(DEV), shared=True).cpu().double()
    held = [plain.held(x[0], "int8") for x in (k, v)]
    for b in range(4):
        want, _, tol, _ = plain.attend(q[b], *held)
        assert bool(((out[b] - want).abs() <= tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol)).all())
