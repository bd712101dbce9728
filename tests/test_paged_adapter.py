"""What the `transformers` side of the paged 8-bit cache passes on, and what it refuses: on the CPU, over a stand-in for the cache itself."""
import pytest
import torch
from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS


class _Pool:
    """Stands for a `PagedKVCache`: notes what it is asked."""
    batch = 1

    def __init__(self):
        self.asked = []

    def attend(self, index, query, **how):
        self.asked.append(how)
        return torch.zeros(query.shape[0], query.shape[2], query.shape[1], 128)


class _Module(torch.nn.Module):
    layer_idx = 0
    num_key_value_groups = 2


def _tagged(n=9, L=3):
    """Keys and values marked as the cache marks L new tokens of n."""
    pool = _Pool()
    k, v = (torch.zeros(1, 2, L, 128) for _ in range(2))
    k._odmkv_paged = (pool, 0, n)
    return pool, k, v


def _sdpa():
    from kvquant.attention_patch import patch_attention_functions
    patch_attention_functions()
    return ALL_ATTENTION_FUNCTIONS["sdpa"]


REFUSED = {"position_bias": dict(position_bias=torch.zeros(1, 4, 3, 9)), "is_causal": dict(is_causal=False), "head_mask": dict(head_mask=torch.ones(4)),
           "sinks": dict(s_aux=torch.zeros(4)), "some other bias": dict(alibi=torch.zeros(4, 9)), "a mask by another name": dict(block_mask=object()),
           "a mask of another kind": dict(extra_mask=torch.ones(3, 9, dtype=torch.bool)), "packed rows": dict(cu_seq_lens_q=torch.tensor([0, 2, 3])),
           "a score function": dict(score_mod=lambda s: s), "dropout": dict(dropout=0.1)}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_what_the_pages_cannot_answer_is_refused(name):
    pool, k, v = _tagged()
    with pytest.raises(RuntimeError, match="cannot be answered from the paged cache"):
        _sdpa()(_Module(), torch.zeros(1, 4, 3, 128), k, v, None, **REFUSED[name])
    assert not pool.asked


def test_a_module_that_is_not_causal_is_refused():
    pool, k, v = _tagged()
    module = _Module()
    module.is_causal = False
    with pytest.raises(RuntimeError, match="cannot be answered from the paged cache"):
        _sdpa()(module, torch.zeros(1, 4, 3, 128), k, v, None)
    # one token sees all there is either way, and a mask says itself what is seen
    pool, k, v = _tagged(L=1)
    _sdpa()(module, torch.zeros(1, 4, 1, 128), k, v, None, is_causal=False)
    pool, k, v = _tagged()
    mask = (torch.arange(9) <= torch.arange(6, 9)[:, None])[None, None]
    _sdpa()(module, torch.zeros(1, 4, 3, 128), k, v, mask)
    assert pool.asked[0]["starts"] is None


def test_what_does_not_bear_on_the_answer_is_passed_over():
    pool, k, v = _tagged()
    _sdpa()(_Module(), torch.zeros(1, 4, 3, 128), k, v, None, scaling=0.5, softcap=20.0, sliding_window=7, position_bias=None, is_causal=True, head_mask=None,
            position_ids=torch.arange(6, 9)[None], cache_position=torch.arange(6, 9), use_cache=True, output_attentions=False)
    assert pool.asked == [dict(scaling=0.5, softcap=20.0, window=7, starts=None)]


def test_keys_that_lose_their_mark_are_refused():
    """Whoever computes with the newest tokens as if they were all: a cast, a copy, another attention function, attention inside the model."""
    from transformers.models.llama.modeling_llama import eager_attention_forward
    from kvquant.hf_cache import paged_tokens
    pool, q = _Pool(), torch.zeros(1, 4, 3, 128)
    k, v = paged_tokens(torch.zeros(1, 2, 3, 128), torch.zeros(1, 2, 3, 128), (pool, 0, 9))
    for call in (lambda: k.half(), lambda: k.to(torch.float16), lambda: k.clone(), lambda: k.transpose(1, 2).contiguous(), lambda: k[:, :, 1:], lambda: q[:, :2] @ k.transpose(2, 3),
                 lambda: torch.cat([k, k], dim=2), lambda: torch.matmul(q[:, :2], v), lambda: v.float().half(), lambda: k.repeat_interleave(2, dim=1), lambda: k + 1,
                 lambda: torch.nn.functional.scaled_dot_product_attention(q[:, :2], k, v), lambda: v.cpu().numpy(),
                 lambda: eager_attention_forward(_Module(), q, k, v, None, 1.0)):
        with pytest.raises(RuntimeError, match="PagedCache"):
            call()
    # looks, and steps that change nothing, leave them as they are
    assert k.shape == (1, 2, 3, 128) and k.dtype == torch.float32 and k.device.type == "cpu" and k.dim() == 4 and k.size(2) == 3 and k.stride(3) == 1 and not k.is_cuda
    assert k.contiguous() is k and k.to(torch.float32) is k and v.float() is v
    _sdpa()(_Module(), q, k.contiguous(), v, None)
    assert len(pool.asked) == 1


def test_rows_as_the_kernels_take_them():
    """Strides of dimensions of one mean nothing; what cannot be read 16 bytes at a time is copied."""
    from kvquant import PagedKVCache
    fits = PagedKVCache._rows_ok
    whole = torch.arange(2 * 4 * 6 * 256, dtype=torch.float16).view(2, 4, 6, 256)
    odd = torch.arange(20000, dtype=torch.float16)
    ok = [whole[..., :128], whole[:, :, 1:2, 128:], whole.transpose(1, 2)[..., :128], whole[:1, :1, :1, :128].expand(2, 4, 5, 128), torch.zeros(2, 4, 0, 128).half()]
    single = [odd.as_strided((2, 4, 1, 128), (1024, 128, 3, 1)), odd.as_strided((1, 4, 2, 128), (7, 128, 512, 1)), odd.as_strided((1, 1, 1, 128), (1, 5, 9, 1)),
              odd.as_strided((2, 1, 3, 128), (1024, 130, 256, 1))]
    copied = [odd.as_strided((2, 4, 1, 128), (1028, 128, 3, 1)), odd[1:].as_strided((2, 2, 2, 128), (512, 256, 128, 1)), whole[..., :128].transpose(2, 3).contiguous().transpose(2, 3),
              odd[1:].as_strided((1, 1, 1, 128), (3, 5, 7, 1))]
    for i, t in enumerate(ok + single + copied):
        f = fits(t)
        assert torch.equal(f, t), i
        assert f.stride(3) == 1 and not any(s % 8 for s in f.stride()[:3]) and f.data_ptr() % 16 == 0, (i, f.stride())
        assert (f.data_ptr() == t.data_ptr()) or i >= len(ok + single), i


def test_a_negative_limit_of_a_row_is_refused():
    import ctypes as C
    from kvquant._lib import Pages, lib
    p = Pages(2, 3, 4, 10, 5, 0, 0, *[4096] * 12, -1)
    assert lib.odmkv_pages_init(C.byref(p), None) == -1 and "shape" in lib.odmkv_last_error().decode()


def _mask(B, L, k_len, starts, window=None, dtype=torch.bool):
    i, j = torch.arange(k_len - L, k_len)[:, None], torch.arange(k_len)
    open_ = (j <= i) & (j >= torch.tensor(starts)[:, None, None])
    if window is not None:
        open_ = open_ & (j > i - window)
    open_ = open_[:, None]
    return open_ if dtype == torch.bool else torch.where(open_, torch.zeros((), dtype=dtype), torch.full((), torch.finfo(dtype).min, dtype=dtype))


@pytest.mark.parametrize("look", [1 << 24, 64, 1])
@pytest.mark.parametrize("dtype", [torch.bool, torch.float16, torch.float32])
def test_masks_are_read_piece_by_piece(dtype, look, monkeypatch):
    from kvquant import attention_patch
    monkeypatch.setattr(attention_patch, "_LOOK", look)
    starts_of = attention_patch._paged_starts
    assert starts_of(_mask(2, 5, 20, [0, 0], dtype=dtype), 2, 5, 20, None, 0) is None
    assert starts_of(_mask(3, 5, 20, [0, 7, 17], dtype=dtype), 3, 5, 20, None, 0).tolist() == [0, 7, 17]
    assert starts_of(_mask(3, 20, 20, [0, 7, 17], dtype=dtype), 3, 20, 20, None, 0).tolist() == [0, 7, 17]        # (queries before a row's start see nothing)
    assert starts_of(_mask(1, 5, 20, [3], dtype=dtype), 4, 5, 20, None, 0).tolist() == [3] * 4
    assert starts_of(_mask(2, 5, 20, [0, 14], window=4, dtype=dtype), 2, 5, 20, 4, 0).tolist() == [0, 14]
    assert starts_of(_mask(2, 5, 20, [0, 9], window=4, dtype=dtype), 2, 5, 20, 4, 0) is None                      # (before every query's window)
    for l, at in ((0, 3), (4, 10), (2, 17)):
        wrong = _mask(2, 5, 20, [0, 0], dtype=dtype)
        wrong[1, 0, l, at] = torch.finfo(dtype).min if dtype != torch.bool and wrong[1, 0, l, at] == 0 else 0 if dtype != torch.bool else not wrong[1, 0, l, at]
        assert starts_of(wrong, 2, 5, 20, None, 0) is False
    if dtype != torch.bool:
        biased = _mask(1, 5, 20, [0], dtype=dtype)
        biased[0, 0, 1, 2] = -3.0
        assert starts_of(biased, 1, 5, 20, None, 0) is False


def test_a_look_at_a_mask_serves_the_layers_above_and_keeps_nothing():
    import gc
    import weakref
    pool, k, v = _tagged()
    pool._looked = {}
    mask = _mask(1, 3, 9, [2])
    modules = [_Module() for _ in range(3)]
    for i, module in enumerate(modules):
        module.layer_idx = i
        _sdpa()(module, torch.zeros(1, 4, 3, 128), k, v, mask)
    starts = [how["starts"] for how in pool.asked]
    assert starts[0].tolist() == [2] and starts[1] is starts[0] and starts[2] is starts[0]
    mask[0, 0, :, 2] = False                              # (written to between forwards: looked at again)
    _sdpa()(modules[1], torch.zeros(1, 4, 3, 128), k, v, mask)
    assert pool.asked[-1]["starts"].tolist() == [3]
    gone = weakref.ref(mask)
    del mask
    gc.collect()
    assert gone() is None


def test_a_cap_too_small_for_32_bits_is_refused():
    import ctypes as C
    from kvquant._lib import Attend, Pages, lib
    pages = Pages(2, 3, 4, 10, 5, 0, 0, *[4096] * 12)
    a = Attend(C.pointer(pages), 4096, 1024, 128, 1024, 4096, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 8, 0, 100, 0.1, 0.0)
    for cap in (1e-38, 2.0 ** -101, 1e-45):
        a.cap = cap
        assert lib.odmkv_pages_attend(C.byref(a), None) == -1 and "cap" in lib.odmkv_last_error().decode()
