"""What the `transformers` side of the paged 8-bit cache asks of a pool whose rows share what they hold: on the CPU, over a stand-in."""
import pytest
import torch

from test_paged_adapter import _Module, _Pool, _sdpa, _tagged


@pytest.mark.parametrize("shares", [False, True])
def test_steps_ask_for_common_blocks_where_the_cache_was_told_so(shares):
    pool, k, v = _tagged(L=1)
    pool.shares = shares
    _sdpa()(_Module(), torch.zeros(1, 4, 1, 128), k, v, None, softcap=7.0)
    assert [asked.get("shared", False) for asked in pool.asked] == [shares] and pool.asked[0]["softcap"] == 7.0


def test_a_prompt_of_its_own_goes_to_its_own_attention(monkeypatch):
    from kvquant import prompt
    asked = []
    monkeypatch.setattr(prompt, "prompt_attention", lambda *rows, **how: asked.append((rows, how)) or torch.zeros(1, 9, 4, 128))
    pool, k, v = _tagged(L=9)
    rows = (torch.ones(1, 2, 9, 128), torch.ones(1, 2, 9, 128))
    k._odmkv_prompt_rows = rows
    q = torch.zeros(1, 4, 9, 128)
    _sdpa()(_Module(), q, k, v, None, softcap=7.0, scaling=0.1, sliding_window=5)
    assert not pool.asked and asked[0][0][0] is q and asked[0][0][1] is rows[0] and asked[0][0][2] is rows[1]
    assert asked[0][1] == dict(scaling=0.1, softcap=7.0, window=5, starts=None)
    with pytest.raises(RuntimeError, match="cannot be answered from the paged cache"):
        _sdpa()(_Module(), q, k, v, None, dropout=0.1)
    holes = torch.ones(9, 9, dtype=torch.bool).tril()
    holes[8, 3] = False
    with pytest.raises(RuntimeError, match="cannot be answered from the paged cache"):
        _sdpa()(_Module(), q, k, v, holes[None, None])


def test_the_switches():
    from transformers import LlamaConfig
    from kvquant import PagedCache
    base = LlamaConfig(hidden_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128, attn_implementation="sdpa")
    cache = PagedCache(base)
    assert not cache.shared and not cache.native_prompt
    cache = PagedCache(base, shared=True, native_prompt=True)
    assert cache.shared and cache.native_prompt
