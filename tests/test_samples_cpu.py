"""CPU-side tests of SampledKVCache's bookkeeping and of what it and PagedKVCache.extend refuse (model_inference): no
kernel is launched."""
import pytest
import torch

import custom_flash_attn
import model_inference as mi

CFG = {"n_heads": 2, "emb_dim": 32, "n_layers": 2}


def test_pages_of_prompts_and_samples_are_apart(monkeypatch):
    calls = []
    monkeypatch.setattr(custom_flash_attn, "decode_shared", lambda *a, **kw: calls.append(a))
    monkeypatch.setattr(custom_flash_attn, "decode_paged", lambda *a, **kw: calls.append(a))
    c = mi.SampledKVCache(CFG, 2, 3, 20, 9, "cpu", page_size=8)
    assert c.table.shape == (2, 3) and c.own_table.shape == (6, 2) and c.k[0].shape == (2 * 3 + 6 * 2, 2, 8, 16)
    for _ in range(2):
        pages = c.table.flatten().tolist() + c.own_table.flatten().tolist()
        assert sorted(pages) == list(range(18)) and c.extends and not c.shared
        c.advance(13)
        c.attend(0, "q", "k", "v")
        assert calls.pop()[3] is c.table
        c.advance(1)
        c.share()
        assert not c.extends and c.positions.tolist() == [14] * 6 and c.seqlens.tolist() == [14] * 2
        for i in range(9):
            assert c.own_lens.tolist() == [i] * 6 and c.positions.tolist() == [14 + i] * 6
            c.attend(1, "q", "k", "v")
            q, k, v, table, lens, own, own_lens, kn, vn = calls.pop()
            assert (k is c.k[1] and v is c.v[1] and table is c.table and lens is c.seqlens and own is c.own_table
                    and own_lens is c.own_lens and (q, kn, vn) == ("q", "k", "v"))
            c.advance(1)
        with pytest.raises(ValueError, match="hold up to 9 tokens"):
            c.attend(0, None, None, None)
        with pytest.raises(ValueError, match="shared already"):
            c.share()
        with pytest.raises(ValueError, match="one new token per step"):
            c.extend(0, None, None, None, None)
        c.reset()
        assert c.seqlens.tolist() == c.positions.tolist() == [0, 0] and c.length == c.own_length == 0


def test_sampled_cache_refuses():
    for kw in (dict(samples=0, new_len=5), dict(samples=2, new_len=0)):
        with pytest.raises(ValueError, match="must be positive"):
            mi.SampledKVCache(CFG, 1, max_len=8, device="cpu", **kw)
    model = mi.GPTModel({**mi.GPT_CONFIG_124M, "emb_dim": 32, "n_heads": 2, "n_layers": 2, "vocab_size": 10, "impl_type": "manual"})
    idx = torch.zeros(1, 6, dtype=torch.long)
    with pytest.raises(ValueError, match="exceeds context_size"):
        mi.generate_samples(model, idx, 2, 10, 15)
    for cache in (mi.SampledKVCache(CFG, 2, 2, 8, 8, "cpu"), mi.SampledKVCache(CFG, 1, 3, 8, 8, "cpu")):
        with pytest.raises(ValueError, match="the cache is for"):
            mi.generate_samples(model, idx, 2, 5, 20, cache=cache)
    with pytest.raises(ValueError, match="shorter than the prompt"):
        mi.generate_samples(model, idx, 2, 10, 20, cache=mi.SampledKVCache(CFG, 1, 2, 8, 8, "cpu"))


def test_extend_refuses_budgets_and_full_tables(monkeypatch):
    with pytest.raises(ValueError, match="budget takes one"):
        mi.PagedKVCache(CFG, 1, 50, "cpu", budget=10).extend(0, None, torch.zeros(1, 2, 2, 16), None, None)
    c = mi.PagedKVCache(CFG, 1, 20, "cpu", page_size=8)
    c.advance(18)
    with pytest.raises(ValueError, match="no place for 7 more tokens"):
        c.extend(0, torch.zeros(1, 7, 2, 16), torch.zeros(1, 7, 2, 16), torch.zeros(1, 7, 2, 16), None)
    calls = []
    monkeypatch.setattr(custom_flash_attn, "append_paged", lambda *a, **kw: calls.append(a))
    monkeypatch.setattr(custom_flash_attn, "attend_paged", lambda *a, **kw: calls.append(a))
    x = torch.zeros(1, 6, 2, 16)
    c.extend(0, x, x, x, torch.zeros(1, 6, 2, 16))
    assert len(calls) == 2 and calls[0][0].shape == (1, 2, 6, 16) and calls[1][3] is c.table
    c.reset()
    with pytest.raises(ValueError, match="no place for 25 more tokens"):
        c.prompt(0, torch.zeros(1, 25, 2, 16), torch.zeros(1, 25, 2, 16), torch.zeros(1, 25, 2, 16), None)
    assert len(calls) == 2


def test_a_budget_refuses_several_tokens_in_the_model():
    att = mi.MultiHeadAttention(32, 32, 64, 0.0, 2, "hip")
    cache = mi.PagedKVCache(CFG, 1, 50, "cpu", budget=10)
    cache.advance(3)
    with torch.no_grad(), pytest.raises(NotImplementedError, match="one new token per step"):
        att(torch.zeros(1, 4, 32), cache, 0)
