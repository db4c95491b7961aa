"""CPU-side tests of the paged cache's bookkeeping and of LogitPenalties (model_inference): no kernel is launched."""
import numpy as np
import pytest
import torch

import custom_flash_attn
import model_inference as mi

CFG = {"n_heads": 2, "emb_dim": 32, "n_layers": 2}


def test_pages_are_held_or_free_once(monkeypatch):
    calls = []
    monkeypatch.setattr(custom_flash_attn, "evict", lambda k, v, table, lens, w, new, budget, **kw: calls.append(
        (table.clone(), new.clone(), lens.clone(), budget, kw["recent"], kw["weights_out"] is w)))
    c = mi.PagedKVCache(CFG, 3, 50, "cpu", page_size=8, budget=20, recent=5, slack=6)
    assert c.table.shape == (3, 7) and c.k[0].shape == (3 * 7 + 3 * 4, 2, 8, 16) and c.weights[1].shape == (3, 2, 56)
    c.advance(26)
    assert c.over()
    old = c.table.clone()
    c.evict()
    assert len(calls) == 2 and c.length == 20 and c.seqlens.tolist() == [20] * 3 and c.positions.tolist() == [26] * 3
    for table, new, lens, budget, recent, in_place in calls:
        assert torch.equal(table, old) and new.shape == (3, 4) and lens.tolist() == [26] * 3
        assert (budget, recent, in_place) == (20, 5, True)
        assert not set(old.flatten().tolist()) & set(new.flatten().tolist())
    for _ in range(5):
        assert sorted(c.table.flatten().tolist() + c._free) == list(range(33))
        c.advance(6)
        assert c.over()
        c.evict()
    calls.clear()
    c.evict()   # nothing over the budget
    assert not calls and not c.over()
    c.reset()
    assert c.table.shape == (3, 7) and c.length == 0


def test_cuts_again_where_budget_and_slack_pass_the_longest_text(monkeypatch):
    monkeypatch.setattr(custom_flash_attn, "evict", lambda *a, **kw: None)
    c = mi.PagedKVCache(CFG, 2, 50, "cpu", page_size=8, budget=10, slack=1000)
    for _ in range(4):
        c.advance(9)
        c.evict()
        assert c.table.shape == (2, 7) and c.length == min(10, int(c.positions[0]))
        assert sorted(c.table.flatten().tolist() + c._free) == list(range(28))


def test_paged_cache_refuses_budgets_that_make_no_sense():
    with pytest.raises(ValueError, match="budget must be positive"):
        mi.PagedKVCache(CFG, 1, 50, "cpu", budget=0)
    with pytest.raises(ValueError, match="recent must be between"):
        mi.PagedKVCache(CFG, 1, 50, "cpu", budget=10, recent=11)
    with pytest.raises(ValueError, match="slack must be positive"):  # the row after a cut needs a place
        mi.PagedKVCache(CFG, 1, 50, "cpu", budget=16, page_size=8, slack=0)
    with pytest.raises(ValueError, match="no budget"):
        mi.PagedKVCache(CFG, 1, 50, "cpu").evict()


@pytest.mark.parametrize("rows", [False, True])
def test_logit_penalties_on_the_cpu(rows):
    g = torch.Generator().manual_seed(4)
    B, V, T = 3, 70, 40
    x = torch.randn(B, V, generator=g) * 3
    idx = torch.randint(0, V, (B, T), generator=g)
    p = dict(repetition=1.3, presence=0.5, frequency=0.25)
    if rows:
        p = {k: torch.rand(B, generator=g) + 0.5 for k in p}
    bias = torch.randn(V, generator=g)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (B, 3), generator=g).to(torch.int32)
    seen = []
    got = mi.LogitPenalties(**p, bias=bias, allowed=lambda text: (seen.append(text), allowed)[1])(x, idx)
    assert seen[0] is idx
    for b in range(B):
        r, s, f = (float(t[b]) if rows else t for t in p.values())
        for v in range(V):
            n, y = int((idx[b] == v).sum()), float(x[b, v])
            if n:
                y = (y / r if y > 0 else y * r) - f * n - s
            y += float(bias[v])
            if not (int(allowed[b, v // 32]) >> (v % 32)) & 1:
                assert got[b, v] == -np.inf
            else:
                assert abs(float(got[b, v]) - y) <= 8 * 2.0 ** -24 * (abs(float(x[b, v])) * 2 + n + 4 + abs(y))


def test_generate_applies_penalties_on_the_cpu():
    cfg = dict(mi.GPT_CONFIG_124M)
    cfg.update({"emb_dim": 64, "n_heads": 2, "n_layers": 1, "vocab_size": 50, "drop_rate": 0.0, "impl_type": "manual"})
    model = mi.GPTModel(cfg).eval()
    mi.init_gpt2_weights(model, 3)
    idx = torch.randint(0, 50, (2, 5), generator=torch.Generator().manual_seed(1))
    out = mi.generate(model, idx, 20, 256, temperature=0.0, penalties=mi.LogitPenalties(presence=1e4))
    for row in out.tolist():
        assert len(set(row[5:])) == 20 and not set(row[5:]) & set(row[:5])


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_logit_penalties_on_the_cpu_take_what_the_device_takes(dtype):
    """int32 texts, and ids outside the vocabulary, which count for nothing."""
    x = torch.tensor([[2.0, -1.0, 3.0, 0.5]])
    idx = torch.tensor([[2, -1, 2, 4, 1, 100]], dtype=dtype)
    got = mi.LogitPenalties(repetition=2.0, presence=0.25, frequency=0.5)(x, idx)
    assert got.tolist() == [[2.0, -1.0 * 2 - 0.5 - 0.25, 3.0 / 2 - 2 * 0.5 - 0.25, 0.5]]
    assert mi.LogitPenalties(presence=1.0)(x, idx[:, :0]).tolist() == x.tolist()


def test_a_token_past_the_table_is_refused(monkeypatch):
    """A cut leaves a table for budget + slack rows; a loop that does not cut again is told so (the step itself would
    give NaN)."""
    steps = []
    monkeypatch.setattr(custom_flash_attn, "evict", lambda *a, **kw: None)
    monkeypatch.setattr(custom_flash_attn, "decode_paged", lambda *a, **kw: steps.append(a))
    c = mi.PagedKVCache(CFG, 2, 50, "cpu", page_size=8, budget=10, slack=5)
    c.advance(20)
    c.evict()
    for _ in range(6):   # two pages
        c.attend(0, None, None, None)
        c.advance(1)
    with pytest.raises(ValueError, match="16 rows"):
        c.attend(0, None, None, None)
    c.evict()
    c.attend(0, None, None, None)
    assert len(steps) == 7
