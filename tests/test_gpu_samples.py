"""GPT-2 over paged caches that take several tokens at a time, and several samples of each prompt behind its shared rows
(needs a GPU)."""
import pytest
import torch

import model_inference as mi

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SMALL = {"n_heads": 4, "emb_dim": 256, "n_layers": 2}


@pytest.fixture(scope="module")
def model():
    cfg = dict(mi.GPT_CONFIG_124M)
    cfg.update({"vocab_size": 1000, "context_length": 256, "drop_rate": 0.0, "qkv_bias": True, "impl_type": "hip", **SMALL})
    m = mi.GPTModel(cfg).eval()
    mi.init_gpt2_weights(m, 5)
    return m.to(DEV)


def _tokens(seed, *shape):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


# Paths of one model whose attention and projections round to bf16 in different places: the gate of the cached path
# against the full forward, 1e-2 of the logits' norm.
def _close(a, b):
    assert (a - b).norm() / b.norm() <= 1e-2


@pytest.mark.parametrize("page", [16, 20])
def test_a_text_in_pieces_gives_the_logits_of_the_whole(model, page):
    idx = _tokens(1, 3, 120)
    cache = mi.PagedKVCache(SMALL, 3, 130, DEV, page_size=page)
    with torch.no_grad():
        whole = model(idx)
        at = 0
        for n in (50, 1, 40, 2, 27):   # a prompt, a step, and pieces behind what is cached
            got = model(idx[:, at:at + n], kv_cache=cache)
            for i in range(n):
                _close(got[:, i], whole[:, at + i])
            at += n
    assert at == 120 and cache.length == 120
    with pytest.raises(ValueError, match="no place for 50 more tokens"):
        model(idx[:, :50], kv_cache=cache)


@pytest.mark.parametrize("samples", [1, 5])
def test_samples_share_their_prompt(model, samples):
    """The same tokens given to every sample of a prompt give the logits of the prompt's own text."""
    idx, more = _tokens(2, 2, 70), _tokens(3, 2, 12)
    cache = mi.SampledKVCache(SMALL, 2, samples, 80, 12, DEV, page_size=16)
    plain = mi.PagedKVCache(SMALL, 2, 100, DEV, page_size=16)
    with torch.no_grad():
        for _ in range(2):
            a, b = (model(idx, kv_cache=c)[:, -1] for c in (cache, plain))
            _close(a, b)
            cache.share()
            for i in range(12):
                b = model(more[:, i:i + 1], kv_cache=plain)[:, -1]
                a = model(more[:, i:i + 1].repeat_interleave(samples, 0), kv_cache=cache)[:, -1]
                for s in range(samples):
                    _close(a[s::samples], b)
            cache.reset()
            plain.reset()


def test_generate_samples(model):
    idx = _tokens(4, 2, 40)
    one = mi.generate_cached(model, idx, 10, 256, temperature=0.0, cache=mi.PagedKVCache(SMALL, 2, 60, DEV))
    out = mi.generate_samples(model, idx, 3, 10, 256, temperature=0.0)
    assert out.shape == (6, 50) and torch.equal(out[:, :40], idx.repeat_interleave(3, 0))
    assert torch.equal(out[0::3], out[1::3]) and torch.equal(out[0::3], out[2::3])   # alike without a temperature
    # (Two ways of rounding may part at a token whose logits are near: the first tokens' logits are the same call's.)
    assert torch.equal(out[0::3, 40], one[:, 40])
    torch.manual_seed(1)
    cache = mi.SampledKVCache(SMALL, 2, 3, 40, 20, DEV)
    a = mi.generate_samples(model, idx, 3, 20, 256, temperature=1.0, top_k=50, cache=cache)
    torch.manual_seed(1)
    b = mi.generate_samples(model, idx, 3, 20, 256, temperature=1.0, top_k=50, cache=cache)
    assert torch.equal(a, b) and len({tuple(r) for r in a[:3].tolist()}) == 3
    out = mi.generate_samples(model, idx, 3, 8, 256, temperature=0.0, penalties=mi.LogitPenalties(presence=1e4))
    for row in out.tolist():
        assert len(set(row[40:])) == 8 and not set(row[40:]) & set(row[:40])
    first = mi.generate_samples(model, idx[:1], 4, 1, 256, temperature=0.0)[0, -1]
    assert mi.generate_samples(model, idx[:1], 4, 5, 256, temperature=0.0, eos_id=int(first)).shape == (4, 40)
    assert mi.generate_samples(model, idx, 2, 0, 256).shape == (4, 40)
