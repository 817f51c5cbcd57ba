"""The model over an 8-bit cache and behind a shared prefix, against itself over the plain cache: in float32, where both
forms compute the same numbers up to the order of fp32 sums; in 16 bits to the parity bound of the model's own tests
(softmax within 2e-2)."""
import pytest
import torch

from olmo_amd.config import ModelConfig, OLMoConfigurationError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from olmo_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def cfg(kind):
    base = dict(rope=True, alibi=False, include_bias=False, weight_tying=False, vocab_size=1000, embedding_size=1024,
                max_sequence_length=512, attention_dropout=0.0, residual_dropout=0.0, embedding_dropout=0.0)
    if kind == "ln":
        return ModelConfig(d_model=128, n_heads=4, n_layers=3, mlp_ratio=8, layer_norm_type="default", layer_norm_with_affine=False,
                           layer_norm_eps=1e-5, attention_layer_norm=False, norm_after=False, **base)
    c = ModelConfig(d_model=512, n_heads=4, n_layers=3, mlp_hidden_size=2048, layer_norm_type="rms", layer_norm_with_affine=True,
                    layer_norm_eps=1e-6, attention_layer_norm=True, norm_after=True, rope_theta=500000, **base)
    if kind == "gqa":
        c.n_heads, c.n_kv_heads = 8, 2
    return c


def build(kind, dtype, dev, **kw):
    from olmo_amd.model import OLMo

    m = OLMo(cfg(kind), device=dev, dtype=dtype, max_cache_len=256, **kw)
    m.reset_parameters(seed=3)
    return m.post_init()


def ids(B, T, dev, seed=0):
    return torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(seed)).to(dev)


def soft_err(a, b):
    return (torch.softmax(a.float(), -1) - torch.softmax(b.float(), -1)).abs().max().item()


# fp32 sums of a few thousand terms in another order, three layers: relative to the largest logit
F32 = 2.0 ** -24 * 4096


def close32(a, b):
    return (a - b).abs().max().item() <= F32 * b.abs().max().item()


# ------------------------------------------------------------------------------------------------
# 8-bit cache
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["ln", "gqa"])
def test_int8_cache_prompts_see_what_is_stored(dev, kind):
    """A prompt attends to its own rows unrounded (the plain model's logits); a continuation attends to the earlier rows as
    stored: the plain model over a cache that holds the values read back gives the same logits."""
    from olmo_amd import ops

    q8, plain = build(kind, torch.float32, dev, kv_cache="int8"), build(kind, torch.float32, dev)
    x = ids(3, 40, dev)
    mask = torch.ones(3, 40, dtype=torch.int64)
    mask[1, :7] = 0
    a, b = q8(x, attention_mask=mask, use_cache=True), plain(x, attention_mask=mask, use_cache=True)
    assert close32(a.logits, b.logits)
    ca, cb = a.attn_key_values[0].cache, b.attn_key_values[0].cache
    assert ca.row_tensors()[0].dtype == torch.int8 and a.attn_key_values[0][0].shape[2] == 40
    for i in range(len(ca.k)):
        k, v = ops.kv_read_q8(ca.layers[i], 0, 40, torch.float32)
        for got, want in ((k, cb.k[i][:, :, :40]), (v, cb.v[i][:, :, :40])):
            step = want.abs().amax(-1, keepdim=True) / 127
            assert ((got - want).abs() <= step * 0.501 + 1e-5 * want.abs().amax()).all()
            want.copy_(got)
    y = ids(3, 5, dev, seed=1)
    mask = torch.cat((mask, torch.ones(3, 5, dtype=torch.int64)), 1)
    a = q8(y, attention_mask=mask, past_key_values=a.attn_key_values, use_cache=True)
    b = plain(y, attention_mask=mask, past_key_values=b.attn_key_values, use_cache=True)
    assert close32(a.logits, b.logits) and a.attn_key_values[0].cache.length == 45


@pytest.mark.parametrize("kind,dtype,B", [("ln", torch.float32, 2), ("gqa", torch.bfloat16, 3), ("rms", torch.float16, 1), ("rms", torch.bfloat16, 20)])
def test_int8_cache_decode(dev, kind, dtype, B):
    """Greedy decoding, captured and eager, gives the same tokens; a decode step stays within the parity bound of the plain
    model fed the same tokens."""
    from olmo_amd.generate import greedy_generate

    q8, plain = build(kind, dtype, dev, kv_cache="int8"), build(kind, dtype, dev)
    x = ids(B, 33, dev, seed=B)
    mask = torch.ones(B, 33, dtype=torch.int64)
    mask[0, :5] = 0
    toks, logits = greedy_generate(q8, x, mask, 12, return_logits=True)
    eager = greedy_generate(q8, x, mask, 12, use_graph=False)
    assert torch.equal(toks, eager)
    full = torch.cat((x, toks), 1)[:, :-1]
    ref = plain(full, attention_mask=torch.cat((mask, torch.ones(B, 11, dtype=torch.int64)), 1)).logits[:, 32:]
    assert soft_err(logits, ref) <= 2e-2


def test_int8_cache_reference_form_and_hf_cache(dev):
    """Plain (k, v) tensors are taken into an 8-bit cache; transformers' cache operations carry the scales."""
    from olmo_amd.hf import HAVE_TRANSFORMERS

    q8, plain = build("gqa", torch.float32, dev, kv_cache="int8"), build("gqa", torch.float32, dev)
    past = [(torch.randn(2, 2, 9, 64, device=dev), torch.randn(2, 2, 9, 64, device=dev)) for _ in range(3)]
    y = ids(2, 3, dev)
    assert soft_err(q8(y, past_key_values=past).logits, plain(y, past_key_values=past).logits) <= 2e-2
    if not HAVE_TRANSFORMERS:
        return
    from olmo_amd.hf import OLMoCache

    out = q8(ids(3, 20, dev), use_cache=True)
    c = OLMoCache(out.attn_key_values[0].cache)
    before = [t[:, :, :20].clone() for t in c.kv.row_tensors()]
    c.reorder_cache(torch.tensor([2, 0, 0]))
    for t, b in zip(c.kv.row_tensors(), before):
        assert torch.equal(t[:, :, :20], b[[2, 0, 0]])
    c.batch_repeat_interleave(2)
    assert c.kv.B == 6 and len(c.kv.row_tensors()) == 12
    for t, b in zip(c.kv.row_tensors(), before):
        assert torch.equal(t[:, :, :20], b[[2, 2, 0, 0, 0, 0]])
    lg = q8(ids(6, 1, dev), past_key_values=c.legacy()).logits
    assert torch.isfinite(lg).all()


def test_int8_cache_refusals(dev):
    from olmo_amd.model import OLMo

    with pytest.raises(OLMoConfigurationError):
        OLMo(cfg("ln"), device=dev, kv_cache="int4")
    q8 = build("ln", torch.float32, dev, kv_cache="int8")
    with pytest.raises(NotImplementedError):
        q8.generate(ids(1, 4, dev), beam_size=2, max_steps=3)
    with pytest.raises(NotImplementedError):
        q8.share_prefix(ids(1, 4, dev))


# ------------------------------------------------------------------------------------------------
# shared prefix
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("P,T", [(1, 1), (37, 6), (64, 40), (100, 1), (130, 70)])
@pytest.mark.parametrize("kind,dtype", [("ln", torch.float32), ("gqa", torch.float32), ("gqa", torch.bfloat16), ("rms", torch.float16)])
def test_shared_prefix_equals_the_whole_prompt(dev, kind, dtype, P, T):
    m = build(kind, dtype, dev)
    head, x = ids(1, P, dev, seed=P), ids(3, T, dev, seed=T)
    mask = torch.ones(3, T, dtype=torch.int64)
    if T > 1:
        mask[0, : T // 2] = 0
        mask[2, :1] = 0
    whole = torch.cat((head.expand(3, P), x), 1)
    ref = m(whole, attention_mask=torch.cat((torch.ones(3, P, dtype=torch.int64), mask), 1), use_cache=True)
    prefix = m.share_prefix(head[0])
    out = m(x, attention_mask=mask, use_cache=True, prefix=prefix)
    seen = mask.bool()  # (what a padding position computes is nobody's business)
    a, b = out.logits[seen.to(dev)], ref.logits[:, P:][seen.to(dev)]
    assert close32(a, b) if dtype == torch.float32 else soft_err(a, b) <= 2e-2
    y = ids(3, 2, dev, seed=9)
    for t in range(2):  # two more tokens, one at a time
        mask = torch.cat((mask, torch.ones(3, 1, dtype=torch.int64)), 1)
        whole_mask = torch.cat((torch.ones(3, P, dtype=torch.int64), mask), 1)
        out = m(y[:, t:t + 1], attention_mask=mask, past_key_values=out.attn_key_values, use_cache=True)
        ref = m(y[:, t:t + 1], attention_mask=whole_mask, past_key_values=ref.attn_key_values, use_cache=True)
        assert close32(out.logits, ref.logits) if dtype == torch.float32 else soft_err(out.logits, ref.logits) <= 2e-2


@pytest.mark.parametrize("kind,dtype", [("ln", torch.float32), ("gqa", torch.bfloat16)])
def test_shared_prefix_generate(dev, kind, dtype):
    """Captured and eager greedy decoding behind a prefix give the same tokens; so does one prefix used twice; the scores
    are those of the whole prompts."""
    m = build(kind, dtype, dev)
    head, x = ids(1, 50, dev), ids(4, 7, dev, seed=2)
    prefix = m.share_prefix(head)
    a = m.generate(x, max_steps=14, prefix=prefix, stop_at_eos=False)
    b = m.generate(x, max_steps=14, prefix=prefix, stop_at_eos=False, use_graph=False)
    assert torch.equal(a.token_ids, b.token_ids)
    again = m.generate(x[1:3], max_steps=14, prefix=prefix, stop_at_eos=False)
    whole = torch.cat((head.expand(4, 50), x), 1)
    if dtype == torch.float32:
        ref = m.generate(whole, max_steps=14, stop_at_eos=False)
        assert torch.equal(a.token_ids, ref.token_ids) and torch.equal(again.token_ids, ref.token_ids[1:3])
        assert close32(a.scores, ref.scores)
    else:
        lg = m(torch.cat((whole, a.token_ids[:, 0]), 1)[:, :-1]).logits[:, 56:].float()
        best, mine = lg.max(-1).values, lg.gather(-1, a.token_ids[:, 0].unsqueeze(-1)).squeeze(-1)
        assert (mine >= best - 3 * 2.0 ** -7 * best.abs().clamp_min(1.0)).all()  # within three bf16 steps of the best
    if dtype == torch.float32:  # the largest alone (16-bit logits tie, and a sampler keeps all that tie)
        from olmo_amd.beam_search import TopKSampler

        s = m.generate(x, max_steps=5, prefix=prefix, stop_at_eos=False, sampler=TopKSampler(k=1))
        assert torch.equal(s.token_ids, a.token_ids[:, :, :5])


def test_shared_prefix_refusals(dev):
    m = build("ln", torch.float32, dev)
    with pytest.raises(ValueError):
        m.share_prefix(ids(1, 256, dev))
    with pytest.raises(ValueError):
        m.share_prefix(torch.empty(0, dtype=torch.int64))
    p = m.share_prefix(ids(1, 10, dev))
    x = ids(2, 4, dev)
    with pytest.raises(ValueError):
        build("gqa", torch.float32, dev)(x, prefix=p)
    with pytest.raises(ValueError):
        m(ids(2, 247, dev), prefix=p)
    with pytest.raises(ValueError):
        m.generate(x, max_steps=250, prefix=p)
    with pytest.raises(NotImplementedError):
        m.generate(x, max_steps=3, beam_size=2, prefix=p)
    with pytest.raises(NotImplementedError):
        m(x, prefix=p, attention_bias=torch.zeros(1, 1, 14, 14))
    plain = m(x, use_cache=True).attn_key_values
    with pytest.raises(ValueError):
        m(x, past_key_values=plain, prefix=p)
