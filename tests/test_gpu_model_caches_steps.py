"""Decode steps of whole models over an 8-bit cache and behind a shared prefix, value for value.

The other side is the plain model whose cache is made to hold what the form under test stores: for the 8-bit cache every row
is rounded to 8 bits (in torch, by the definition) as soon as it is written.  fp32: equal up to the order of fp32 sums
(``close32``).  16 bits: ``near``, relative to the logits' own size.  The bounds have power: what a step computes with a wrong
mask, position or prefix is shown to lie outside them."""
import contextlib

import pytest
import torch

from .test_gpu_model_caches import build, cfg, close32, dev, ids  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu

# A logit has gone through 35 roundings to 8 bits (11 a layer, three layers, final norm and head), each off by at most 2^-8 of
# what is rounded, 2^-8 / sqrt(3) in the root mean square; both sides have their own, and a stored row may be one code (1 / 127
# of its maximum, about 2^-5.5 of its root mean square / sqrt(12)) apart: 2^-8 / sqrt(3) * sqrt(2 * 35) = 0.019, and 0.007
# twice a layer for keys and values.  Together below 0.026; a norm in front of the head may double it.
NEAR = 0.052


def distance(a, b):
    a, b = a.float(), b.float()
    return ((a - b).pow(2).mean() / b.pow(2).mean()).sqrt().item()


def near(a, b, dtype):
    return close32(a, b) if dtype == torch.float32 else distance(a, b) <= NEAR


def round8(x):
    s = (x.float().abs().amax(-1, keepdim=True) / 127).clamp_min(torch.finfo(torch.float32).tiny)
    return ((x.float() / s).round() * s).to(x.dtype)


@contextlib.contextmanager
def rows_rounded(monkeypatch):
    """Every cache row that a plain decode step writes is rounded to 8 bits before the step's attention reads it."""
    from olmo_amd import ops

    write = ops.qknorm_rope_kvwrite

    def rounding(qkv, qw, kw, sin, cos, kc, vc, B, T, H, Hkv, hd, past_len, eps, past_len_dev=None):
        assert past_len_dev is None
        q = write(qkv, qw, kw, sin, cos, kc, vc, B, T, H, Hkv, hd, past_len, eps)
        for c in (kc, vc):
            c[:, :, past_len:past_len + T] = round8(c[:, :, past_len:past_len + T])
        return q

    with monkeypatch.context() as m:
        m.setattr(ops, "attn_decode_fused", lambda *a, **k: None)  # declines: the row is written by a launch of its own
        m.setattr(ops, "qknorm_rope_kvwrite", rounding)
        yield


def round_cache(cache):
    for t in cache.row_tensors():
        t[:, :, : cache.length] = round8(t[:, :, : cache.length])


def int4(dev, **kw):
    """Models whose decode steps at up to 8 rows are the chained blocks of int4 linears."""
    from olmo_amd.synthetic import build_random_model

    c = cfg("rms")
    c.n_heads = 4
    m = build_random_model(c, torch.bfloat16, quantized=True, seed=2, device=dev, max_cache_len=256)
    m.kv_cache = kw.get("kv_cache")
    return m


MODELS = [("ln", torch.float32, 2), ("gqa", torch.float32, 3), ("gqa", torch.bfloat16, 3), ("rms", torch.float16, 2), ("rms", torch.bfloat16, 20),
          ("int4", torch.bfloat16, 1), ("int4", torch.bfloat16, 4)]


def make(kind, dtype, dev, **kw):
    return int4(dev, **kw) if kind == "int4" else build(kind, dtype, dev, **kw)


@pytest.mark.parametrize("kind,dtype,B", MODELS)
def test_int8_decode_steps(dev, monkeypatch, kind, dtype, B):  # noqa: F811
    print("int8 steps", kind, dtype, B, flush=True)
    q8, plain = make(kind, dtype, dev, kv_cache="int8"), make(kind, dtype, dev)
    T = 40
    x = ids(B, T, dev, seed=B)
    mask = torch.ones(B, T, dtype=torch.int64)
    mask[0, :15] = 0
    a, b = q8(x, attention_mask=mask, use_cache=True), plain(x, attention_mask=mask, use_cache=True)
    other = plain(x, use_cache=True)
    round_cache(b.attn_key_values[0].cache), round_cache(other.attn_key_values[0].cache)
    y = ids(B, 4, dev, seed=B + 1)
    for t in range(4):
        mask = torch.cat((mask, torch.ones(B, 1, dtype=torch.int64)), 1)
        step = dict(attention_mask=mask, use_cache=True)
        a = q8(y[:, t:t + 1], past_key_values=a.attn_key_values, **step)
        with rows_rounded(monkeypatch):
            b = plain(y[:, t:t + 1], past_key_values=b.attn_key_values, **step)
            other = plain(y[:, t:t + 1], past_key_values=other.attn_key_values, use_cache=True)  # the same without the mask
        assert near(a.logits, b.logits, dtype)
        assert not near(other.logits[:1], b.logits[:1], dtype)
    if kind == "int4":
        assert q8._chain_ok[B] and plain._chain_ok[B]
    # a token one position further on (the cache begins with one more row): outside the bound
    shifted = plain(torch.cat((x[:, :1], x), 1), use_cache=True)
    ones = plain(x, use_cache=True)
    with rows_rounded(monkeypatch):
        shifted = plain(y[:, :1], past_key_values=shifted.attn_key_values, use_cache=True)
        ones = plain(y[:, :1], past_key_values=ones.attn_key_values, use_cache=True)
    assert not near(shifted.logits, ones.logits, dtype)


@pytest.mark.parametrize("kind,dtype,B", MODELS)
def test_int8_captured_steps(dev, monkeypatch, kind, dtype, B):  # noqa: F811
    """Replayed steps of a captured graph: the logits of the plain model fed the same tokens, rows rounded."""
    from olmo_amd.generate import greedy_generate

    q8, plain = make(kind, dtype, dev, kv_cache="int8"), make(kind, dtype, dev)
    x = ids(B, 33, dev, seed=B)
    mask = torch.ones(B, 33, dtype=torch.int64)
    mask[-1, :9] = 0
    toks, logits = greedy_generate(q8, x, mask, 9, return_logits=True)
    eager, eager_logits = greedy_generate(q8, x, mask, 9, return_logits=True, use_graph=False)
    assert torch.equal(toks, eager) and torch.equal(logits, eager_logits)
    b = plain(x, attention_mask=mask, use_cache=True)
    assert near(logits[:, 0], b.logits[:, -1], dtype)
    round_cache(b.attn_key_values[0].cache)
    for t in range(8):
        mask = torch.cat((mask, torch.ones(B, 1, dtype=torch.int64)), 1)
        with rows_rounded(monkeypatch):
            b = plain(toks[:, t:t + 1], attention_mask=mask, past_key_values=b.attn_key_values, use_cache=True)
        assert near(logits[:, t + 1], b.logits[:, 0], dtype)


def test_int8_takes_the_reference_form(dev):  # noqa: F811
    """Plain (k, v) tensors become codes: the plain model over the same rows rounded."""
    q8, plain = build("gqa", torch.float32, dev, kv_cache="int8"), build("gqa", torch.float32, dev)
    gen = torch.Generator().manual_seed(4)
    past = [tuple(torch.randn(2, 2, 9, 64, generator=gen).to(dev) for _ in range(2)) for _ in range(3)]
    y = ids(2, 3, dev)
    cache = plain._ingest_reference_cache(past, 3)
    exact = plain(y, past_key_values=past).logits
    round_cache(cache)
    want = plain(y, past_key_values=cache.views()).logits
    assert close32(q8(y, past_key_values=past).logits, want) and not close32(exact, want)


@pytest.mark.parametrize("P,T", [(1, 1), (37, 6), (100, 1), (130, 70)])
@pytest.mark.parametrize("kind,dtype,B", MODELS)
def test_steps_behind_a_prefix(dev, kind, dtype, B, P, T):  # noqa: F811
    print("prefix steps", kind, dtype, B, P, T, flush=True)
    m = make(kind, dtype, dev)
    head, x, y = ids(1, P, dev, seed=P), ids(B, T, dev, seed=T), ids(B, 3, dev, seed=9)
    mask = torch.ones(B, T, dtype=torch.int64)
    if T > 1:
        mask[0, : T // 2] = 0
    whole = torch.cat((head.expand(B, P), x), 1)
    full = lambda n: torch.cat((torch.ones(B, P, dtype=torch.int64), mask, torch.ones(B, n, dtype=torch.int64)), 1)
    ref = m(whole, attention_mask=full(0), use_cache=True)
    out = m(x, attention_mask=mask, use_cache=True, prefix=m.share_prefix(head))
    seen = mask.bool().to(dev)
    assert near(out.logits[seen], ref.logits[:, P:][seen], dtype)
    bare = m(x, attention_mask=mask, use_cache=True)  # the same without the prefix
    if P > 1:
        assert not near(bare.logits[seen], ref.logits[:, P:][seen], dtype)
    for t in range(3):
        own = torch.cat((mask, torch.ones(B, t + 1, dtype=torch.int64)), 1)
        out = m(y[:, t:t + 1], attention_mask=own, past_key_values=out.attn_key_values, use_cache=True)
        ref = m(y[:, t:t + 1], attention_mask=full(t + 1), past_key_values=ref.attn_key_values, use_cache=True)
        assert near(out.logits, ref.logits, dtype)
    if kind == "int4":
        assert m._chain_ok[B]


@pytest.mark.parametrize("B", [1, 4])
def test_captured_int4_steps_behind_a_prefix(dev, B):  # noqa: F811
    from olmo_amd.generate import greedy_generate

    m = int4(dev)
    head, x = ids(1, 60, dev, seed=1), ids(B, 5, dev, seed=2)
    prefix = m.share_prefix(head)
    toks, logits = greedy_generate(m, x, None, 9, return_logits=True, prefix=prefix)
    eager, eager_logits = greedy_generate(m, x, None, 9, return_logits=True, use_graph=False, prefix=prefix)
    assert torch.equal(toks, eager) and torch.equal(logits, eager_logits)
    whole = torch.cat((head.expand(B, 60), x, toks[:, :-1]), 1)
    assert near(logits, m(whole).logits[:, 64:], torch.bfloat16)


def test_loaders_take_the_form_of_the_cache(dev, tmp_path):  # noqa: F811
    """``from_quantized`` and ``load_unsharded_checkpoint`` hand ``kv_cache`` on: the loaded model decodes over codes, to the
    same logits as the model that was saved."""
    import yaml
    from dataclasses import asdict

    from olmo_amd.checkpoint import BaseQuantizeConfig, load_unsharded_checkpoint
    from olmo_amd.hf import OLMoConfig, OLMoForCausalLM
    from olmo_amd.model import QuantKVCache
    from olmo_amd.qlinear import OLMoGPTQForCausalLM

    def steps(m):
        x = ids(2, 12, dev, seed=1)
        out = m(x, use_cache=True)
        assert isinstance(out.attn_key_values[0].cache, QuantKVCache)
        step = m(x[:, :1], past_key_values=out.attn_key_values, use_cache=True)
        return out.logits, step.logits

    m = int4(dev, kv_cache="int8")
    hf = OLMoForCausalLM(OLMoConfig.from_model_config(m.config, use_cache=True), model=m)
    OLMoGPTQForCausalLM(hf, True, BaseQuantizeConfig(bits=4, group_size=128, desc_act=False)).save_quantized(str(tmp_path / "q"))
    loaded = OLMoGPTQForCausalLM.from_quantized(str(tmp_path / "q"), device=str(dev), max_cache_len=256, kv_cache="int8")
    for a, b in zip(steps(loaded.model.model), steps(m)):
        assert torch.equal(a, b)

    m = build("gqa", torch.float32, dev, kv_cache="int8")
    d = tmp_path / "u"
    d.mkdir()
    conf = {k: v for k, v in asdict(m.config).items() if k != "extra"}
    (d / "config.yaml").write_text(yaml.safe_dump({"model": conf}))
    torch.save({k: v.cpu() for k, v in m.state_dict().items()}, d / "model.pt")
    loaded = load_unsharded_checkpoint(str(d), device=str(dev), dtype=torch.float32, max_cache_len=256, kv_cache="int8")
    for a, b in zip(steps(loaded), steps(m)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind,dtype,B", MODELS)
def test_prompts_of_one_token(dev, monkeypatch, kind, dtype, B):  # noqa: F811
    """The shortest conversation: one token, then steps behind it, eager and captured, over codes and behind a prefix that fills
    the model's length but for what follows."""
    from olmo_amd.generate import greedy_generate

    print("one token", kind, dtype, B, flush=True)
    q8, plain = make(kind, dtype, dev, kv_cache="int8"), make(kind, dtype, dev)
    x = ids(B, 1, dev, seed=B)
    a, b = q8(x, use_cache=True), plain(x, use_cache=True)
    assert near(a.logits, b.logits, dtype)
    toks, logits = greedy_generate(q8, x, None, 6, return_logits=True)
    assert torch.equal(logits[:, 0], a.logits[:, 0])
    round_cache(b.attn_key_values[0].cache)
    for t in range(5):
        with rows_rounded(monkeypatch):
            b = plain(toks[:, t:t + 1], past_key_values=b.attn_key_values, use_cache=True)
        assert near(logits[:, t + 1], b.logits[:, 0], dtype)
    head = ids(1, 250, dev, seed=7)  # 250 + 1 + 5: all 256 positions
    prefix = plain.share_prefix(head)
    toks, logits = greedy_generate(plain, x, None, 6, return_logits=True, prefix=prefix)
    whole = plain(torch.cat((head.expand(B, 250), x, toks[:, :-1]), 1)).logits[:, 250:]
    assert near(logits, whole, dtype)
    with pytest.raises(ValueError):
        greedy_generate(plain, x, None, 8, prefix=prefix)
