"""The values that a model computes over an 8-bit cache and behind a shared prefix.

Logits are compared relative to their own size: fp32 forms that compute the same numbers in another order of sums to
``F32`` of the largest logit (test_gpu_model_caches.py)."""
import gc
import weakref

import pytest
import torch

from .test_gpu_model_caches import build, close32, dev, ids  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["ln", "gqa"])
@pytest.mark.parametrize("T", [1, 2])
def test_int8_prompt_sees_its_own_rows_unrounded(dev, kind, T):  # noqa: F811
    """Also a prompt of one token: the logits of the plain model, whatever the codes will hold."""
    q8, plain = build(kind, torch.float32, dev, kv_cache="int8"), build(kind, torch.float32, dev)
    x = ids(3, T, dev, seed=T)
    a, b = q8(x, use_cache=True), plain(x, use_cache=True)
    assert close32(a.logits, b.logits)
    assert a.attn_key_values[0].cache.length == T


def test_prefix_workspaces_go_with_their_caches(dev):  # noqa: F811
    """Decode steps behind prefixes of many lengths leave nothing behind in the model: the workspace belongs to the sequences'
    cache, is the same from step to step and is given back with it."""
    m = build("gqa", torch.bfloat16, dev)
    x = ids(4, 3, dev)

    def steps(P):
        out = m(x, use_cache=True, prefix=m.share_prefix(ids(1, P, dev)))
        for _ in range(3):
            out = m(x[:, :1], past_key_values=out.attn_key_values, use_cache=True)
        cache = weakref.ref(out.attn_key_values[0].cache)
        del out
        gc.collect()
        assert cache() is None
        m.generate(x, max_steps=6, prefix=m.share_prefix(ids(1, P, dev)), stop_at_eos=False)

    steps(50)
    torch.cuda.synchronize()
    kept, held = len(m._attn_ws), torch.cuda.memory_allocated()
    for P in range(51, 75):
        steps(P)
    torch.cuda.synchronize()
    assert len(m._attn_ws) == kept and torch.cuda.memory_allocated() <= held


@pytest.mark.parametrize("form", ["int8", "prefix"])
def test_sessions_of_two_caches_share_no_workspace(dev, form, monkeypatch):  # noqa: F811
    """What the attention of one session's captured steps writes while it runs is not another session's.  (Read from the calls'
    arguments: a race between two streams shows only now and then.)"""
    from olmo_amd import ops
    from olmo_amd.generate import DecodeSession

    name = "attn_decode_q8" if form == "int8" else "attn_shared_prefix"
    call, at, used = getattr(ops, name), 2 if form == "int8" else 5, []
    monkeypatch.setattr(ops, name, lambda *a, **k: (used.append((a[at].data_ptr(), a[at].numel())), call(*a, **k))[1])
    m = build("gqa", torch.bfloat16, dev, kv_cache="int8" if form == "int8" else None)
    prefix = None if form == "int8" else m.share_prefix(ids(1, 40, dev))
    sessions = []
    for i in range(2):
        out = m(ids(2, 130, dev, seed=i), use_cache=True, last_logits_only=True, prefix=prefix)
        sessions.append(DecodeSession(m, out.attn_key_values[0].cache, out.logits.argmax(-1), None))
    ranges = []
    for s in sessions:
        used.clear()
        s.step()
        s.capture()
        assert len(set(used)) == 1 and used[0][1] > 0
        ranges.append(used[0])
    (a, n), (b, m) = sorted(ranges)
    assert a + 4 * n <= b


@pytest.mark.parametrize("kind,Hkv", [("gqa", 2), ("mqa", 1)])
def test_a_prefix_holds_its_own_rows_alone(dev, kind, Hkv):  # noqa: F811
    """Whatever the count of kv heads: the memory behind a prefix is its rows', not that of a cache of the model's length."""
    from olmo_amd.model import OLMo

    from .test_gpu_model_caches import cfg

    c = cfg("gqa")
    c.n_kv_heads = Hkv
    m = OLMo(c, device=dev, dtype=torch.bfloat16, max_cache_len=256)
    m.reset_parameters(seed=3)
    x = ids(1, 37, dev, seed=5)
    p = m.share_prefix(x[0])  # (on a model that has not run yet)
    storages = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes() for t in (*p.k, *p.v)}
    assert sum(storages.values()) == sum(t.numel() * t.element_size() for t in (*p.k, *p.v)) == 2 * 3 * Hkv * 37 * 64 * 2
    want = m(x, use_cache=True).attn_key_values
    for i, (k, v) in enumerate(want):
        assert torch.equal(p.k[i], k[0]) and torch.equal(p.v[i], v[0])


def test_transformers_cache_emptied_behind_a_prefix_keeps_the_prefix(dev):  # noqa: F811
    """``crop`` and ``reset`` take back the sequences' own rows; the prefix is no row of theirs."""
    from olmo_amd.hf import HAVE_TRANSFORMERS, OLMoCache, OLMoConfig, OLMoForCausalLM

    if not HAVE_TRANSFORMERS:
        pytest.skip("transformers is not installed")
    m = build("gqa", torch.float32, dev)
    hf = OLMoForCausalLM(OLMoConfig.from_model_config(m.config, use_cache=True), model=m)
    prefix, x, y = m.share_prefix(ids(1, 40, dev)), ids(2, 9, dev, seed=1), ids(2, 5, dev, seed=2)
    want = m(y, prefix=prefix).logits
    c = OLMoCache(m(x, use_cache=True, prefix=prefix).attn_key_values[0].cache)
    for empty in (lambda: c.crop(-9), c.reset):
        empty()
        assert c.get_seq_length() == 0
        out = hf(y, past_key_values=c, use_cache=True)
        assert torch.equal(out.logits, want)
        assert out.past_key_values is c and c.get_seq_length() == 5 and c.kv.prefix is prefix
