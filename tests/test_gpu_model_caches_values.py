"""The values that a model computes over an 8-bit cache and behind a shared prefix.

Logits are compared relative to their own size: fp32 forms that compute the same numbers in another order of sums to
``F32`` of the largest logit (test_gpu_model_caches.py)."""
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
