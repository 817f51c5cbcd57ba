"""Attention under a shared prefix in float32 with heads of 128: each choice of row tiles for the prefix and for the own keys,
with and without masked own keys, against the definition in 64 bits (tolerances of test_gpu_shared_prefix.py)."""
import pytest
import torch

from .test_gpu_shared_prefix import F32MIN, call, case, dev, reference  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,T,P,past,H,Hkv", [
    (9, 1, 70, 64, 8, 8), (16, 1, 515, 31, 2, 2),                        # one tile over one
    (17, 1, 1, 0, 4, 4), (40, 1, 300, 100, 8, 8), (5, 1, 1030, 33, 40, 8), (64, 1, 2049, 7, 6, 2),  # two over one
    (2, 20, 33, 0, 3, 3), (3, 17, 129, 40, 8, 2), (1, 70, 260, 9, 4, 4), (2, 257, 64, 1, 2, 1),  # two over two
])
def test_row_tiles(dev, masked, B, T, P, past, H, Hkv):  # noqa: F811
    print("prefix fp32 128", masked, B, T, P, past, H, Hkv, flush=True)
    q, kp, vp, kc, vc = case(torch.float32, B, T, P, past, H, Hkv, 128, seed=B + P)
    n, bias = past + T, None
    if masked:  # each sequence's first keys, other depths; rows that are masked hold nothing finite; a finite penalty
        bias = torch.zeros(B, n)
        bias[:, n // 2] = -1.75
        for b in range(B):
            bias[b, : (b * n) // B] = F32MIN
            m = bias[b, :n] <= -1e30
            kc[b, :, :n][:, m], vc[b, :, :n][:, m] = float("nan"), float("inf")
    ref, tol = reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, 128, bias)
    out = call(dev, q, kp, vp, kc, vc, B, T, P, past, H, Hkv, 128, bias)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
