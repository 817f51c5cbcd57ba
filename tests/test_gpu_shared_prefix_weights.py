"""The weights of attention under a shared prefix keep more bits than the 16-bit type has: the result's own rounding is the only
one that counts, as in the attention over a cache that begins with a copy of the prefix.

Values come in pairs v, -v of nearly the same weight, so results are small next to the weights that made them, and queries pick
one channel, so scores are next to exact: a weight rounded to the type shows."""
import math

import pytest
import torch

from .test_gpu_shared_prefix import call, dev  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


def paired_case(dtype, B, T, P, past, H, Hkv, hd, seed):
    gen = torch.Generator().manual_seed(seed)
    n = past + T

    def keys(*shape):  # pairs 2^-6 apart, in [1, 2)
        k = 1 + torch.randint(0, 126, (*shape[:-2], (shape[-2] + 1) // 2, 1, shape[-1]), generator=gen) / 128
        return torch.cat((k, k + 2.0 ** -6), -2).flatten(-3, -2)[..., : shape[-2], :].to(dtype)

    def values(*shape):
        v = torch.randn((*shape[:-2], (shape[-2] + 1) // 2, 1, shape[-1]), generator=gen).to(dtype)
        return torch.cat((v, -v), -2).flatten(-3, -2)[..., : shape[-2], :].contiguous()

    q = torch.zeros(B, T, H, hd)
    q.scatter_(-1, torch.randint(0, hd, (B, T, H, 1), generator=gen), 8.0)
    return q.view(B, T, H * hd).to(dtype), keys(Hkv, P, hd), values(Hkv, P, hd), keys(B, Hkv, n, hd), values(B, Hkv, n, hd)


def reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd):
    """Output in 64 bits and the tolerance of fp32 scores, maxima and sums and of weights in two numbers of the type: bf16
    8 + 8 bits, fp16 11 + 11 with an absolute error of at most 2^-25 next to a sum that is at least 2^7."""
    f8, dtype, n, G = torch.float64, q.dtype, past + T, H // Hkv
    out, tol = (torch.empty(B, T, H, hd, dtype=f8) for _ in range(2))
    hide = torch.cat((torch.zeros(T, P, dtype=torch.bool), torch.arange(n)[None, :] > past + torch.arange(T)[:, None]), 1)
    for b in range(B):
        for h in range(Hkv):
            k, v = torch.cat((kp[h], kc[b, h])).to(f8), torch.cat((vp[h], vc[b, h])).to(f8)
            qq = q[b].view(T, H, hd)[:, h * G:(h + 1) * G].to(f8)
            size = (qq.abs() @ k.abs().T / math.sqrt(hd)).amax(-1, keepdim=True)
            p = torch.softmax((qq @ k.T / math.sqrt(hd)).masked_fill(hide[:, None, :], float("-inf")), -1)
            # one term of a score is not zero: its product, the scaling, the difference to the maximum, the exponential
            rel = 8 * 2.0 ** -24 * (size + 1) + (P + n + 64) * 2.0 ** -24 + (torch.finfo(dtype).eps / 2) ** 2
            out[b, :, h * G:(h + 1) * G] = p @ v
            tol[b, :, h * G:(h + 1) * G] = rel * (p @ v.abs()) + 2.0 ** -32 * (P + n) * v.abs().max()
    out, tol = out.view(B, T, H * hd), tol.view(B, T, H * hd)
    return out, tol + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -25


CASES = [  # B, T, P, past, H, Hkv, hd
    (1, 1, 2, 1, 1, 1, 64), (3, 1, 6, 3, 4, 2, 32), (20, 1, 10, 1, 2, 2, 128), (5, 1, 300, 41, 16, 2, 128), (17, 1, 40, 7, 8, 8, 64),
    (2, 3, 8, 3, 8, 4, 128), (3, 20, 16, 0, 1, 1, 64), (2, 70, 12, 1, 2, 1, 32),  # several tokens, read in runs of keys
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,P,past,H,Hkv,hd", CASES)
def test_weights_are_not_rounded_to_the_type(dev, dtype, B, T, P, past, H, Hkv, hd):  # noqa: F811
    print("prefix weights", dtype, B, T, P, past, H, Hkv, hd, flush=True)
    args = paired_case(dtype, B, T, P, past, H, Hkv, hd, seed=P + T)
    ref, tol = reference(*args, B, T, P, past, H, Hkv, hd)
    out = call(dev, *args, B, T, P, past, H, Hkv, hd)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("B,T,P,past,H,Hkv,hd", [(1, 33, 6, 1, 1, 1, 64), (2, 40, 64, 3, 2, 2, 128), (3, 130, 30, 0, 4, 2, 128), (1, 65, 6, 1, 1, 1, 64),
                                                 (2, 80, 64, 3, 2, 2, 128)])
def test_fp16_weights_of_prompts(dev, B, T, P, past, H, Hkv, hd):  # noqa: F811
    """The one-pass form for prompts keeps them too in fp16 (bf16 prompts have weights of 8 bits, as ``attn_prefill``)."""
    print("prefix weights, prompt", B, T, P, past, H, Hkv, hd, flush=True)
    args = paired_case(torch.float16, B, T, P, past, H, Hkv, hd, seed=P + T)
    ref, tol = reference(*args, B, T, P, past, H, Hkv, hd)
    out = call(dev, *args, B, T, P, past, H, Hkv, hd)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


def test_fp16_weights_far_below_the_largest(dev):  # noqa: F811
    """One key far above many: each of the others weighs 2^-25.6 of it, all of them together 1 % of it."""
    B, H, hd, P = 2, 4, 64, 500_000
    q = torch.zeros(B, 1, H, hd)
    q[..., 3] = 8.0
    kp, vp = torch.zeros(H, P, hd), torch.ones(H, P, hd)
    kp[:, 7, 3], vp[:, 7] = 17.75, 0.0  # e^17.75 = 2^25.6
    kc, vc = torch.full((B, H, 1, hd), -8.0), torch.zeros(B, H, 1, hd)
    h = lambda t: t.half()
    out = call(dev, h(q).view(B, 1, H * hd), h(kp), h(vp), h(kc), h(vc), B, 1, P, 0, H, H, hd).cpu().double()
    want = (P - 1) / (P - 1 + math.exp(17.75) + math.exp(-8))
    # scores and exponents near 18 and 26 in fp32, then sums of P terms; the result's rounding
    assert (out - want).abs().max() <= (64 * 2.0 ** -24 * 26 + 2.0 ** -11 + 2.0 ** -12) * want
