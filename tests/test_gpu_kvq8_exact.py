"""The 8-bit cache's codes and results where one rounding decides: equal to the definition, or within the roundings that the
result cannot do without."""
import pytest
import torch

from .test_gpu_kvq8 import TINY, _ops, dev, write_case  # noqa: F401  (dev: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,H,Hkv,hd", [(2, 9, 8, 8, 32), (3, 300, 4, 2, 64), (1, 1, 32, 32, 128), (2, 2100, 40, 40, 128), (1, 4100, 3, 1, 64)])
def test_codes_are_the_rounded_quotients(dev, dtype, B, T, H, Hkv, hd):  # noqa: F811
    """scale = max(max |x| / 127, FLT_MIN) and code = rint(x / scale), each one fp32 operation: equal to the last bit.  The
    values are what a product with 1 / scale gets wrong: halves of the row's maximum and other fractions m / 254 of it, next to
    ties.  The values are used as they come (v is neither normed nor rotated)."""
    ops = _ops()
    print("codes", dtype, B, T, H, Hkv, hd, flush=True)
    qkv, _, _, sin, cos = write_case(dtype, B, T, H, Hkv, hd, False, T, seed=hd + T)
    gen = torch.Generator().manual_seed(T)
    v = qkv.view(B, T, H + 2 * Hkv, hd)[:, :, H + Hkv:]
    top = (0.5 + torch.rand(B, T, Hkv, 1, generator=gen)).to(dtype).float()
    odd = 2 * torch.randint(-127, 127, (B, T, Hkv, hd), generator=gen) + 1
    near = (top * odd / 254).to(dtype)
    near[..., 0::4] = (top / 2).to(dtype) * torch.where(odd[..., 0::4] > 0, 1, -1)
    near[..., 3] = top[..., 0].to(dtype)
    v.copy_(near)
    c = ops.KVQ8.empty(B, Hkv, T, hd, dev)
    ops.qknorm_rope_kvwrite_q8(qkv.to(dev), None, None, sin.to(dev), cos.to(dev), c, B, T, H, Hkv, hd, 0, 1e-6)
    x = near.float().transpose(1, 2)
    scale = (x.abs().amax(-1) / 127).clamp_min(TINY)
    assert torch.equal(c.v_scale.cpu(), scale)
    assert torch.equal(c.v.cpu().float(), (x / scale.unsqueeze(-1)).round())
