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


@pytest.mark.parametrize("power", [-126, -118, -104, -98, -96, -60, 60, 125])
def test_codes_of_tiny_and_huge_rows(dev, power):  # noqa: F811
    """The same where quotients, residuals or reciprocals come near the ends of fp32's range."""
    ops = _ops()
    T, H, hd = 64, 2, 64
    gen = torch.Generator().manual_seed(power + 200)
    odd = 2 * torch.randint(-127, 127, (1, T, H, hd), generator=gen) + 1
    x = (0.5 + torch.rand(1, T, H, 1, generator=gen)) * odd / 254
    x[..., 0::4] = x.abs().amax(-1, keepdim=True) / 2
    x = torch.ldexp(x, torch.tensor(float(power)))
    qkv = torch.zeros(1, T, 3 * H * hd)
    qkv.view(1, T, 3 * H, hd)[:, :, 2 * H:] = x
    sin, cos = ops.rope_tables(hd, 10000.0, T, dev)
    c = ops.KVQ8.empty(1, H, T, hd, dev)
    ops.qknorm_rope_kvwrite_q8(qkv.to(dev), None, None, sin, cos, c, 1, T, H, H, hd, 0, 1e-6)
    x = x.transpose(1, 2)
    scale = (x.abs().amax(-1) / 127).clamp_min(TINY)
    assert torch.equal(c.v_scale.cpu(), scale)
    want = (x.double() / scale.double().unsqueeze(-1)).float().round()  # (53 bits, then 24: the fp32 quotient)
    assert torch.equal(c.v.cpu().float(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,keys,H,Hkv,hd", [(1, 4, 1, 1, 64), (3, 12, 4, 2, 32), (2, 300, 8, 8, 128), (20, 60, 16, 2, 64)])
def test_decode_weights_keep_16_bits(dev, dtype, B, keys, H, Hkv, hd):  # noqa: F811
    """Weight times scale is multiplied in two bf16 numbers.  Values come in pairs v, -v of nearly the same weight and queries
    pick one channel: results are small next to their weights, scores next to exact, so a weight of 8 bits would show (the
    reference with such weights is outside the tolerance)."""
    ops, f8 = _ops(), torch.float64
    print("q8 weights", dtype, B, keys, H, Hkv, hd, flush=True)
    gen = torch.Generator().manual_seed(keys + hd)
    k = torch.randint(40, 110, (B, Hkv, keys // 2, 1, hd), generator=gen)
    k = torch.cat((k, k + 1), -2).flatten(2, 3).to(torch.int8)
    v = torch.randint(-127, 128, (B, Hkv, keys // 2, 1, hd), generator=gen)
    v = torch.cat((v, -v), -2).flatten(2, 3).to(torch.int8)
    ks = torch.full((B, Hkv, keys), 2.0 ** -6)
    vs = (0.01 + 0.02 * torch.rand(B, Hkv, keys // 2, 1, generator=gen)).expand(-1, -1, -1, 2).flatten(2).contiguous()
    q = torch.zeros(B, H, hd)
    q.scatter_(-1, torch.randint(0, hd, (B, H, 1), generator=gen), 8.0)
    q = q.to(dtype)
    cache = ops.KVQ8(*(t.to(dev) for t in (k, v, ks, vs)))
    ws = ops.attn_decode_q8_workspace(B, H, Hkv, hd, keys, dev)
    out = ops.attn_decode_q8(q.view(B, 1, H * hd).to(dev), cache, ws, B, H, Hkv, hd, keys - 1, keys)
    x = q.to(f8).view(B, Hkv, H // Hkv, hd) @ (k.to(f8) * ks.to(f8).unsqueeze(-1)).transpose(-1, -2) / hd ** 0.5
    p, values = torch.softmax(x, -1), v.to(f8) * vs.to(f8).unsqueeze(-1)
    ref = p @ values
    # scores: product, scale, difference to the maximum, exponential; the sums; weight times scale to 8 + 8 bits; the result
    rel = 8 * 2.0 ** -24 * (x.amax(-1, keepdim=True) + 1) + (keys + 64) * 2.0 ** -24 + 2.0 ** -16
    tol = rel * (p @ values.abs()) + torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -25
    assert ((out.cpu().to(f8).view_as(ref) - ref).abs() <= tol).all()
    e = torch.exp(x - x.amax(-1, keepdim=True)) * vs.to(f8)[:, :, None]
    once = e.bfloat16().to(f8) @ v.to(f8) / torch.exp(x - x.amax(-1, keepdim=True)).sum(-1, keepdim=True)
    assert ((once - ref).abs() > tol).any()
