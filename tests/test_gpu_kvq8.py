"""The 8-bit cache (write, read back, decode attention) against its definition in 64 bits.

Tolerances are sums of half steps: a rounding to a type is off by at most ``finfo.eps / 2`` relative to the value
(bf16 2^-8, fp16 2^-11, fp32 2^-24), an fp32 sum of n terms by at most ``n * 2^-24`` of the sum of their magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32MIN = torch.finfo(torch.float32).min
TINY = torch.finfo(torch.float32).tiny


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from olmo_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def _ops():
    from olmo_amd import ops

    return ops


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------
# write, read back
# ------------------------------------------------------------------------------------------------
def write_case(dtype, B, T, H, Hkv, hd, norm, n, seed=0, scale=0.7):
    gen = torch.Generator().manual_seed(seed)
    qkv = (scale * torch.randn(B, T, (H + 2 * Hkv) * hd, generator=gen)).to(dtype)
    qw = (1 + 0.1 * torch.randn(H * hd, generator=gen)).to(dtype) if norm else None
    kw = (1 + 0.1 * torch.randn(Hkv * hd, generator=gen)).to(dtype) if norm else None
    sin, cos = _ops().rope_tables(hd, 500000.0, n, "cpu")
    return qkv, qw, kw, sin, cos


def write_ref(qkv, qw, kw, sin, cos, B, T, H, Hkv, hd, past, eps):
    """q, k ``[B, T, heads, hd]``, v in 64 bits, and for q and k the sum of the magnitudes that a channel is made of."""
    f8 = torch.float64
    q, k, v = qkv.to(f8).split((H * hd, Hkv * hd, Hkv * hd), dim=-1)

    def turn(x, w, heads):
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.to(f8)
        x = x.reshape(B, T, heads, hd)
        s, c = (t[past:past + T].to(f8)[:, None, :] for t in (sin, cos))
        other = torch.cat((-x[..., hd // 2:], x[..., :hd // 2]), -1)
        return x * c + other * s, x.abs() * c.abs() + other.abs() * s.abs()

    return turn(q, qw, H), turn(k, kw, Hkv), v.reshape(B, T, Hkv, hd)


# fp32 from input to result: the sum of squares (at most 64 terms per thread, then 10 steps) gives its root half of 80 * 2^-24,
# normalisation, weight and rotation a few roundings more: below 2^-18 of the magnitudes that enter
REL32 = 2.0 ** -18


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,past,H,Hkv,hd,norm", [
    (1, 1, 0, 1, 1, 32, True), (2, 1, 9, 8, 8, 32, False), (3, 5, 2, 4, 2, 64, True), (1, 1, 30, 32, 32, 128, True),
    (2, 7, 0, 40, 8, 128, True), (1, 3, 11, 40, 40, 128, False), (1, 2, 1, 128, 1, 128, True), (2, 1, 3, 6, 3, 64, True),
    (1, 33, 0, 33, 33, 32, True),
])
def test_write_and_read_back(dev, dtype, B, T, past, H, Hkv, hd, norm):
    ops = _ops()
    n, eps = past + T + 5, 1e-6
    print("write_q8", dtype, B, T, past, H, Hkv, hd, norm, flush=True)
    qkv, qw, kw, sin, cos = write_case(dtype, B, T, H, Hkv, hd, norm, n, seed=B + T + H)
    (q8, qa), (k8, ka), v8 = write_ref(qkv, qw, kw, sin, cos, B, T, H, Hkv, hd, past, eps)
    c = ops.KVQ8.empty(B, Hkv, n, hd, dev)
    for t in (c.k, c.v):
        t.fill_(77)
    for t in (c.k_scale, c.v_scale):
        t.fill_(-5.0)
    kf, vf = (torch.full((B, Hkv, n - 2, hd), 9.0, dtype=dtype, device=dev) for _ in range(2))  # of a length of their own
    d = lambda t: None if t is None else t.to(dev)
    q = ops.qknorm_rope_kvwrite_q8(d(qkv), d(qw), d(kw), d(sin), d(cos), c, B, T, H, Hkv, hd, past, eps, kcache=kf, vcache=vf)
    h = half(dtype)
    assert ((q.cpu().double().view(B, T, H, hd) - q8).abs() <= h * q8.abs() + REL32 * qa + 2.0 ** -25).all()
    new = slice(past, past + T)
    kf, vf = kf.cpu(), vf.cpu()
    k8, ka, v8 = k8.transpose(1, 2), ka.transpose(1, 2), v8.transpose(1, 2)
    assert ((kf[:, :, new].double() - k8).abs() <= h * k8.abs() + REL32 * ka + 2.0 ** -25).all()
    assert torch.equal(vf[:, :, new].double(), v8)
    codes, scales = {"k": c.k.cpu(), "v": c.v.cpu()}, {"k": c.k_scale.cpu(), "v": c.v_scale.cpu()}
    off = {"k": REL32 * ka, "v": torch.zeros_like(v8)}
    for name, x in (("k", k8), ("v", v8)):
        s, code = scales[name][:, :, new].double(), codes[name][:, :, new].double()
        want = (x.abs().amax(-1) / 127).clamp_min(TINY)
        assert ((s - want).abs() <= 2.0 ** -23 * want + off[name].amax(-1) / 127).all(), name
        # rounding to a code: half a step; x / scale in fp32: two roundings of at most 127 steps
        assert ((code - x / s.unsqueeze(-1)).abs() <= 0.5 + 127 * 3 * 2.0 ** -24 + off[name] / s.unsqueeze(-1)).all(), name
        assert (code.abs() <= 127).all()
        rest = torch.ones(n, dtype=torch.bool)
        rest[new] = False
        assert (codes[name][:, :, rest] == 77).all() and (scales[name][:, :, rest] == -5.0).all(), "rows outside were written"
    assert (kf[:, :, past + T:] == 9).all() and (vf[:, :, :past] == 9).all()
    # the values of the codes: one fp32 product, one rounding
    k, v = ops.kv_read_q8(c, past, T, dtype)
    for got, name in ((k, "k"), (v, "v")):
        assert torch.equal(got.cpu(), (codes[name][:, :, new].float() * scales[name][:, :, new].unsqueeze(-1)).to(dtype))
    # into the same rows of caches
    ko, vo = (torch.full((B, Hkv, n + 3, hd), 3.0, dtype=dtype, device=dev) for _ in range(2))
    ops.kv_read_q8(c, past, T, dtype, out=(ko, vo))
    assert torch.equal(ko[:, :, new], k) and torch.equal(vo[:, :, new], v)
    assert (ko[:, :, past + T:] == 3).all() and (vo[:, :, :past] == 3).all()
    assert ops.kv_read_q8(c, n, 0, dtype)[0].shape == (B, Hkv, 0, hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,H,Hkv,hd", [(2, 2051, 40, 8, 128), (1, 4097, 24, 24, 128), (1, 4100, 14, 2, 128), (3, 1400, 5, 5, 32),
                                          (1, 4099, 72, 1, 128), (1, 4200, 32, 4, 64)])
def test_write_many_rows(dev, dtype, B, T, H, Hkv, hd):
    """The launch forms for many rows; the reference in 64 bits on the device."""
    ops = _ops()
    print("write_q8 rows", dtype, B, T, H, Hkv, hd, flush=True)
    qkv, qw, kw, sin, cos = (t.to(dev) for t in write_case(dtype, B, T, H, Hkv, hd, True, T, seed=T))
    (q8, qa), (k8, ka), v8 = write_ref(qkv, qw, kw, sin, cos, B, T, H, Hkv, hd, 0, 1e-6)
    c = ops.KVQ8.empty(B, Hkv, T, hd, dev)
    q = ops.qknorm_rope_kvwrite_q8(qkv, qw, kw, sin, cos, c, B, T, H, Hkv, hd, 0, 1e-6)
    # a lane adds up to 16 * 16 squares here before the exchange: half of (256 + 6) * 2^-24 for the root, below 2^-16
    rel = 2.0 ** -16
    assert ((q.double().view(B, T, H, hd) - q8).abs() <= half(dtype) * q8.abs() + rel * qa + 2.0 ** -25).all()
    for codes, scale, x, off in ((c.k, c.k_scale, k8, rel * ka), (c.v, c.v_scale, v8, torch.zeros_like(v8))):
        x, off, s = x.transpose(1, 2), off.transpose(1, 2), scale.double()
        assert ((s - x.abs().amax(-1) / 127).abs() <= 2.0 ** -23 * s + off.amax(-1) / 127).all()
        assert ((codes.double() - x / s.unsqueeze(-1)).abs() <= 0.5 + 127 * 3 * 2.0 ** -24 + off / s.unsqueeze(-1)).all()


def test_write_rows_of_zeros_tiny_huge_and_not_finite(dev):
    """Row maxima from nothing to the largest number; a row with an infinity or a NaN reads back as NaN, its neighbours
    are untouched by it."""
    ops = _ops()
    B, T, H, hd = 1, 8, 2, 64
    v = torch.randn(T, H, hd, generator=torch.Generator().manual_seed(3))
    v[0] = 0.0
    v[1] *= 1e-38
    v[2] *= 1e-42
    v[3] *= 1e37
    v[4, 0, 5], v[5, 1, 63], v[6, 0, 0] = float("inf"), float("nan"), float("-inf")
    qkv = torch.zeros(B, T, 3 * H * hd)
    qkv[0, :, 2 * H * hd:] = v.reshape(T, H * hd)
    sin, cos = ops.rope_tables(hd, 10000.0, T, dev)
    c = ops.KVQ8.empty(B, H, T, hd, dev)
    ops.qknorm_rope_kvwrite_q8(qkv.to(dev), None, None, sin, cos, c, B, T, H, H, hd, 0, 1e-6)
    k, got = ops.kv_read_q8(c, 0, T, torch.float32)
    assert (k == 0).all()
    got = got.cpu()[0].transpose(0, 1)  # [T, H, hd]
    bad = ~torch.isfinite(v).all(-1)
    assert bad.sum() == 3 and torch.isnan(got[bad]).all() and torch.isfinite(got[~bad]).all()
    step = (v.abs().amax(-1) / 127).clamp_min(TINY).unsqueeze(-1)
    assert ((got - v).abs() <= step * (0.5 + 2.0 ** -12))[~bad].all()
    assert (got[0] == 0).all() and (got[3].abs().amax(-1) > 1e37).all()


def test_write_position_from_the_device(dev):
    """A captured decode write replayed at successive positions equals writes at host positions; past the cache's
    end nothing is written."""
    ops = _ops()
    B, H, Hkv, hd, n, eps = 3, 8, 2, 64, 6, 1e-6
    rows = [write_case(torch.bfloat16, B, 1, H, Hkv, hd, True, n, seed=i) for i in range(n + 2)]
    _, qw, kw, sin, cos = [None if t is None else t.to(dev) for t in rows[0]]
    a, b = (ops.KVQ8.empty(B, Hkv, n, hd, dev) for _ in range(2))
    for c in (a, b):
        c.k.zero_(), c.v.zero_(), c.k_scale.zero_(), c.v_scale.zero_()
    x, pos = rows[0][0].to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    run = lambda: ops.qknorm_rope_kvwrite_q8(x, qw, kw, sin, cos, a, B, 1, H, Hkv, hd, 0, eps, past_len_dev=pos)
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = run()
    for i in range(n + 2):
        x.copy_(rows[i][0])
        pos.fill_(i)
        g.replay()
        if i < n:
            qe = ops.qknorm_rope_kvwrite_q8(x, qw, kw, sin, cos, b, B, 1, H, Hkv, hd, i, eps)
            assert torch.equal(q, qe)
    for s, t in ((a.k, b.k), (a.v, b.v), (a.k_scale, b.k_scale), (a.v_scale, b.v_scale)):
        assert torch.equal(s, t)


# ------------------------------------------------------------------------------------------------
# decode attention
# ------------------------------------------------------------------------------------------------
def codes_case(dev, B, Hkv, n, hd, seed):
    ops = _ops()
    gen = torch.Generator().manual_seed(seed)
    k = torch.randint(-127, 128, (B, Hkv, n, hd), generator=gen, dtype=torch.int8)
    v = torch.randint(-127, 128, (B, Hkv, n, hd), generator=gen, dtype=torch.int8)
    ks = 0.01 + 0.02 * torch.rand(B, Hkv, n, generator=gen)
    vs = 0.01 + 0.02 * torch.rand(B, Hkv, n, generator=gen)
    return ops.KVQ8(*(t.to(dev) for t in (k, v, ks, vs))), (k, v, ks, vs)


def decode_ref(q, host, keys, H, Hkv, hd, bias, dtype):
    """The output in 64 bits and the tolerance of a kernel that keeps scores, maxima and sums in fp32 and, for 16-bit types,
    rounds the weight of a key to bf16 once."""
    f8 = torch.float64
    k, v, ks, vs = (t[:, :, :keys].to(f8) for t in host)
    k, v = k * ks.unsqueeze(-1), v * vs.unsqueeze(-1)
    B, G = q.shape[0], H // Hkv
    qq = q.to(f8).view(B, Hkv, G, hd)
    x = qq @ k.transpose(-1, -2) / math.sqrt(hd)
    size = (qq.abs() @ k.abs().transpose(-1, -2) / math.sqrt(hd)).amax(-1, keepdim=True)
    if bias is not None:
        b = bias[:, None, None, :keys].to(f8)
        x = torch.where(b <= -1e30, torch.finfo(dtype).min, x + b)
        size = size + torch.where(b <= -1e30, 0.0, b.abs()).amax(-1, keepdim=True)
    p = torch.softmax(x, -1)
    out = (p @ v).reshape(B, 1, H * hd)
    rel = 2 * (hd + 8) * 2.0 ** -24 * size + (keys + 64) * 2.0 ** -24 + (0 if dtype == torch.float32 else 2.0 ** -8)
    tol = (rel * (p @ v.abs())).reshape(B, 1, H * hd)
    return out, half(dtype) * out.abs() + tol + 2.0 ** -25


DECODE = [
    (1, 1, 1, 1, 32), (2, 2, 4, 2, 64), (1, 31, 3, 3, 128), (2, 32, 8, 8, 32), (1, 33, 16, 16, 128), (3, 127, 6, 2, 64),
    (2, 128, 40, 8, 128), (1, 129, 8, 1, 128), (2, 517, 34, 2, 32), (1, 2049, 32, 32, 128), (5, 700, 4, 4, 64),
    (1, 4100, 48, 2, 128), (40, 300, 16, 16, 64), (70, 97, 32, 8, 32), (33, 2100, 8, 8, 32), (17, 2051, 16, 8, 64), (32, 515, 8, 8, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,keys,H,Hkv,hd", DECODE)
def test_decode(dev, dtype, B, keys, H, Hkv, hd):
    ops = _ops()
    print("decode_q8", dtype, B, keys, H, Hkv, hd, flush=True)
    n = keys + 37
    cache, host = codes_case(dev, B, Hkv, n, hd, seed=keys + H)
    q = torch.randn(B, 1, H * hd, generator=torch.Generator().manual_seed(keys)).to(dtype)
    # rows past the last key are whatever memory holds
    cache.k_scale[:, :, keys:], cache.v_scale[:, :, keys:] = float("nan"), float("inf")
    ws = ops.attn_decode_q8_workspace(B, H, Hkv, hd, n, dev).fill_(float("nan"))
    ref, tol = decode_ref(q, host, keys, H, Hkv, hd, None, dtype)
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, Hkv, hd, keys - 1, keys)
    assert out.dtype == dtype and ((out.cpu().double() - ref).abs() <= tol).all()
    pos = torch.tensor([keys - 1], dtype=torch.int32, device=dev)  # the position on the device, a grid for the whole cache
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, Hkv, hd, 0, n, past_len_dev=pos)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    # sequence 0 left-padded (its masked rows hold nothing finite), the last sequence with nothing but masked keys, and
    # a finite penalty
    bias = torch.zeros(B, n)
    bias[:, keys // 2] = -1.5
    bias[0, : keys // 3] = F32MIN
    ref_bias = bias.clone()
    host = [t.clone() for t in host]
    if B > 1:
        bias[-1] = float("-inf")
        ref_bias[-1] = F32MIN
    cache.k_scale[0, :, : keys // 3], cache.v_scale[0, :, : keys // 3] = float("inf"), float("nan")
    ref, tol = decode_ref(q, host, keys, H, Hkv, hd, ref_bias, dtype)
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, Hkv, hd, keys - 1, keys, key_bias=bias.to(dev))
    assert ((out.cpu().double() - ref).abs() <= tol).all()


def test_decode_extreme_scores(dev):
    """One key far above all others (its value comes out), scores far from zero, and a NaN row that is not masked."""
    ops = _ops()
    B, H, hd, keys = 1, 2, 64, 300
    cache, host = codes_case(dev, B, H, keys, hd, seed=1)
    q = torch.randn(B, 1, H * hd, generator=torch.Generator().manual_seed(0)).bfloat16()
    cache.k_scale[0, :, 200], host[2][0, :, 200] = 50.0, 50.0
    cache.k[0, :, 200], host[0][0, :, 200] = 127, 127
    q = q.abs()
    ws = ops.attn_decode_q8_workspace(B, H, H, hd, keys, dev)
    ref, tol = decode_ref(q, host, keys, H, H, hd, None, torch.bfloat16)
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, H, hd, keys - 1, keys)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    cache.v_scale[0, 0, 200] = float("nan")
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, H, hd, keys - 1, keys).cpu().view(H, hd)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_decode_is_deterministic_and_replays(dev):
    """The same bits from call to call, on another stream, and from a graph replayed at growing positions."""
    ops = _ops()
    B, H, Hkv, hd, n = 2, 8, 2, 128, 900
    cache, _ = codes_case(dev, B, Hkv, n, hd, seed=5)
    q = torch.randn(B, 1, H * hd, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    ws = ops.attn_decode_q8_workspace(B, H, Hkv, hd, n, dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    run = lambda: ops.attn_decode_q8(q, cache, ws, B, H, Hkv, hd, 0, n, past_len_dev=pos)
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    side = torch.cuda.Stream()
    ws2 = ops.attn_decode_q8_workspace(B, H, Hkv, hd, n, dev)
    for p in (0, 30, 31, 32, 500, 898, 899, 100):
        pos.fill_(p)
        g.replay()
        eager = run()
        assert torch.equal(out, eager)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = ops.attn_decode_q8(q, cache, ws2, B, H, Hkv, hd, 0, n, past_len_dev=pos)
        side.synchronize()
        assert torch.equal(other, eager)


def test_write_then_decode_long_cache(dev):
    """Rows whose byte offsets pass 32 bits: the last of many sequences in a long cache."""
    ops = _ops()
    B, H, hd, n = 36, 16, 128, 32768  # 2.4e9 codes
    c = ops.KVQ8.empty(B, H, n, hd, dev)
    past = n - 2
    qkv, qw, kw, sin, cos = write_case(torch.bfloat16, B, 1, H, H, hd, True, n, seed=9)
    d = lambda t: t.to(dev)
    c.k.fill_(1), c.v.zero_(), c.k_scale.fill_(0.0), c.v_scale.fill_(1.0)
    q = ops.qknorm_rope_kvwrite_q8(d(qkv), d(qw), d(kw), d(sin), d(cos), c, B, 1, H, H, hd, past, 1e-6)
    v = qkv[..., 2 * H * hd:].double().view(B, H, hd)
    k, got = ops.kv_read_q8(c, past, 1, torch.float32)
    assert ((got.cpu()[:, :, 0].double() - v).abs() <= v.abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
    ws = ops.attn_decode_q8_workspace(B, H, H, hd, n, dev)
    bias = torch.full((B, n), F32MIN, device=dev)
    bias[:, past] = 0.0  # only the new key: its value comes out (weight 1, exact; one rounding of scale and of the result)
    out = ops.attn_decode_q8(q, c, ws, B, H, H, hd, past, n, key_bias=bias).cpu().double().view(B, H, hd)
    got = got.cpu()[:, :, 0].double()
    assert ((out - got).abs() <= (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -15) * got.abs()).all()


# ------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------
def test_refusals(dev):
    ops = _ops()
    B, H, Hkv, hd, n = 2, 4, 2, 64, 16
    c = ops.KVQ8.empty(B, Hkv, n, hd, dev)
    qkv, qw, kw, sin, cos = (t.to(dev) for t in write_case(torch.bfloat16, B, 1, H, Hkv, hd, True, n))
    w = lambda **o: ops.qknorm_rope_kvwrite_q8(**{**dict(qkv=qkv, q_weight=qw, k_weight=kw, sin_tab=sin, cos_tab=cos, cache=c, B=B, T=1,
                                                         H=H, Hkv=Hkv, hd=hd, past_len=0, eps=1e-6), **o})
    w()
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    for bad in (dict(past_len=n), dict(past_len=-1), dict(k_weight=None), dict(kcache=torch.zeros(B, Hkv, n, hd, device=dev)),
                dict(past_len=3, kcache=qkv.new_zeros(B, Hkv, 3, hd), vcache=qkv.new_zeros(B, Hkv, 3, hd)),
                dict(Hkv=4), dict(H=5), dict(B=3), dict(q_weight=qw.float()), dict(sin_tab=sin.double()), dict(past_len_dev=pos.long()),
                dict(qkv=qkv.repeat(1, 2, 1), T=2, past_len_dev=pos), dict(qkv=qkv.repeat(1, 1, 2)[..., ::2])):
        with pytest.raises((ValueError, TypeError)):
            w(**bad)
    with pytest.raises(TypeError):
        ops.KVQ8(c.k.int(), c.v.int(), c.k_scale, c.v_scale)
    with pytest.raises(TypeError):
        ops.KVQ8(c.k, c.v, c.k_scale[:, :, :-1].contiguous(), c.v_scale)
    with pytest.raises(ValueError):
        ops.kv_read_q8(c, 10, 7, torch.bfloat16)
    with pytest.raises(TypeError):
        ops.kv_read_q8(c, 0, 1, torch.float64)
    with pytest.raises(ValueError):
        ops.kv_read_q8(c, 0, 4, torch.float32, out=(torch.zeros(B, Hkv, 3, hd, device=dev),) * 2)
    q = torch.zeros(B, 1, H * hd, dtype=torch.bfloat16, device=dev)
    ws = torch.zeros(1 << 16, device=dev)
    a = lambda **o: ops.attn_decode_q8(**{**dict(q=q, cache=c, ws=ws, B=B, H=H, Hkv=Hkv, hd=hd, past_len=3, n_keys_max=n), **o})
    a()
    big = ops.KVQ8.empty(B, Hkv, 2048, hd, dev)
    for bad in (dict(past_len=n), dict(n_keys_max=n + 1), dict(past_len=4, n_keys_max=4), dict(B=3), dict(hd=32),
                dict(key_bias=torch.zeros(B, n - 1, device=dev)), dict(key_bias=torch.zeros(B, n, dtype=torch.bfloat16, device=dev)),
                dict(past_len_dev=pos.long()), dict(cache=big, n_keys_max=2048, ws=ws[:16]), dict(q=q.double())):
        with pytest.raises((ValueError, TypeError)):
            a(**bad)
    # a buffer that does not start on 16 bytes
    odd = torch.zeros(B * H * hd + 1, dtype=torch.bfloat16, device=dev)[1:].view(B, 1, H * hd)
    with pytest.raises(ValueError):
        a(q=odd)
