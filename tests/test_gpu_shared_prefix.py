"""Attention of a batch that shares a prefix against its definition in 64 bits; tolerances as in test_gpu_kvq8.py."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32MIN = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    from olmo_amd import _lib

    _lib.lib()
    return torch.device("cuda:0")


def _ops():
    from olmo_amd import ops

    return ops


def case(dtype, B, T, P, past, H, Hkv, hd, seed, slack=5):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen).to(dtype)
    n = past + T + slack
    return r(B, T, H * hd), r(Hkv, P + slack, hd), r(Hkv, P + slack, hd), r(B, Hkv, n, hd), r(B, Hkv, n, hd)


def reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd, bias=None):
    """Output in 64 bits; tolerance of a kernel that keeps scores, maxima and sums in fp32 and rounds the weight of a key once
    to the activation type (fp16: weights below its range are off by at most 2^-25 each, next to a sum that is at least 1)."""
    f8, dtype, n, G = torch.float64, q.dtype, past + T, H // Hkv
    out, tol = (torch.empty(B, T, H, hd, dtype=f8) for _ in range(2))
    at = torch.arange(n)
    hide = torch.cat((torch.zeros(T, P, dtype=torch.bool), at[None, :] > past + torch.arange(T)[:, None]), 1)
    for b in range(B):
        add, off = torch.zeros(P + n, dtype=f8), hide
        if bias is not None:
            masked = bias[b, :n] <= -1e30
            add[P:] = torch.where(masked, 0.0, bias[b, :n]).to(f8)
            off = hide | torch.cat((torch.zeros(P, dtype=torch.bool), masked))
        for h in range(Hkv):
            k = torch.cat((kp[h, :P], kc[b, h, :n])).to(f8)
            v = torch.cat((vp[h, :P], vc[b, h, :n])).to(f8)
            dead = off.all(0)
            k[dead], v[dead] = 0.0, 0.0
            qq = q[b].view(T, H, hd)[:, h * G:(h + 1) * G].to(f8)
            x = qq @ k.T / math.sqrt(hd) + add
            size = (qq.abs() @ k.abs().T / math.sqrt(hd) + add.abs()).amax(-1, keepdim=True)
            p = torch.softmax(x.masked_fill(off[:, None, :], float("-inf")), -1)
            rel = 2 * (hd + 8) * 2.0 ** -24 * size + (P + n + 64) * 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
            out[b, :, h * G:(h + 1) * G] = p @ v
            tol[b, :, h * G:(h + 1) * G] = rel * (p @ v.abs()) + (2.0 ** -25 * (~off).sum(-1)[:, None, None] * v.abs().max() if dtype == torch.float16 else 0)
    out, tol = out.view(B, T, H * hd), tol.view(B, T, H * hd)
    return out, tol + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -25


def call(dev, q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd, bias=None, **kw):
    ops = _ops()
    n = kw.pop("n_keys_max", past + T)
    ws = ops.attn_shared_prefix_workspace(B, T, H, Hkv, hd, P, n, q.dtype, dev).fill_(float("nan"))
    d = lambda t: t.to(dev)
    return ops.attn_shared_prefix(d(q), d(kp), d(vp), d(kc), d(vc), ws, B, T, H, Hkv, hd, P, past, n,
                                  key_bias=None if bias is None else bias.to(dev), **kw)


SHAPES = [  # B, T, P, past, H, Hkv, hd
    (1, 1, 1, 0, 1, 1, 32), (2, 1, 31, 0, 4, 2, 64), (4, 1, 32, 5, 8, 8, 32), (3, 1, 33, 31, 16, 16, 128), (5, 1, 517, 100, 6, 2, 64),
    (16, 1, 300, 40, 40, 8, 128), (33, 1, 1100, 3, 4, 4, 128), (70, 1, 129, 64, 8, 1, 128), (2, 1, 4100, 700, 16, 16, 128),
    (2, 2, 5, 0, 2, 2, 32), (3, 17, 65, 0, 4, 4, 64), (2, 33, 40, 12, 8, 2, 128), (1, 130, 300, 0, 4, 4, 128), (4, 65, 129, 63, 3, 3, 64),
    (2, 257, 64, 1, 2, 1, 128), (1, 300, 1000, 100, 2, 2, 32),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,P,past,H,Hkv,hd", SHAPES)
def test_shared_prefix(dev, dtype, B, T, P, past, H, Hkv, hd):
    print("shared_prefix", dtype, B, T, P, past, H, Hkv, hd, flush=True)
    q, kp, vp, kc, vc = case(dtype, B, T, P, past, H, Hkv, hd, seed=P + T)
    n = past + T
    kp[:, P:], vp[:, P:], kc[:, :, n:], vc[:, :, n:] = (float("nan"),) * 4  # behind the last rows: whatever memory holds
    ref, tol = reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd)
    out = call(dev, q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd)
    assert out.dtype == dtype and ((out.cpu().double() - ref).abs() <= tol).all()
    if T == 1:  # the position on the device, a grid for the whole cache
        pos = torch.tensor([past], dtype=torch.int32, device=dev)
        out = call(dev, q, kp, vp, kc, vc, B, T, P, 0, H, Hkv, hd, n_keys_max=kc.shape[2], past_len_dev=pos)
        assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,P,past,H,Hkv,hd", [(3, 1, 50, 40, 4, 2, 64), (4, 1, 129, 200, 16, 16, 128), (2, 1, 7, 0, 2, 2, 32),
                                                 (3, 40, 33, 0, 4, 2, 128), (2, 150, 64, 9, 2, 2, 64), (2, 70, 100, 3, 8, 4, 32)])
def test_shared_prefix_masked_own_keys(dev, dtype, B, T, P, past, H, Hkv, hd):
    """Left padding of different depth, a finite penalty, a sequence whose own keys are all masked: masked keys weigh
    nothing although their rows hold NaN and infinities."""
    print("shared_prefix masked", dtype, B, T, P, past, H, Hkv, hd, flush=True)
    q, kp, vp, kc, vc = case(dtype, B, T, P, past, H, Hkv, hd, seed=T + past)
    n = past + T
    bias = torch.zeros(B, n + 3)
    bias[:, n // 2] = -2.25
    for b in range(B):
        bias[b, : (b * n) // B] = F32MIN if b % 2 else float("-inf")
    bias[-1] = F32MIN
    for b in range(B):
        m = bias[b, :n] <= -1e30
        kc[b, :, :n][:, m], vc[b, :, :n][:, m] = float("nan"), float("inf")
    ref, tol = reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd, bias)
    out = call(dev, q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd, bias)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,P,past", [(3, 1, 300, 65), (2, 70, 130, 10)])
def test_shared_prefix_equals_a_copied_prefix(dev, dtype, B, T, P, past):
    """The attention the framework has, over caches that begin with a copy of the prefix: both are within their tolerance of
    the definition, so within twice that of each other."""
    ops = _ops()
    H, Hkv, hd = 8, 4, 128
    q, kp, vp, kc, vc = case(dtype, B, T, P, past, H, Hkv, hd, seed=7, slack=0)
    ref, tol = reference(q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd)
    out = call(dev, q, kp, vp, kc, vc, B, T, P, past, H, Hkv, hd)
    kf = torch.cat((kp.expand(B, Hkv, P, hd), kc), 2).contiguous().to(dev)
    vf = torch.cat((vp.expand(B, Hkv, P, hd), vc), 2).contiguous().to(dev)
    if T == 1:
        ws = ops.attn_decode_workspace(B, H, hd, P + past + 1, dev)
        old = ops.attn_decode(q.to(dev), kf, vf, ws, B, H, Hkv, hd, P + past, P + past + 1)
    else:
        old = ops.attn_prefill(q.to(dev), kf, vf, B, T, H, Hkv, hd, P + past)
    assert ((out.double() - old.double()).cpu().abs() <= 2 * tol).all()


def test_shared_prefix_replays(dev):
    """The same bits from call to call, on another stream, and from a graph replayed at growing positions."""
    ops = _ops()
    B, H, Hkv, hd, P, n = 3, 8, 2, 128, 200, 300
    q, kp, vp, kc, vc = (t.to(dev) for t in case(torch.bfloat16, B, 1, P, n - 1, H, Hkv, hd, seed=2, slack=0))
    ws = ops.attn_shared_prefix_workspace(B, 1, H, Hkv, hd, P, n, q.dtype, dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    run = lambda w: ops.attn_shared_prefix(q, kp, vp, kc, vc, w, B, 1, H, Hkv, hd, P, 0, n, past_len_dev=pos)
    run(ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(ws)
    side, ws2 = torch.cuda.Stream(), torch.empty_like(ws)
    for p in (0, 31, 32, 150, 299, 7):
        pos.fill_(p)
        g.replay()
        eager = run(ws)
        assert torch.equal(out, eager)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            other = run(ws2)
        side.synchronize()
        assert torch.equal(other, eager)


def test_shared_prefix_refusals(dev):
    ops = _ops()
    B, T, P, past, H, Hkv, hd = 2, 2, 10, 3, 4, 2, 64
    q, kp, vp, kc, vc = (t.to(dev) for t in case(torch.bfloat16, B, T, P, past, H, Hkv, hd, seed=0))
    n = past + T
    ws = ops.attn_shared_prefix_workspace(B, T, H, Hkv, hd, P, n, q.dtype, dev)
    a = lambda **o: ops.attn_shared_prefix(**{**dict(q=q, kprefix=kp, vprefix=vp, kcache=kc, vcache=vc, ws=ws, B=B, T=T, H=H, Hkv=Hkv,
                                                     hd=hd, prefix_len=P, past_len=past, n_keys_max=n), **o})
    a()
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    for bad in (dict(prefix_len=0), dict(prefix_len=kp.shape[1] + 1), dict(past_len=past + 1), dict(past_len=-1), dict(n_keys_max=99),
                dict(n_keys_max=1), dict(q=q.float()), dict(kprefix=kp[0]), dict(vprefix=vp[:, :-1].contiguous()), dict(B=3),
                dict(kcache=kc[:, :, :, :32].contiguous()), dict(past_len_dev=pos), dict(ws=ws[:4]), dict(H=2),
                dict(key_bias=torch.zeros(B, n - 1, device=dev)), dict(kcache=kc.transpose(1, 2))):
        with pytest.raises((ValueError, TypeError)):
            a(**bad)
