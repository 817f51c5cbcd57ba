"""The 8-bit cache and the shared prefix as programs use them: very many runs of keys, launches sized for more keys than there
are, captured multi-token calls, calls on two streams at once, caches of more sequences than the batch, sequences interleaved."""
import pytest
import torch

from .test_gpu_kvq8 import codes_case, decode_ref, dev, write_case  # noqa: F401  (dev: the fixture)
from .test_gpu_model_caches import build, close32, ids
from .test_gpu_shared_prefix import call, case, reference

pytestmark = pytest.mark.gpu


def _ops():
    from olmo_amd import ops

    return ops


def test_one_row_over_very_many_runs(dev):
    """A single (sequence, head): hundreds of partial results are joined."""
    ops = _ops()
    B, H, hd, keys = 1, 1, 32, 33001
    cache, host = codes_case(dev, B, H, keys, hd, seed=3)
    q = torch.randn(B, 1, hd, generator=torch.Generator().manual_seed(4)).bfloat16()
    ws = ops.attn_decode_q8_workspace(B, H, H, hd, keys, dev).fill_(float("nan"))
    ref, tol = decode_ref(q, host, keys, H, H, hd, None, torch.bfloat16)
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, H, hd, keys - 1, keys)
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    for dtype, P, past in ((torch.float16, 30001, 20000), (torch.float32, 129, 40000), (torch.bfloat16, 40000, 0)):
        args = (B, 1, P, past, H, H, hd)
        x = case(dtype, *args, seed=5)
        ref, tol = reference(*x, *args)
        assert ((call(dev, *x, *args).cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 128), (torch.bfloat16, 32)])
@pytest.mark.parametrize("T,past", [(1, 0), (1, 70), (9, 5), (40, 65), (130, 3)])
def test_launch_for_more_keys_than_there_are(dev, dtype, hd, T, past):
    """n_keys_max beyond past_len + T: the rows behind are whatever memory holds."""
    B, P, H, Hkv = 2, 150, 8, 2
    args = (B, T, P, past, H, Hkv, hd)
    print("n_keys_max", dtype, args, flush=True)
    q, kp, vp, kc, vc = case(dtype, *args, seed=T, slack=190)
    kc[:, :, past + T:], vc[:, :, past + T:] = float("nan"), float("inf")
    ref, tol = reference(q, kp, vp, kc, vc, *args)
    for n in (past + T + 1, past + T + 190):
        out = call(dev, q, kp, vp, kc, vc, *args, n_keys_max=n)
        assert ((out.cpu().double() - ref).abs() <= tol).all()
        bias = torch.zeros(B, n + 2)
        out = call(dev, q, kp, vp, kc, vc, *args, bias=bias, n_keys_max=n)
        assert ((out.cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("B,T,P,past,H,Hkv,hd", [(1, 1000, 64, 0, 8, 1, 128), (1, 700, 1, 0, 3, 1, 64), (2, 520, 100, 1, 6, 2, 128)])
def test_more_parts_than_the_first_rows_have_tiles(dev, B, T, P, past, H, Hkv, hd):
    """A long prompt behind a short prefix: the keys are cut for the last rows, so the first rows' later parts are empty."""
    args = (B, T, P, past, H, Hkv, hd)
    print("empty parts", args, flush=True)
    for dtype in (torch.bfloat16, torch.float16):
        x = case(dtype, *args, seed=T)
        ref, tol = reference(*x, *args)
        assert ((call(dev, *x, *args).cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("T", [3, 50])
def test_captured_calls_of_several_tokens_and_two_streams(dev, T):
    """Both forms for several tokens replay, and two calls run at once on two streams, each with its workspace."""
    ops = _ops()
    B, H, Hkv, hd, P, past = 2, 8, 2, 128, 900, 33
    x = [[t.to(dev) for t in case(torch.bfloat16, B, T, P, past, H, Hkv, hd, seed=s, slack=0)] for s in (1, 2)]
    ws = [ops.attn_shared_prefix_workspace(B, T, H, Hkv, hd, P, past + T, torch.bfloat16, dev) for _ in x]
    run = lambda i: ops.attn_shared_prefix(*x[i], ws[i], B, T, H, Hkv, hd, P, past, past + T)
    first = [run(0).clone(), run(1).clone()]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(0)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        out.zero_()
        g.replay()
        assert torch.equal(out, first[0])
        torch.cuda.synchronize()
        both = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                both.append(run(i))
        torch.cuda.synchronize()
        assert torch.equal(both[0], first[0]) and torch.equal(both[1], first[1])


def test_cache_of_more_sequences_than_the_batch(dev):
    """Only the batch's sequences and rows are written; the others stay as they were."""
    ops = _ops()
    B, more, H, Hkv, hd, n, past, T = 2, 5, 8, 2, 64, 40, 7, 3
    qkv, qw, kw, sin, cos = (t.to(dev) for t in write_case(torch.bfloat16, B, T, H, Hkv, hd, True, n, seed=6))
    small, large = ops.KVQ8.empty(B, Hkv, n, hd, dev), ops.KVQ8.empty(more, Hkv, n, hd, dev)
    for c in (small, large):
        for t in (c.k, c.v):
            t.fill_(5)
        for t in (c.k_scale, c.v_scale):
            t.fill_(0.25)
    q = [ops.qknorm_rope_kvwrite_q8(qkv, qw, kw, sin, cos, c, B, T, H, Hkv, hd, past, 1e-6) for c in (small, large)]
    assert torch.equal(*q)
    for name in ("k", "v", "k_scale", "v_scale"):
        s, t = getattr(small, name), getattr(large, name)
        old = 5 if name in "kv" else 0.25
        assert torch.equal(s, t[:B]) and (t[B:] == old).all()
        assert (s[:, :, :past] == old).all() and (s[:, :, past + T:] == old).all() and (s[:, :, past:past + T] != old).any()
    x = torch.randn(B, 1, H * hd, device=dev).bfloat16()
    ws = ops.attn_decode_q8_workspace(B, H, Hkv, hd, n, dev)
    a, b = (ops.attn_decode_q8(x, c, ws, B, H, Hkv, hd, past + T - 1, past + T) for c in (small, large))
    assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_heavy_penalty_is_not_a_mask(dev, dtype):
    """The only key that is not masked carries a penalty near the end of fp16's range: its value comes out."""
    ops = _ops()
    B, H, Hkv, hd, keys = 2, 4, 2, 64, 200
    cache, host = codes_case(dev, B, Hkv, keys, hd, seed=8)
    q = torch.randn(B, 1, H * hd, generator=torch.Generator().manual_seed(9)).to(dtype)
    bias = torch.full((B, keys), float("-inf"))
    bias[0, 7], bias[1, 199] = -60000.0, -50000.0
    ws = ops.attn_decode_q8_workspace(B, H, Hkv, hd, keys, dev)
    out = ops.attn_decode_q8(q.to(dev), cache, ws, B, H, Hkv, hd, keys - 1, keys, key_bias=bias.to(dev)).cpu().double().view(B, Hkv, H // Hkv, hd)
    for b, at in ((0, 7), (1, 199)):  # weight 1, exact; scale and result are rounded, in fp32 or to the type (or bf16, twice)
        v = (host[1][b, :, at].double() * host[3][b, :, at, None].double())[:, None]
        assert ((out[b] - v).abs() <= (2.0 ** -15 + torch.finfo(dtype).eps / 2) * v.abs() + 2.0 ** -25).all()


def test_position_of_no_elements_is_refused(dev):
    ops = _ops()
    c = ops.KVQ8.empty(1, 2, 8, 64, dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.attn_decode_q8(torch.zeros(1, 1, 128, device=dev), c, ops.attn_decode_q8_workspace(1, 2, 2, 64, 8, dev), 1, 2, 2, 64, 0, 8,
                           past_len_dev=none)


def test_one_prompt_is_a_prefix_two_are_refused(dev):
    m = build("ln", torch.float32, dev)
    with pytest.raises(ValueError):
        m.share_prefix(ids(2, 10, dev))
    with pytest.raises(ValueError):
        m.share_prefix(ids(1, 10, dev).view(1, 1, 10))
    assert m.share_prefix(ids(10, 1, dev)[:, 0]).length == 10  # a strided row


@pytest.mark.parametrize("kind", ["ln", "gqa"])
def test_prefixes_interleaved_with_other_sequences(dev, kind):
    """Steps behind two prefixes and without one, in turn, in one model: each gives what it gives alone."""
    m = build(kind, torch.float32, dev)
    heads = [ids(1, 20, dev, seed=1), ids(1, 77, dev, seed=2)]
    prefixes = [m.share_prefix(h) for h in heads] + [None]
    x, steps = ids(2, 5, dev, seed=3), [ids(2, k, dev, seed=4 + k) for k in (1, 6, 1)]

    def alone(p):
        out = m(x, use_cache=True, prefix=p)
        r = [out.logits]
        for s in steps:
            out = m(s, past_key_values=out.attn_key_values, use_cache=True)
            r.append(out.logits)
        return r

    want = [alone(p) for p in prefixes]
    outs = [m(x, use_cache=True, prefix=p) for p in prefixes]
    got = [[o.logits] for o in outs]
    for s in steps:
        outs = [m(s, past_key_values=o.attn_key_values, use_cache=True) for o in outs]
        for g, o in zip(got, outs):
            g.append(o.logits)
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    for h, w in zip(heads, want):  # and what the whole prompt gives
        whole = torch.cat((h.expand(2, -1), x, *steps), 1)
        assert close32(torch.cat(w, 1), m(whole).logits[:, h.shape[1]:])


@pytest.mark.parametrize("kind,dtype", [("ln", torch.float32), ("gqa", torch.float32)])
def test_generate_behind_a_prefix_with_padded_rest(dev, kind, dtype):
    m = build(kind, dtype, dev)
    head, x = ids(1, 40, dev, seed=5), ids(3, 9, dev, seed=6)
    mask = torch.ones(3, 9, dtype=torch.int64)
    mask[0, :4], mask[2, :8] = 0, 0
    prefix = m.share_prefix(head)
    a = m.generate(x, attention_mask=mask, max_steps=10, prefix=prefix, stop_at_eos=False)
    b = m.generate(x, attention_mask=mask, max_steps=10, prefix=prefix, stop_at_eos=False, use_graph=False)
    whole = torch.cat((head.expand(3, 40), x), 1)
    ref = m.generate(whole, attention_mask=torch.cat((torch.ones(3, 40, dtype=torch.int64), mask), 1), max_steps=10, stop_at_eos=False)
    assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.token_ids, ref.token_ids)
    assert close32(a.scores, ref.scores)
