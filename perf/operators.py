"""Measured cases of the operators around the key/value cache of a serving process: the 8-bit cache (written with the
QK-norm and the rotation, read back, attended to by one new token per sequence) and attention of a batch whose sequences
share one prefix.  ``run`` is the plain form of an operator (float32 torch, rounded once at the end), or with ``own`` the
call into ``olmo_amd.ops``; ``exact`` is the definition in 64 bits.

Head counts and sizes are those of the presets of ``olmo_amd/config.py`` (8 heads of 32; 16, 32, 40 heads of 128), with
grouped keys as ``n_kv_heads`` allows; listed lengths run up to the presets' 4096 positions, drawn ones to four times that
(``max_cache_len`` is the user's)."""
import math

import torch

own = False

THETA, EPS = 500000.0, 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MASKED = torch.finfo(torch.float32).min  # what a padding mask becomes in the key bias


def listed():
    return [
        # one token of one user appended to the cache of a 7B-shaped layer: the call's own latency
        {"name": "write 1x1 32 heads", "op": "write", "dtype": "bf16", "B": 1, "T": 1, "H": 32, "Hkv": 32, "hd": 128, "past": 2047},
        # one token each of a batch of 64 users, 13B-shaped heads with grouped keys
        {"name": "write 64x1 40/8 heads", "op": "write", "dtype": "fp16", "B": 64, "T": 1, "H": 40, "Hkv": 8, "hd": 128, "past": 777},
        # a prompt of 2048 tokens, 7B
        {"name": "write 1x2048 32 heads", "op": "write", "dtype": "bf16", "B": 1, "T": 2048, "H": 32, "Hkv": 32, "hd": 128, "past": 0},
        # a batch of prompts of odd length, 13B
        {"name": "write 8x1021 40 heads", "op": "write", "dtype": "bf16", "B": 8, "T": 1021, "H": 40, "Hkv": 40, "hd": 128, "past": 3},
        # one user at a short context, 1B: the smallest attention call
        {"name": "decode 1x517 16 heads", "op": "decode", "dtype": "bf16", "B": 1, "H": 16, "Hkv": 16, "hd": 128, "keys": 517, "pad": 0},
        # one user at the presets' longest context, 7B
        {"name": "decode 1x4096 32 heads", "op": "decode", "dtype": "bf16", "B": 1, "H": 32, "Hkv": 32, "hd": 128, "keys": 4096, "pad": 0},
        # a left-padded batch with grouped keys
        {"name": "decode 16x2049 40/8 heads", "op": "decode", "dtype": "fp16", "B": 16, "H": 40, "Hkv": 8, "hd": 128, "keys": 2049, "pad": 300},
        # a large batch at long context, 7B: what the 8-bit cache is for
        {"name": "decode 48x4001 32 heads", "op": "decode", "dtype": "bf16", "B": 48, "H": 32, "Hkv": 32, "hd": 128, "keys": 4001, "pad": 0},
        # four users under a short instruction, the float32 preset
        {"name": "prefix 4x1 517 8 heads", "op": "prefix", "dtype": "fp32", "B": 4, "T": 1, "H": 8, "Hkv": 8, "hd": 32, "prefix": 517, "past": 20, "pad": 0},
        # a batch under a long common prompt, 7B
        {"name": "prefix 32x1 4001 32 heads", "op": "prefix", "dtype": "bf16", "B": 32, "T": 1, "H": 32, "Hkv": 32, "hd": 128, "prefix": 4001, "past": 128, "pad": 0},
        # grouped keys, questions of different length (left-padded)
        {"name": "prefix 16x1 2049 40/8 heads", "op": "prefix", "dtype": "fp16", "B": 16, "T": 1, "H": 40, "Hkv": 8, "hd": 128, "prefix": 2049, "past": 300, "pad": 100},
        # the questions themselves: a prefill of 8 x 250 tokens behind the prefix
        {"name": "prefix 8x250 2048 32 heads", "op": "prefix", "dtype": "bf16", "B": 8, "T": 250, "H": 32, "Hkv": 32, "hd": 128, "prefix": 2048, "past": 0, "pad": 0},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["write", "decode", "prefix"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        hd = rng.choice([32, 64, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8, 16, 32])
        H = Hkv * rng.choice([1, 1, 2, 3, 5, 8])
        if H > 64:
            continue
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if op == "write":  # values read back in 16 bits: the form a 16-bit model keeps
            c = {"op": op, "dtype": "fp16" if dtype == "fp32" else dtype, "B": spread(1, 64), "T": rng.choice([1, spread(2, 4096)]),
                 "H": H, "Hkv": Hkv, "hd": hd, "past": rng.choice([0, spread(1, 2048)])}
        elif op == "decode":
            keys = spread(1, 16384)
            c = {"op": op, "dtype": dtype, "B": spread(1, 64), "H": H, "Hkv": Hkv, "hd": hd, "keys": keys,
                 "pad": rng.choice([0, rng.randrange(keys)])}
        else:
            past = rng.choice([0, spread(1, 1024)])
            c = {"op": op, "dtype": dtype, "B": spread(1, 64), "T": rng.choice([1, 1, spread(2, 512)]), "H": H, "Hkv": Hkv, "hd": hd,
                 "prefix": spread(1, 16384), "past": past, "pad": rng.choice([0, rng.randrange(past + 1)])}
        if _cost(c) <= most:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / (1.5e14 if case["dtype"] == "fp32" else 2.5e15))


def work(case):
    c, e = case, torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    B, H, Hkv, hd = c["B"], c["H"], c["Hkv"], c["hd"]
    if c["op"] == "write":
        rows = B * c["T"]
        codes = 2 * Hkv * (hd + 4)  # a token's codes and scales
        # the projection in, q out, the codes written and read once, the values read back out
        nbytes = rows * ((H + 2 * Hkv) * hd * e + H * hd * e + 2 * codes + 2 * Hkv * hd * e) + (H + Hkv) * hd * e + c["T"] * hd * 8
        return {"bytes": nbytes, "flops": rows * (H + 2 * Hkv) * hd * 8}
    if c["op"] == "decode":
        bias = 4 * B * c["keys"] if c["pad"] else 0
        return {"bytes": 2 * B * Hkv * c["keys"] * (hd + 4) + 2 * B * H * hd * e + bias, "flops": 4 * B * H * c["keys"] * hd}
    T, P, past = c["T"], c["prefix"], c["past"]
    seen = sum(past + t + 1 for t in range(T))
    nbytes = 2 * P * Hkv * hd * e + 2 * B * Hkv * (past + T) * hd * e + 2 * B * T * H * hd * e + (4 * B * (past + T) if c["pad"] else 0)
    return {"bytes": nbytes, "flops": 4 * B * H * hd * (T * P + seen)}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _quantised(gen, shape, spread, dev):
    """Rows of normal values with a few strong channels, as cached keys have them, in 8 bits: codes and row scales."""
    x = torch.randn(shape, generator=gen, device=dev)
    x[..., :: max(2, shape[-1] // 4)] *= spread
    s = (x.abs().amax(-1) / 127.0).clamp_min(torch.finfo(torch.float32).tiny)
    return (x / s.unsqueeze(-1)).round_().to(torch.int8), s


def _padding(gen, B, n, pad, dev):
    """Left padding: sequence b has its first ``0 .. pad`` keys masked."""
    if not pad:
        return None
    first = torch.randint(0, pad + 1, (B, 1), generator=gen, device=dev)
    return torch.where(torch.arange(n, device=dev) < first, MASKED, 0.0).contiguous()


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, B, H, Hkv, hd = DTYPES[c["dtype"]], c["B"], c["H"], c["Hkv"], c["hd"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    s = {"case": dict(c)}
    if c["op"] == "write":
        T, past = c["T"], c["past"]
        n = past + T + 7
        s["qkv"] = normal(B, T, (H + 2 * Hkv) * hd, scale=0.7)
        s["qw"], s["kw"] = 1.0 + normal(H * hd, scale=0.1), 1.0 + normal(Hkv * hd, scale=0.1)
        inv = 1.0 / (THETA ** (torch.arange(0, hd, 2, dtype=torch.float) / hd))
        ang = torch.arange(n, dtype=torch.float)[:, None] * inv[None, :]
        ang = torch.cat((ang, ang), dim=-1)
        s["sin"], s["cos"] = ang.sin().contiguous().to(dev), ang.cos().contiguous().to(dev)
        s["kq"], s["vq"] = (torch.zeros(B, Hkv, n, hd, dtype=torch.int8, device=dev) for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros(B, Hkv, n, dtype=torch.float32, device=dev) for _ in range(2))
    elif c["op"] == "decode":
        n = c["keys"]
        s["q"] = normal(B, 1, H * hd)
        s["kq"], s["ks"] = _quantised(gen, (B, Hkv, n, hd), 3.0, dev)
        s["vq"], s["vs"] = _quantised(gen, (B, Hkv, n, hd), 1.0, dev)
        s["bias"] = _padding(gen, B, n, c["pad"], dev)
        if own:
            from olmo_amd import ops
            s["ws"] = ops.attn_decode_q8_workspace(B, H, Hkv, hd, n, dev)
    else:
        T, P, n = c["T"], c["prefix"], c["past"] + c["T"]
        s["q"] = normal(B, T, H * hd)
        s["kp"], s["vp"] = normal(Hkv, P, hd), normal(Hkv, P, hd)
        s["kc"], s["vc"] = normal(B, Hkv, n, hd), normal(B, Hkv, n, hd)
        s["bias"] = _padding(gen, B, n, c["pad"], dev)
        if own:
            from olmo_amd import ops
            s["ws"] = ops.attn_shared_prefix_workspace(B, T, H, Hkv, hd, P, n, dtype, dev)
    if own and c["op"] in ("write", "decode"):
        from olmo_amd import ops
        s["cache"] = ops.KVQ8(s["kq"], s["vq"], s["ks"], s["vs"])
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
def _normed_rotated(x, w, heads, hd, sin, cos):
    """``[B, T, heads * hd]``: RMS norm over the whole width, then the rotation of every head."""
    B, T, _ = x.shape
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    x = x.view(B, T, heads, hd)
    half = torch.cat((-x[..., hd // 2 :], x[..., : hd // 2]), dim=-1)
    return x * cos[:, None, :] + half * sin[:, None, :]


def _codes(x):
    s = (x.abs().amax(-1) / 127.0).clamp_min(torch.finfo(torch.float32).tiny)
    return (x / s.unsqueeze(-1)).round().to(torch.int8), s


def _write(s):
    c = s["case"]
    B, T, H, Hkv, hd, past = c["B"], c["T"], c["H"], c["Hkv"], c["hd"], c["past"]
    q, k, v = s["qkv"].split((H * hd, Hkv * hd, Hkv * hd), dim=-1)
    sin, cos = s["sin"][past : past + T], s["cos"][past : past + T]
    q = _normed_rotated(q, s["qw"], H, hd, sin, cos).to(s["qkv"].dtype).view(B, T, H * hd)
    k = _normed_rotated(k, s["kw"], Hkv, hd, sin, cos).transpose(1, 2)
    v = v.float().view(B, T, Hkv, hd).transpose(1, 2)
    new = slice(past, past + T)
    s["kq"][:, :, new], s["ks"][:, :, new] = _codes(k)
    s["vq"][:, :, new], s["vs"][:, :, new] = _codes(v)
    k = (s["kq"][:, :, new].float() * s["ks"][:, :, new].unsqueeze(-1)).to(q.dtype)
    v = (s["vq"][:, :, new].float() * s["vs"][:, :, new].unsqueeze(-1)).to(q.dtype)
    return {"q": q, "k": k, "v": v}


def _decode(s):
    c = s["case"]
    B, H, Hkv, hd = c["B"], c["H"], c["Hkv"], c["hd"]
    q = s["q"].float().view(B, Hkv, H // Hkv, hd)
    k = s["kq"].float() * s["ks"].unsqueeze(-1)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    if s["bias"] is not None:
        b = s["bias"][:, None, None, :]
        x = torch.where(b <= -1e30, torch.finfo(s["q"].dtype).min, x + b)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, s["vq"].float() * s["vs"].unsqueeze(-1)) / p.sum(-1, keepdim=True)
    return o.view(B, 1, H * hd).to(s["q"].dtype)


def _prefix(s):
    c = s["case"]
    B, T, H, Hkv, hd, P, past = c["B"], c["T"], c["H"], c["Hkv"], c["hd"], c["prefix"], c["past"]
    G, n = H // Hkv, past + T
    q = s["q"].float().view(B, T, Hkv, G, hd).permute(0, 2, 3, 1, 4)                        # [B, Hkv, G, T, hd]
    shared = q.permute(1, 0, 2, 3, 4).reshape(Hkv, B * G * T, hd)
    xp = torch.matmul(shared, s["kp"].float().transpose(-1, -2).contiguous()).view(Hkv, B, G, T, P).permute(1, 0, 2, 3, 4)
    xo = torch.matmul(q.reshape(B, Hkv, G * T, hd), s["kc"].float().transpose(-1, -2).contiguous()).view(B, Hkv, G, T, n)
    at = torch.arange(n, device=q.device)
    hidden = (at[None, :] > past + torch.arange(T, device=q.device)[:, None]).view(1, 1, 1, T, n)
    xo = xo / math.sqrt(hd)
    if s["bias"] is not None:
        b = s["bias"].view(B, 1, 1, 1, n)
        hidden = hidden | (b <= -1e30)
        xo = xo + b
    xo = xo.masked_fill(hidden, float("-inf"))
    x = torch.cat((xp / math.sqrt(hd), xo), dim=-1)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    pp = p[..., :P].permute(1, 0, 2, 3, 4).reshape(Hkv, B * G * T, P)
    o = torch.matmul(pp, s["vp"].float()).view(Hkv, B, G, T, hd).permute(1, 0, 2, 3, 4)
    o = o + torch.matmul(p[..., P:].reshape(B, Hkv, G * T, n), s["vc"].float()).view(B, Hkv, G, T, hd)
    o = o / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H * hd).to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        from olmo_amd import ops
        if c["op"] == "write":
            q = ops.qknorm_rope_kvwrite_q8(s["qkv"], s["qw"], s["kw"], s["sin"], s["cos"], s["cache"], c["B"], c["T"], c["H"], c["Hkv"],
                                           c["hd"], c["past"], EPS)
            k, v = ops.kv_read_q8(s["cache"], c["past"], c["T"], s["qkv"].dtype)
            return {"q": q, "k": k, "v": v}
        if c["op"] == "decode":
            return ops.attn_decode_q8(s["q"], s["cache"], s["ws"], c["B"], c["H"], c["Hkv"], c["hd"], c["keys"] - 1, c["keys"],
                                      key_bias=s["bias"])
        return ops.attn_shared_prefix(s["q"], s["kp"], s["vp"], s["kc"], s["vc"], s["ws"], c["B"], c["T"], c["H"], c["Hkv"], c["hd"],
                                      c["prefix"], c["past"], c["past"] + c["T"], key_bias=s["bias"])
    return {"write": _write, "decode": _decode, "prefix": _prefix}[c["op"]](s)


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c, f8 = case, torch.float64
    B, H, Hkv, hd = c["B"], c["H"], c["Hkv"], c["hd"]
    G = H // Hkv
    if c["op"] == "write":
        T, past = c["T"], c["past"]
        x = s["qkv"].to(f8).view(B, T, H + 2 * Hkv, hd)
        sin, cos = (s[n][past : past + T].to(f8)[:, None, :] for n in ("sin", "cos"))

        def turned(y, w):
            y = y / ((y ** 2).flatten(2).mean(-1)[..., None, None] + EPS).sqrt() * w.to(f8).view(-1, hd)
            a, b = y.chunk(2, dim=-1)
            return torch.cat((a * cos[..., : hd // 2] - b * sin[..., : hd // 2], b * cos[..., hd // 2 :] + a * sin[..., hd // 2 :]), dim=-1)

        def stored(y):
            step = y.abs().amax(-1, keepdim=True) / 127
            return ((y / step).round() * step).transpose(1, 2)

        return {"q": turned(x[:, :, :H], s["qw"]).reshape(B, T, H * hd), "k": stored(turned(x[:, :, H : H + Hkv], s["kw"])),
                "v": stored(x[:, :, H + Hkv :])}
    if c["op"] == "decode":
        out = torch.empty(B, H, hd, dtype=f8, device=s["q"].device)
        for b in range(B):
            k = s["kq"][b].to(f8) * s["ks"][b].to(f8)[..., None]
            v = s["vq"][b].to(f8) * s["vs"][b].to(f8)[..., None]
            x = (s["q"][b].to(f8).view(Hkv, G, 1, hd) * hd ** -0.5 @ k.transpose(1, 2)[:, None]).squeeze(2)
            if s["bias"] is not None:
                x = torch.where(s["bias"][b] <= -1e30, torch.finfo(s["q"].dtype).min, x + s["bias"][b].to(f8))
            out[b] = (torch.softmax(x, -1) @ v).view(H, hd)
        return out.view(B, 1, H * hd)
    T, P, past = c["T"], c["prefix"], c["past"]
    out = torch.empty(B, T, H, hd, dtype=f8, device=s["q"].device)
    kpos = torch.cat((torch.full((P,), -1, device=out.device), torch.arange(past + T, device=out.device)))
    hide = kpos[None, :] > past + torch.arange(T, device=out.device)[:, None]
    for b in range(B):
        off = hide
        bias = torch.zeros(P + past + T, dtype=f8, device=out.device)
        if s["bias"] is not None:
            bias[P:] = s["bias"][b].to(f8)
            off = hide | (bias <= -1e30)
        for h in range(Hkv):
            k = torch.cat((s["kp"][h], s["kc"][b, h])).to(f8)
            v = torch.cat((s["vp"][h], s["vc"][b, h])).to(f8)
            q = s["q"][b].view(T, H, hd)[:, h * G : (h + 1) * G].to(f8)
            x = (q.reshape(T * G, hd) @ k.T / hd ** 0.5).view(T, G, -1) + bias
            x = x.masked_fill(off[:, None, :], float("-inf"))
            out[b, :, h * G : (h + 1) * G] = (torch.softmax(x, -1).view(T * G, -1) @ v).view(T, G, hd)
    return out.view(B, T, H * hd)
