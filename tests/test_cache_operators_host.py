"""Host-side checks of the 8-bit cache and the shared-prefix attention (no GPU)."""

def test_quantised_cache_and_shared_prefix_entries_refuse_without_launching():
    """Arguments outside what the kernels handle come back as a status before any device call (the pointers are never
    dereferenced)."""
    import ctypes

    from olmo_amd import _lib

    h = _lib.lib()
    buf = ctypes.create_string_buffer(128)
    p = (ctypes.addressof(buf) + 15) & ~15
    EINVAL, EUNSUP = 1, 2

    def write(qkv=p, qw=p, kw=p, kq=p, kc=None, vc=None, Lfull=0, B=1, T=1, H=4, Hkv=2, hd=64, Lmax=8, n_pos=8, past=0, dev=None, dt=1):
        return h.olmo355_qknorm_rope_kvwrite_q8(qkv, qw, kw, p, p, p, kq, p, p, p, kc, vc, Lfull, B, T, H, Hkv, hd, Lmax, n_pos, past, dev, 1e-6,
                                                dt, None)

    for bad in (dict(qkv=None), dict(kw=None), dict(kc=p), dict(kq=p + 4), dict(qkv=p + 2), dict(B=0), dict(T=0), dict(H=3), dict(past=8),
                dict(past=-1), dict(T=9), dict(n_pos=0), dict(past=2**31 - 1), dict(kc=p, vc=p, Lfull=3, past=3), dict(kc=p, vc=p)):
        assert write(**bad) == EINVAL, bad
    for bad in (dict(hd=96), dict(dt=3), dict(dev=p, T=2), dict(H=256, Hkv=256, hd=128)):
        assert write(**bad) == EUNSUP, bad

    def read(kq=p, B=1, Hkv=2, hd=64, Lmax=8, start=0, n=8, Lout=8, at=0, dt=1):
        return h.olmo355_kv_read_q8(kq, p, p, p, p, p, B, Hkv, hd, Lmax, start, n, Lout, at, dt, None)

    for bad in (dict(kq=None), dict(n=0), dict(n=9), dict(start=1), dict(at=1), dict(start=-1), dict(Lout=7), dict(kq=p + 8),
                dict(start=2**31 - 1)):
        assert read(**bad) == EINVAL, bad
    assert read(hd=80) == EUNSUP and read(dt=7) == EUNSUP

    need = h.olmo355_attn_decode_q8_workspace_bytes(1, 32, 32, 128, 4096)
    assert need > 0 and h.olmo355_attn_decode_q8_workspace_bytes(0, 32, 32, 128, 4096) == 0
    assert h.olmo355_attn_decode_q8_workspace_bytes(64, 32, 32, 128, 4096) == 0  # one workgroup per (sequence, kv head)

    def decode(q=p, ws=p, wsb=need, B=1, H=32, Hkv=32, hd=128, Lmax=4096, past=9, n=4096, bias=None, stride=0, dt=1):
        return h.olmo355_attn_decode_q8(q, p, p, p, p, bias, p, ws, wsb, B, H, Hkv, hd, Lmax, past, None, n, stride, dt, None)

    for bad in (dict(q=None), dict(ws=None), dict(wsb=need - 1), dict(n=4097), dict(past=4096), dict(past=-1), dict(bias=p, stride=4095),
                dict(Hkv=5), dict(q=p + 8), dict(n=0)):
        assert decode(**bad) == EINVAL, bad
    assert decode(hd=256) == EUNSUP and decode(dt=9) == EUNSUP

    need = h.olmo355_attn_shared_prefix_workspace_bytes(4, 1, 32, 8, 128, 1000, 64, 1)
    assert need > 0 and h.olmo355_attn_shared_prefix_workspace_bytes(4, 1, 32, 8, 128, 0, 64, 1) == 0

    def prefix(q=p, ws=p, wsb=need, B=4, T=1, H=32, Hkv=8, hd=128, P=1000, Pmax=1000, Lmax=64, past=0, dev=None, n=64, bias=None,
               stride=0, dt=1):
        return h.olmo355_attn_shared_prefix(q, p, p, p, p, bias, p, ws, wsb, B, T, H, Hkv, hd, P, Pmax, Lmax, past, dev, n, stride, dt, None)

    for bad in (dict(q=None), dict(ws=None), dict(wsb=need - 1), dict(P=0), dict(P=1001), dict(n=65), dict(past=64), dict(past=-1),
                dict(T=65), dict(Hkv=7), dict(bias=p, stride=63), dict(q=p + 4), dict(past=2**31 - 1)):
        assert prefix(**bad) == EINVAL, bad
    assert prefix(hd=48) == EUNSUP and prefix(dt=5) == EUNSUP and prefix(dev=p, T=2, wsb=2**40) == EUNSUP


def test_a_workspace_for_n_keys_serves_fewer():
    """The runs a call takes depend on its count of keys; the workspace of the largest count holds every smaller one's."""
    from olmo_amd import _lib

    h = _lib.lib()
    for B, H, Hkv, hd in ((1, 32, 32, 128), (3, 40, 8, 128), (17, 8, 8, 64), (9, 32, 32, 32), (12, 32, 32, 128), (33, 8, 8, 64), (70, 48, 2, 32), (5, 8, 8, 128), (5, 1, 1, 128)):
        sizes = [h.olmo355_attn_decode_q8_workspace_bytes(B, H, Hkv, hd, n) for n in (1, 127, 129, 2048, 2049, 2100, 4096, 100000)]
        assert sizes == sorted(sizes), (B, H, Hkv, hd, sizes)
        for T in (1, 3, 40, 250):
            for dtype in (0, 1):
                sizes = [h.olmo355_attn_shared_prefix_workspace_bytes(B, T, H, Hkv, hd, P, n, dtype)
                         for P, n in ((1, 250), (100, 250), (129, 257), (129, 600), (1000, 1000), (2000, 1000), (2000, 5000), (60000, 5000), (60000, 9000))]
                assert sizes == sorted(sizes), (B, T, H, Hkv, hd, dtype, sizes)
