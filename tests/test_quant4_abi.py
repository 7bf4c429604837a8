"""Host side of the 4-bit operators: sizes, refusals before any launch, and where a cache position is found."""
import ctypes

import numpy as np
import pytest

P, I, Z, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float


def _cache(et, **kw):
    d = dict(num_pages=10, page=16, nkv=4, dh_qk=64, dh_v=64, k_codes=0x1000, k_params=0x2000, v_codes=0x3000,
             v_params=0x4000)
    d.update(kw)
    return et.KV4Desc(**d)


def _sizes(et, **kw):
    c, a, b = _cache(et, **kw), Z(0), Z(0)
    return et.lib().et_kv4_sizes(ctypes.byref(c), ctypes.byref(a), ctypes.byref(b)), a.value, b.value


def test_cache_sizes(et):
    assert _sizes(et) == (0, 10 * 4 * 16 * 32, 10 * 4 * 16 * 8)
    assert _sizes(et, dh_qk=16, dh_v=80) == (0, 10 * 4 * 16 * 48, 10 * 4 * 16 * 12)
    # past 2^32 bytes
    assert _sizes(et, num_pages=1 << 21, page=64, dh_qk=128)[1] == (1 << 21) * 4 * 64 * 64
    for bad, st in ((dict(page=8), -3), (dict(page=24), -3), (dict(dh_qk=40), -3), (dict(dh_v=144), -3),
                    (dict(nkv=0), -1), (dict(num_pages=0), -1), (dict(dh_v=-16), -1)):
        assert _sizes(et, **bad)[0] == st, bad
    assert et.lib().et_kv4_sizes(None, None, None) == -1


def test_cache_whose_bytes_pass_64_bits_is_refused(et):
    c = _cache(et, num_pages=2 ** 31 - 1, nkv=2 ** 21, page=2 ** 30)
    a, b = Z(0), Z(0)
    et.lib().et_kv4_sizes.argtypes = [P, P, P]
    assert et.lib().et_kv4_sizes(ctypes.addressof(c), ctypes.byref(a), ctypes.byref(b)) == -3
    c = _cache(et, num_pages=2 ** 31 - 1, nkv=1, page=16, dh_qk=128, dh_v=128)
    assert et.lib().et_kv4_sizes(ctypes.addressof(c), ctypes.byref(a), ctypes.byref(b)) == 0
    assert a.value == (2 ** 31 - 1) * 16 * 64


def test_positions_outside_the_table_or_the_cache_are_not_followed(et):
    fn = et.lib().et_debug_kv4_row
    fn.restype, fn.argtypes = ctypes.c_longlong, [P, P, I, ctypes.c_longlong, I]
    big = _cache(et, num_pages=1 << 24, page=64, nkv=16, dh_qk=128, dh_v=128)
    table = np.array([3, 0, 9, -1, 10, (1 << 24) - 1, 1 << 24, 2**31 - 1, -2**31], np.int32)
    at = table.ctypes.data_as(P)
    c = _cache(et)
    assert [fn(ctypes.byref(c), at, 9, 16 * e + 5, 2) for e in range(9)] == [
        (3 * 4 + 2) * 16 + 5, 2 * 16 + 5, (9 * 4 + 2) * 16 + 5, -1, -1, -1, -1, -1, -1]
    assert [fn(ctypes.byref(c), at, 3, p, 0) for p in (-1, -2**31, 47, 48, 2**31, 2**40)] == [-1, -1, 9 * 64 + 15, -1, -1, -1]
    # rows of a cache past 2^32 are found by 64-bit arithmetic
    assert fn(ctypes.byref(big), at, 9, 5 * 64 + 63, 15) == (((1 << 24) - 1) * 16 + 15) * 64 + 63
    assert fn(ctypes.byref(big), at, 9, 6 * 64, 0) == -1


def _write(et, fn="et_kv4_write_fwd", **kw):
    a = dict(c=_cache(et), K=0x5000, V=0x6000, ldk=256, ldv=256, table=0x7000, table_ld=4, start=None, n=None, batch=2,
             seq=3)
    a.update(kw)
    c = a.pop("c")
    f = getattr(et.lib(), fn)
    f.argtypes = [P, P, P, I, I, P, I, P, P, I, I, P]
    return f(ctypes.byref(c) if c is not None else None, *a.values(), None)


@pytest.mark.parametrize("fn", ["et_kv4_write_fwd", "et_kv4_read_fwd"])
def test_cache_calls_refuse(et, fn):
    before = et.lib().et_launch_count()
    for bad, st in ((dict(c=None), -1), (dict(K=None), -1), (dict(V=None), -1), (dict(table=None), -1),
                    (dict(table_ld=0), -1), (dict(batch=0), -1), (dict(seq=0), -1), (dict(ldk=248), -3),
                    (dict(ldv=260), -3), (dict(K=0x5008), -2), (dict(V=0x6002), -2),
                    (dict(c=_cache(et, k_codes=None)), -1), (dict(c=_cache(et, v_params=0x4008)), -2),
                    (dict(c=_cache(et, page=20)), -3), (dict(batch=1 << 20, seq=1 << 20), -3)):
        assert _write(et, fn, **bad) == st, bad
    assert et.lib().et_launch_count() == before


def _att(et, **kw):
    a = dict(c=_cache(et), Q=0x5000, Z=0x6000, table=0x7000, table_ld=4, kv_len=0x8000, q_len=None, batch=2, seq=1,
             nhead=8, ldq=512, ldz=512, max_len=64, kind=1, mask=None, ldm=0, scale=0.125, ws=0x10000, bytes=1 << 30)
    a.update(kw)
    c = a.pop("c")
    f = et.lib().et_attention_kv4_fwd
    f.argtypes = [P] * 4 + [I] + [P] * 2 + [I] * 7 + [P, I, F, P, Z, P]
    return f(ctypes.byref(c) if c is not None else None, *a.values(), None)


def test_attention_refuses(et):
    before = et.lib().et_launch_count()
    nan, inf = float("nan"), float("inf")
    for bad, st in ((dict(c=None), -1), (dict(Q=None), -1), (dict(Z=None), -1), (dict(table=None), -1),
                    (dict(kv_len=None), -1), (dict(batch=0), -1), (dict(seq=-1), -1), (dict(max_len=0), -1),
                    (dict(nhead=6), -3), (dict(nhead=0), -1), (dict(ldq=504), -3), (dict(ldz=510), -3),
                    (dict(max_len=65), -3), (dict(kind=2), -1), (dict(kind=7), -1), (dict(kind=3), -1),
                    (dict(kind=3, mask=0x9000, ldm=63), -1), (dict(scale=0.0), -1), (dict(scale=nan), -1),
                    (dict(scale=inf), -1), (dict(scale=1e-30), -1), (dict(scale=1e30), -1),
                    (dict(scale=-1.0), -1), (dict(Q=0x5004), -2), (dict(Z=0x6008), -2),
                    (dict(batch=65536), -3), (dict(seq=1 << 22, batch=1), -3),
                    (dict(seq=100000, batch=1, kind=7), -1),  # (the length is taken)
                    (dict(table_ld=4096, max_len=65536, ws=None), -6),
                    (dict(table_ld=4096, max_len=65536, bytes=64), -6),
                    (dict(table_ld=4096, max_len=65536, ws=0x10004), -2)):
        assert _att(et, **bad) == st, bad
    assert et.lib().et_launch_count() == before


def test_attention_workspace(et):
    """Scratch is only asked for where the sequence is split, never past 64 splits of it, and 0 for what is refused."""
    fn = et.lib().et_attention_kv4_workspace_bytes
    c = _cache(et)
    at = ctypes.addressof(c)
    assert fn(at, 64, 16, 8, 100000) == 0 and fn(at, 1, 1, 8, 16) == 0
    per_split = 8 * (64 + 2) * 4
    n = fn(at, 1, 1, 8, 100000)
    assert n > 0 and n % per_split == 0 and n // per_split <= 64
    assert fn(at, 1, 1, 7, 100000) == 0 and fn(None, 1, 1, 8, 1000) == 0


def test_linear_w4_refuses(et):
    lib = et.lib()
    a, b = Z(0), Z(0)
    lib.et_w4_sizes.argtypes = [I, I, I, P, P]
    assert lib.et_w4_sizes(208, 48, 64, ctypes.byref(a), ctypes.byref(b)) == 0
    assert (a.value, b.value) == (3 * 2 * 1024, 3 * 2 * 16 * 2 * 4)
    for bad in ((208, 48, 16), (208, 40, 64), (200, 48, 64)):
        assert lib.et_w4_sizes(*bad, ctypes.byref(a), ctypes.byref(b)) == -3
    assert lib.et_w4_sizes(0, 48, 64, ctypes.byref(a), ctypes.byref(b)) == -1

    def fwd(**kw):
        v = dict(codes=0x1000, params=0x2000, group=64, bias=None, X=0x3000, Y=0x4000, T=1, inn=128, out=64, act=0)
        v.update(kw)
        lib.et_linear_w4_fwd.argtypes = [P, P, I, P, P, P, I, I, I, I, P]
        return lib.et_linear_w4_fwd(*v.values(), None)

    before = lib.et_launch_count()
    for bad, st in ((dict(codes=None), -1), (dict(params=None), -1), (dict(X=None), -1), (dict(Y=None), -1),
                    (dict(T=0), -1), (dict(T=65535 * 128 + 1), -3), (dict(act=3), -1), (dict(group=48), -3), (dict(inn=120), -3), (dict(out=24), -3),
                    (dict(X=0x3008), -2), (dict(Y=0x4004), -2), (dict(codes=0x1008), -2), (dict(params=0x2004), -2)):
        assert fwd(**bad) == st, bad
    lib.et_w4_pack.argtypes = [P, I, I, I, P, P, P]
    assert lib.et_w4_pack(None, 128, 64, 64, 0x1000, 0x2000, None) == -1
    assert lib.et_w4_pack(0x3008, 128, 64, 64, 0x1000, 0x2000, None) == -2
    assert lib.et_w4_pack(0x3000, 128, 64, 65, 0x1000, 0x2000, None) == -3
    lib.et_w4_densify.argtypes = [P, P, I, I, I, P, P]
    assert lib.et_w4_densify(0x1000, 0x2000, 128, 64, 64, None, None) == -1
    assert lib.et_w4_densify(0x1000, 0x2000, 128, 60, 64, 0x3000, None) == -3
    assert lib.et_launch_count() == before


def test_linear_w4_plan(et):
    """Few tokens never expand the weights, many always do, and one side gives way to the other once."""
    few = et.lib().et_debug_w4_few_pay
    for inn, out in ((8192, 8192), (4096, 1024), (768, 2304), (1024, 4096), (512, 512), (16, 16), (8192, 28672)):
        chosen = [few(t, inn, out) for t in (1, 8, 16, 32, 64, 128, 512, 4096)]
        assert chosen[:2] == [1, 1] and chosen[-1] == 0, (inn, out, chosen)
        assert chosen == sorted(chosen, reverse=True), (inn, out, chosen)


def test_cached_layer_refuses(et):
    lib = et.lib()
    d = et.EncoderLayerDesc()
    for n, (lin, inn, out) in enumerate(((d.qkv, 256, 768), (d.o, 256, 256), (d.ffn1, 256, 512), (d.ffn2, 512, 256))):
        lin.in_, lin.out, lin.weight, lin.bias = inn, out, 0x100000 * (n + 1), None
    for n, name in enumerate(("ln1_gamma", "ln1_beta", "ln2_gamma", "ln2_beta")):
        setattr(d, name, 0x10000 * (n + 1))
    d.hidden, d.nhead, d.kdim, d.vdim, d.ff, d.act = 256, 4, 256, 256, 512, 2
    at = ctypes.addressof(d)
    good = _cache(et)
    size = lib.et_encoder_layer_cached_workspace_bytes
    need = size(at, ctypes.addressof(good), 2, 1, 64)
    assert need > 0
    before = lib.et_launch_count()
    for bad, want in ((dict(nkv=2), -3), (dict(dh_qk=48), -3), (dict(dh_v=32), -3), (dict(page=15), -3),
                      (dict(num_pages=0), -1), (dict(v_codes=None), -1), (dict(k_params=0x2004), -2)):
        c = _cache(et, **bad)
        assert lib.et_encoder_layer_cached_fwd(P(at), ctypes.byref(c), P(0x2000000), P(0x3000000), 2, 1, P(0x7000), 4,
                                               P(0x8000), P(0x9000), None, 64, P(0x40000000), Z(1 << 40),
                                               None) == want, bad

    def fwd(x=0x2000000, out=0x3000000, start=0x8000, kv=0x9000, ws=0x40000000, n=need, table=0x7000, most=64):
        return lib.et_encoder_layer_cached_fwd(P(at), ctypes.byref(good), P(x), P(out), 2, 1, P(table), 4, P(start),
                                               P(kv), None, most, P(ws), Z(n), None)

    assert fwd(table=None) == -1 and fwd(most=65) == -3
    # 4-bit weights that no kernel takes are found before the first launch
    keep = d.ffn2.format
    d.ffn2.format, d.ffn2.row_ptr, d.ffn2.nnz_tiles = et.FMT_W4, 0x700000, 48
    assert fwd() == -3
    d.ffn2.nnz_tiles, d.ffn2.row_ptr = 64, None
    assert fwd() == -1
    d.ffn2.format, d.ffn2.nnz_tiles = keep, 0

    assert fwd(x=None) == -1 and fwd(start=None) == -1 and fwd(kv=None) == -1
    assert fwd(ws=None) == -6 and fwd(n=need - 1) == -6
    assert fwd(x=0x2000008) == -2 and fwd(out=0x3000004) == -2 and fwd(ws=0x40000010) == -2
    assert lib.et_launch_count() == before


def test_python_wrappers_refuse_host_tensors(et):
    """No computation on the CPU: a tensor that is not on the current device is refused."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the CPU suite's case")
    with pytest.raises(Exception):
        et.W4Weight(torch.zeros((16, 128), dtype=torch.float16))


def test_cached_layer_refuses_its_weights_before_the_cache_is_written(et):
    """What a later product of the layer would refuse is found before the projection and the cache's write are
    launched, for every weight format and with the status of the product's own call."""
    lib = et.lib()
    d = et.EncoderLayerDesc()
    dims = (("qkv", 256, 768), ("o", 256, 256), ("ffn1", 256, 512), ("ffn2", 512, 256))
    for n, (name, inn, out) in enumerate(dims):
        lin = getattr(d, name)
        lin.in_, lin.out, lin.weight, lin.bias = inn, out, 0x100000 * (n + 1), None
    for n, name in enumerate(("ln1_gamma", "ln1_beta", "ln2_gamma", "ln2_beta")):
        setattr(d, name, 0x10000 * (n + 1))
    d.hidden, d.nhead, d.kdim, d.vdim, d.ff, d.act = 256, 4, 256, 256, 512, 2
    c = _cache(et)
    before = lib.et_launch_count()

    def fwd():
        return lib.et_encoder_layer_cached_fwd(P(ctypes.addressof(d)), ctypes.byref(c), P(0x2000000), P(0x3000000), 2, 1,
                                               P(0x7000), 4, P(0x8000), P(0x9000), None, 64, P(0x40000000), Z(1 << 40), None)

    arrays = dict(row_ptr=0x700000, row_off=0x710000, weight=0x720000, pk_mask=0x730000, pk_off=0x740000)
    wrong = {et.FMT_DENSE: ((dict(weight=None), -1), (dict(weight=0x720008), -2)),
             et.FMT_W4: ((dict(weight=0x720008), -2), (dict(row_ptr=0x700004), -2), (dict(row_ptr=None), -1)),
             et.FMT_1X16: ((dict(row_ptr=None), -1), (dict(row_off=None), -1), (dict(weight=0x720002), -2)),
             et.FMT_CSR: ((dict(row_ptr=None), -1), (dict(weight=None), -1), (dict(nnz_tiles=-1), -1)),
             et.FMT_ROW: ((dict(row_ptr=None), -1), (dict(weight=0x720008), -2), (dict(bias=0x720002), -2)),
             et.FMT_COL: ((dict(nnz_tiles=0), -1), (dict(nnz_tiles=60), -3), (dict(weight=0x720008), -2),
                          (dict(bias=0x720002), -2)),
             et.FMT_TILE: ((dict(row_off=None), -1), (dict(weight=0x720008), -2), (dict(bias=0x720002), -2)),
             et.FMT_TILE_PACKED: ((dict(pk_mask=None), -1), (dict(pk_off=None), -1), (dict(weight=0x720008), -2)),
             99: ((dict(), -1),)}
    for name, inn, out in dims[1:]:  # (the projection is the first to run in any case)
        lin = getattr(d, name)
        for fmt, cases in wrong.items():
            for bad, status in cases:
                for k, v in {**arrays, "bias": None, "nnz_tiles": 64, **bad}.items():
                    setattr(lin, k, v)
                lin.format = fmt
                assert fwd() == status, (name, fmt, bad)
        lin.format, lin.weight, lin.bias = et.FMT_DENSE, 0x720000, None
    for name in ("ln1_gamma", "ln1_beta", "ln2_gamma", "ln2_beta"):
        kept = getattr(d, name)
        for lin, fmt in ((d.o, et.FMT_1X16), (d.ffn2, et.FMT_1X16)):  # (no dense product: the LayerNorm runs by itself)
            lin.format, lin.nnz_tiles, lin.row_ptr, lin.row_off = fmt, 64, 0x700000, 0x710000
        setattr(d, name, kept + 2)
        assert fwd() == -2, name
        setattr(d, name, kept)
    # pruned hidden units: the pair runs as two dense products
    for lin, fmt in ((d.ffn1, et.FMT_ROW), (d.ffn2, et.FMT_COL)):
        lin.format, lin.nnz_tiles, lin.row_ptr, lin.weight, lin.bias = fmt, 64, 0x700000, 0x720000, None
    for lin, bad, status in ((d.ffn1, dict(weight=None), -1), (d.ffn1, dict(bias=0x720008), -2),
                             (d.ffn2, dict(weight=0x720008), -2)):
        kept = {k: getattr(lin, k) for k in bad}
        for k, v in bad.items():
            setattr(lin, k, v)
        assert fwd() == status, bad
        for k, v in kept.items():
            setattr(lin, k, v)
    assert lib.et_launch_count() == before
