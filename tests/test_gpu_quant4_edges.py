"""Ends of the 4-bit operators' ranges: values at the type's limits, NaN that is seen with next to no weight, groups of
unequal size, refusals that leave lengths and caches alone, and the cached layer in every weight format.

Tolerances count roundings as in test_gpu_quant4.py: an fp16 result is off by at most 2^-11 of its value (2^-25 near
zero), fp32 sums of n terms by n 2^-23 of the sum of their sizes."""
import numpy as np
import pytest

import quant4_ref as ref

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11
U32 = 2.0 ** -23


def _rng(seed):
    return np.random.default_rng(seed)


def _dev(a, cuda):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(cuda)


def _end_weights(rng, out, inn):
    """Rows with groups that reach the type's end in every way, in all sizes of group."""
    w = rng.normal(0, 0.03, (out, inn)).astype(np.float16)
    kind = np.arange(out) % 6
    u = rng.random((out, 32))
    w[kind == 0, :32] = (u * 65504)[kind == 0]               # s = 4368, 15 s = 65520
    w[kind == 1, :32] = ((2 * u - 1) * 65504)[kind == 1]     # s = 8736, 15 s + m = 65536
    w[kind == 2, :32] = (-u * 65504)[kind == 2]
    w[kind == 3, :32] = (65472 + 32 * (u > 0.5))[kind == 3]  # two neighbours
    for k, v in ((0, (0, 65504)), (1, (-65504, 65504)), (2, (-65504, 0)), (3, (65472, 65504))):
        w[kind == k, 0], w[kind == k, 5] = v
    return w


@pytest.mark.parametrize("few", [0, 1], ids=["expanded", "few"])
@pytest.mark.parametrize("T,inn,out,group", [(20, 256, 48, 32), (3, 144, 96, 64), (200, 272, 144, 128)])
def test_linear_w4_weights_at_the_types_end(et, cuda, few, T, inn, out, group):
    """s is rounded, so 15 s + m may lie beyond 65504; read back it is limited there, and no product may see an
    infinity: half a step of the type (2^-11) is all that the limit takes away."""
    rng = _rng(inn)
    w = _end_weights(rng, out, inn)
    c, s, m = ref.quantise(w, group)
    w64 = ref.values(c, s, m)[:, :inn]
    assert (w64 > 65504).any()
    x = rng.normal(0, 2.0 ** -13, (T, inn))
    x[:, :32] *= rng.random((T, 32)) < 0.2
    x[::2, :32] = 0
    x[1] = 0
    x = x.astype(np.float16)
    q = et.W4Weight(_dev(w, cuda), group)
    et.lib().et_debug_set_w4_few(few)
    try:
        y = et.linear_w4(_dev(x, cuda), q).cpu().numpy().astype(np.float64)
    finally:
        et.lib().et_debug_set_w4_few(-1)
    assert et.device_error() == 0 and not y[1].any()
    x64 = x.astype(np.float64)
    want = x64 @ w64.T
    parts = ref.values(c, s, np.zeros_like(m))[:, :inn] + np.abs(ref.values(np.zeros_like(c), s, m)[:, :inn])
    err = (inn + 16) * U32 * (np.abs(x64) @ parts.T) + (0 if few else HALF * (np.abs(x64) @ np.abs(w64).T))
    tol = HALF * np.abs(want) + 2.0 ** -25 + err
    bad = ~(np.abs(y - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], y[bad][:4], want[bad][:4])


def test_values_are_limited_at_both_ends(et, cuda):
    """Arrays that a caller fills may hold any finite (s, m): read back and made dense, values stay within +-65504."""
    rng = _rng(2)
    pairs = np.array([[4400, 0], [-4400, 0], [60000, -65504], [-60000, 65504], [-1, -65504], [1, 65504], [-65504, -65504],
                      [65504, 65504]], np.float16)
    c = rng.integers(0, 16, (16, 128)).astype(np.uint8)
    c[:, ::9] = 15
    sm = pairs[rng.integers(0, len(pairs), (16, 4))]
    s, m = sm[..., 0], sm[..., 1]
    want = ref.values(c, s, m).clip(-65504, 65504).astype(np.float16)
    codes, params = ref.w4_arrays(c, s, m, 32)
    q = et.W4Weight.from_arrays(_dev(codes, cuda), _dev(params, cuda), 128, 16, 32)
    assert np.array_equal(q.densify().cpu().numpy(), want)
    cache = et.KV4Cache(1, 16, 1, 128, 128, device=cuda)
    for codes_, params_, rows in ((cache.k_codes, cache.k_params, ref.k_rows), (cache.v_codes, cache.v_params, ref.v_rows)):
        codes_.copy_(_dev(rows(c)[None, None], cuda))
        params_.copy_(_dev(sm[None, None], cuda))
    k, v = et.kv4_read(cache, _dev(np.zeros((1, 1), np.int32), cuda), 1, 16)
    assert np.array_equal(k.cpu().numpy(), want) and np.array_equal(v.cpu().numpy(), want)
    # and the product over expanded weights sees no infinity
    x = np.zeros((9, 128), np.float16)
    x[np.arange(9), np.arange(9) * 14] = 2.0 ** -12
    et.lib().et_debug_set_w4_few(0)
    try:
        y = et.linear_w4(_dev(x, cuda), q).cpu().numpy()
    finally:
        et.lib().et_debug_set_w4_few(-1)
    assert np.array_equal(y, (want[:, np.arange(9) * 14].astype(np.float64).T * 2.0 ** -12).astype(np.float16))
    assert et.device_error() == 0


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("pattern", ["alone", "most"])
@pytest.mark.parametrize("length,parts", [(100, 1), (900, 4), (9000, 36)])
def test_attention_seen_nan_of_no_weight(et, cuda, length, parts, pattern, where):
    """A NaN in V reaches the rows that see it whatever its weight, in one block, a cluster or two kernels: its score
    lies 128 below the others' (e^-128 is no number of the exponential's), alone or with all tokens but the last 32."""
    rng = _rng(length)
    heads, dh, seq = 2, 64, 3
    pages = (length + 15) // 16
    cache = et.KV4Cache(pages, 16, heads, dh, dh, device=cuda)
    need = cache.workspace_bytes(1, seq, heads, length)
    assert (need > 0) == (parts > 4)
    table = _dev(np.arange(pages, dtype=np.int32)[None], cuda)
    k = rng.normal(0, 1, (length, heads * dh)).astype(np.float16)
    v = rng.normal(0, 1, (length, heads * dh)).astype(np.float16)
    at = {"first": 3, "middle": length // 2, "last": length - 2}[where]  # the last: hidden from query 0
    low = np.zeros(length, bool)
    low[at] = True
    if pattern == "most":
        low[: length - 32] = True
    k[low] = -16.0
    q = np.ones((seq, heads * dh), np.float16)
    bad = v.copy()
    bad[at, 70] = np.nan  # head 1, group 0
    et.kv4_write(cache, _dev(k, cuda), _dev(bad, cuda), table, None, 1, length)
    z = et.attention_kv4(cache, _dev(q, cuda), table, _dev(np.array([length], np.int32), cuda), 1, seq, heads, max_len=length)
    assert et.device_error() == 0
    z = z.cpu().numpy().astype(np.float64)
    seen = np.zeros(z.shape, bool)
    seen[[r for r in range(seq) if at <= length - seq + r], dh: dh + 32] = True
    assert np.array_equal(np.isnan(z), seen), np.argwhere(np.isnan(z) != seen)[:4]
    plain = [ref.values(*ref.quantise(x.reshape(length, heads, dh), 32)) for x in (k, v)]
    for h in range(heads):
        cols = slice(h * dh, (h + 1) * dh)
        want = ref.attention(q[:, cols].astype(np.float64), plain[0][:, h], plain[1][:, h], length - seq + 1 + np.arange(seq),
                             dh ** -0.5)
        # scores: fp32 sums of dh products, twice (c s and m apart), of at most |k| <= 16 and |q| = 1
        err = dh ** -0.5 * (dh + 8) * U32 * 2 * 16 * dh
        tol = HALF * np.abs(want) + 2.0 ** -25 + 8.0 * (2 * err + 64 * U32 + length ** 0.5 * 8 * U32)
        assert not (np.abs(z[:, cols] - want) > tol).any()


def test_attention_masked_nan_is_hidden_whatever_its_score(et, cuda):
    """-inf in an additive mask hides a NaN of V, the type's lowest value does not."""
    rng = _rng(31)
    length = 9000
    cache = et.KV4Cache(563, 16, 1, 64, 64, device=cuda)
    table = _dev(np.arange(563, dtype=np.int32)[None], cuda)
    x = rng.normal(0, 1, (length, 64)).astype(np.float16)
    x[5000, 40] = np.nan
    et.kv4_write(cache, _dev(np.nan_to_num(x), cuda), _dev(x, cuda), table, None, 1, length)
    q = _dev(rng.normal(0, 1, (2, 64)).astype(np.float16), cuda)
    mask = np.zeros((2, length), np.float16)
    mask[0, 5000], mask[1, 5000] = -np.inf, -65504.0
    z = et.attention_kv4(cache, q, table, _dev(np.array([length], np.int32), cuda), 1, 2, 1, max_len=length,
                         mask_kind=et.MASK_ADDITIVE, mask=_dev(mask, cuda)).cpu().numpy()
    want = np.zeros((2, 64), bool)
    want[1, 32:] = True
    assert et.device_error() == 0 and np.array_equal(np.isnan(z), want)


def test_mask_of_another_kind_is_refused(et, cuda):
    """A mask that would not be read is refused, not dropped."""
    import torch
    cache = et.KV4Cache(4, 16, 2, 64, 64, device=cuda)
    t = torch.zeros((1, 2), dtype=torch.int32, device=cuda)
    n = torch.ones(1, dtype=torch.int32, device=cuda)
    q = torch.zeros((1, 128), dtype=torch.float16, device=cuda)
    mask = torch.zeros((1, 32), dtype=torch.float16, device=cuda)
    for kw in ({}, {"mask_kind": et.MASK_CAUSAL}, {"mask_kind": et.MASK_NONE}):
        with pytest.raises(et.EtError):
            et.attention_kv4(cache, q, t, n, 1, 1, 2, mask=mask, **kw)
    et.attention_kv4(cache, q, t, n, 1, 1, 2, mask=mask, mask_kind=et.MASK_ADDITIVE)
    assert et.device_error() == 0


def _weights(et, seed, hidden, ff, qk=None):
    qk = hidden if qk is None else qk
    r = lambda n, shape, std: et.synth.normal(seed, n, shape, std)
    w = {"wqkv": r(1, (2 * qk + hidden, hidden), 0.04), "bqkv": r(2, (2 * qk + hidden,), 0.1),
         "wo": r(3, (hidden, hidden), 0.04), "bo": r(4, (hidden,), 0.1), "w1": r(5, (ff, hidden), 0.04),
         "b1": r(6, (ff,), 0.1), "w2": r(7, (hidden, ff), 0.04), "b2": r(8, (hidden,), 0.1),
         "ln1_g": 1 + r(9, (hidden,), 0.1), "ln1_b": r(10, (hidden,), 0.1), "ln2_g": 1 + r(11, (hidden,), 0.1),
         "ln2_b": r(12, (hidden,), 0.1)}
    return {k: np.asarray(v, np.float16) for k, v in w.items()}


def test_cached_stack_keeps_its_lengths_when_a_layer_refuses(et, cuda):
    """What only the library's own checks find - an x off a 16-byte boundary, a layer's weights - leaves the lengths
    as they were, and the same tokens can be passed again."""
    import torch
    hidden, batch, seq = 128, 2, 6
    layers = [et.EncoderLayer(_weights(et, 51 + i, hidden, 256), 2, et.ACT_GELU) for i in range(2)]
    stack = et.CachedStack(layers, batch, 33, page=16, device=cuda)
    x = _dev(_rng(19).normal(0, 1, (batch * seq, hidden)).astype(np.float16), cuda)
    first = stack.forward(x, seq).clone()
    want = stack.forward(x, seq).clone()
    stack.reset()
    assert torch.equal(stack.forward(x, seq), first)
    wide = torch.zeros(batch * seq * hidden + 8, dtype=torch.float16, device=cuda)
    off = wide[1: 1 + batch * seq * hidden].view(batch * seq, hidden)
    off.copy_(x)
    assert off.is_contiguous() and off.data_ptr() % 16
    with pytest.raises(et.EtError):
        stack.forward(off, seq)
    assert stack.kv_len.tolist() == [seq, seq] and stack.used == seq
    kept = layers[1].desc.ln1_gamma
    layers[1].desc.ln1_gamma = None  # the second layer refuses, after the first has run
    with pytest.raises(et.EtError):
        stack.forward(x, seq)
    layers[1].desc.ln1_gamma = kept
    assert stack.kv_len.tolist() == [seq, seq] and stack.used == seq
    assert torch.equal(stack.forward(x, seq), want) and et.device_error() == 0


@pytest.mark.parametrize("batch", [2, 130])
def test_cached_layer_takes_vectors_off_a_boundary(et, cuda, batch):
    """Where a Linear and its LayerNorm run as one kernel, bias, gamma and beta may lie anywhere: such layers are taken."""
    import torch
    from conftest import assert_close
    hidden, ff, nhead = 256, 512, 4
    w = _weights(et, 81, hidden, ff)
    layers = [et.EncoderLayer(w, nhead, et.ACT_GELU) for _ in range(2)]
    keep = []

    def off(name, size):
        t = torch.zeros(size + 8, dtype=torch.float16, device=cuda)
        t[1: 1 + size] = _dev(w[name], cuda)
        keep.append(t)
        return t.data_ptr() + 2

    d = layers[1].desc
    d.ln1_gamma, d.ln1_beta, d.ln2_gamma, d.ln2_beta = (off(n, hidden) for n in ("ln1_g", "ln1_b", "ln2_g", "ln2_b"))
    d.o.bias, d.ffn2.bias = off("bo", hidden), off("b2", hidden)
    x = _dev(_rng(3).normal(0, 1, (batch, hidden)).astype(np.float16), cuda)
    outs = []
    for layer in layers:
        stack = et.CachedStack([layer], batch, 16, page=16, device=cuda)
        outs.append(stack.forward(x, 1).clone())
    assert_close(outs[1].cpu().numpy(), outs[0].cpu().numpy(), "off a boundary")
    assert et.device_error() == 0


FORMATS = ["dense", "tile", "tile_packed", "1x16", "csr", "row", "col", "w4", "pair"]


def _in_format(et, cuda, w, fmt):
    """The weights pruned for a format, the layer in it, and the projection as an operator of its own."""
    import torch
    synth = et.synth
    w = dict(w)
    names = ("wqkv", "wo", "w1", "w2")
    out, ff = w["wqkv"].shape[0], w["w1"].shape[0]
    bias = _dev(w["bqkv"], cuda)
    keep = {n: np.ascontiguousarray(synth.choose_ids(7, i, w[n].shape[0 if fmt == "row" else 1], 0.5)).astype(np.int32)
            for i, n in enumerate(names)}
    hidden_units = keep["w2"]
    for i, n in enumerate(names):
        m = np.zeros_like(w[n])
        if fmt in ("tile", "tile_packed"):
            w[n] = np.asarray(synth.prune_tiles(w[n], 3, i, 0.5), np.float16)
        elif fmt in ("1x16", "csr"):
            w[n] = np.asarray(synth.prune_1x16(w[n], 3, i, 0.5), np.float16)
        elif fmt == "row":
            m[keep[n]] = w[n][keep[n]]
            w[n] = m
        elif fmt == "col":
            m[:, keep[n]] = w[n][:, keep[n]]
            w[n] = m
    if fmt == "pair":  # pruned hidden units of the feed-forward block
        m = np.zeros_like(w["w2"])
        m[:, hidden_units] = w["w2"][:, hidden_units]
        w["w2"] = m
    ids = lambda n: _dev(keep[n], cuda)
    d = lambda a: _dev(np.asarray(a), cuda)
    if fmt in ("tile", "tile_packed"):
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, tile_sparse="unpacked" if fmt == "tile" else "packed")
        rp, ro, tiles = synth.dense_to_tile(w["wqkv"])
        if fmt == "tile":
            a = [d(rp), d(ro), d(tiles)]
            project = lambda x: et.linear_tile(x, *a, out, bias)
        else:
            pk = et.PackedTiles(rp, ro, tiles, w["wqkv"].shape[1], out, cuda)
            project = lambda x: et.linear_tile_packed(x, pk, bias)
    elif fmt in ("1x16", "csr"):
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, formats={n: fmt for n in names})
        a = [d(v) for v in (synth.dense_to_1x16 if fmt == "1x16" else synth.dense_to_csr)(w["wqkv"])]
        op = et.linear_1x16 if fmt == "1x16" else et.linear_csr
        project = lambda x: op(x, *a, out, bias)
    elif fmt == "row":
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, formats={n: ("row", keep[n]) for n in names})
        rows, of = d(w["wqkv"][keep["wqkv"]]), ids("wqkv")
        project = lambda x: et.linear_row(x, of, rows, out, bias)
    elif fmt == "col":
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, formats={n: ("col", keep[n]) for n in names})
        cols, of = d(w["wqkv"][:, keep["wqkv"]]), ids("wqkv")
        project = lambda x: et.linear_col(x, of, cols, bias)
    elif fmt == "w4":
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, formats={n: "w4" for n in names})
        q = {n: et.W4Weight(d(w[n]), 128) for n in names}
        project = lambda x: et.linear_w4(x, q["wqkv"], bias)
        for n in names:
            w[n] = q[n].densify().cpu().numpy()
    else:
        formats = {"w1": ("row", hidden_units), "w2": ("col", hidden_units)} if fmt == "pair" else {}
        layer = et.EncoderLayer(w, 4, et.ACT_GELU, formats=formats)
        dense = d(w["wqkv"])
        project = lambda x: et.linear_dense(x, dense, bias)
    return w, layer, project


@pytest.mark.parametrize("fmt", FORMATS)
def test_cached_layer_in_every_format(et, cuda, fmt):
    """A prompt in two chunks of up to 50 tokens (the second on top of cached ones, across pages, one sequence a token
    short), then two single tokens: the cache to the bit of the format's own projection, what follows to the path's
    tolerance of the same layer in dense weights."""
    import torch
    from conftest import assert_close
    hidden, ff, nhead, batch, page, per = 256, 512, 4, 2, 16, 7
    most = page * per
    w, layer, project = _in_format(et, cuda, _weights(et, 71, hidden, ff), fmt)
    dev = {k: _dev(v, cuda) for k, v in w.items()}
    caches = [et.KV4Cache(batch * per, page, nhead, 64, 64, device=cuda) for _ in range(2)]
    table = _dev(_rng(1).permutation(batch * per).reshape(batch, per).astype(np.int32), cuda)
    kv = torch.zeros(batch, dtype=torch.int32, device=cuda)
    for step, (seq, new) in enumerate(((50, [50, 49]), (50, [49, 50]), (1, None), (1, None))):
        n = None if new is None else _dev(np.array(new, np.int32), cuda)
        x = _dev(_rng(step).normal(0, 1, (batch * seq, hidden)).astype(np.float16), cuda)
        start = kv.clone()
        kv += 1 if new is None else n
        assert int(kv.max()) <= most
        ws = torch.empty(layer.cached_workspace_bytes(caches[0], batch, seq, most), dtype=torch.uint8, device=cuda)
        out = torch.empty_like(x)
        layer.forward_cached(x, out, caches[0], table, start, kv, batch, seq, most, ws, n)
        qkv = project(x)
        et.kv4_write(caches[1], qkv[:, hidden: 2 * hidden], qkv[:, 2 * hidden:], table, start, batch, seq, new_len=n)
        for a in ("k_codes", "k_params", "v_codes", "v_params"):
            assert torch.equal(getattr(caches[0], a), getattr(caches[1], a)), (step, a)
        z = et.attention_kv4(caches[1], qkv[:, :hidden], table, kv, batch, seq, nhead, max_len=most, q_len=n)
        y = et.skip_layernorm(et.linear_dense(z, dev["wo"], dev["bo"]), x, dev["ln1_g"], dev["ln1_b"])
        f = et.linear_dense(y, dev["w1"], dev["b1"], et.ACT_GELU)
        want = et.skip_layernorm(et.linear_dense(f, dev["w2"], dev["b2"]), y, dev["ln2_g"], dev["ln2_b"])
        assert et.device_error() == 0
        live = np.concatenate([np.arange(seq) < (seq if new is None else new[b]) for b in range(batch)])
        assert_close(out.cpu().numpy()[live], want.cpu().numpy()[live], f"{fmt} step {step}")


@pytest.mark.parametrize("ratio", [2.0 ** -8, 2.0 ** -12])
@pytest.mark.parametrize("seq", [1, 12])
def test_attention_groups_of_unequal_size(et, cuda, seq, ratio):
    """Groups of a head whose ranges differ: p s enters the second product as two fp16 numbers, so to 2^-22 of itself or
    to 2^-24 of the row's largest over all groups, times a code's distance from 8; the sums' share as ever."""
    rng = _rng(seq)
    length, heads, dh = 300, 2, 128
    cache = et.KV4Cache(19, 16, heads, dh, dh, device=cuda)
    table = _dev(np.arange(19, dtype=np.int32)[None], cuda)
    k = rng.normal(0, 1, (length, heads * dh)).astype(np.float16)
    v = rng.normal(0, 1, (length, heads, 4, 32)) * ratio ** np.array([0, 1, 0.5, 1])[:, None]
    v = v.reshape(length, heads * dh).astype(np.float16)
    q = rng.normal(0, 1, (seq, heads * dh)).astype(np.float16)
    et.kv4_write(cache, _dev(k, cuda), _dev(v, cuda), table, None, 1, length)
    z = et.attention_kv4(cache, _dev(q, cuda), table, _dev(np.array([length], np.int32), cuda), 1, seq, heads,
                         max_len=length, mask_kind=et.MASK_NONE).cpu().numpy().astype(np.float64)
    assert et.device_error() == 0
    (ck, sk, mk), (cv, sv, mv) = (ref.quantise(x.reshape(length, heads, dh), 32) for x in (k, v))
    k64, v64 = ref.values(ck, sk, mk), ref.values(cv, sv, mv)
    sv, mv = sv.astype(np.float64), mv.astype(np.float64)
    for h in range(heads):
        qq = q[:, h * dh: (h + 1) * dh].astype(np.float64)
        score = qq @ k64[:, h].T * dh ** -0.5
        p = np.exp(score - score.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        big_k = float((16 * sk[:, h] + np.abs(mk[:, h])).max())
        err = dh ** -0.5 * (dh + 8) * U32 * big_k * np.abs(qq).sum(-1, keepdims=True)
        for g in range(4):
            cols = slice(32 * g, 32 * g + 32)
            want = p @ v64[:, h, cols]
            ps = p * sv[:, h, g]
            largest = (p[..., None] * sv[:, h]).max((1, 2))[:, None]
            halves = 8 * np.maximum(2.0 ** -22 * ps, 2.0 ** -24 * largest).sum(-1, keepdims=True)
            size = (p * (8 * sv[:, h, g] + np.abs(mv[:, h, g] + 8 * sv[:, h, g]))).sum(-1, keepdims=True)
            tol = HALF * np.abs(want) + 2.0 ** -25 + halves + size * (2 * err + (64 + length) * U32)
            off = np.abs(z[:, h * dh + 32 * g: h * dh + 32 * g + 32] - want)
            assert not (off > tol).any(), (h, g, off.max(), tol.min())
