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
