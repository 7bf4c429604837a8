"""The 4-bit cache, the attention over it and the 4-bit Linear against plain 64-bit computations.

Tolerances count roundings: an fp16 result is off by at most half a step, 2^-11 of its value (2^-25 near
zero); fp32 sums of n terms by n 2^-23 of the sum of their sizes (a tensor core cuts where others
round); what the fp16 result and the sums do not explain is named where it is added."""
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


def _table(rng, batch, per, pages):
    return rng.permutation(pages)[: batch * per].reshape(batch, per).astype(np.int32)


def _fill(et, cache, rng, cuda, scale=1.0, nan=None):
    """Random contents of the whole cache; returns the codes and (s, m) in plain order [pages, nkv, page, ...].
    Features past a head's width have code 0, groups past it s = m = 0."""
    out = []
    for codes, params, d, rows in ((cache.k_codes, cache.k_params, cache.dh_qk, ref.k_rows),
                                   (cache.v_codes, cache.v_params, cache.dh_v, ref.v_rows)):
        lead = tuple(codes.shape[:3])
        ng = codes.shape[-1] // 16
        c = rng.integers(0, 16, lead + (32 * ng,), dtype=np.uint8)
        c[..., d:] = 0
        s = (scale * rng.uniform(0.1, 0.35, lead + (ng,))).astype(np.float16)
        m = (-7.5 * s + scale * rng.normal(0, 0.3, lead + (ng,))).astype(np.float16)
        s[..., -(-d // 32):] = 0
        m[..., -(-d // 32):] = 0
        if nan is not None:  # positions that no call may look at
            s[nan], m[nan] = np.nan, np.nan
        codes.copy_(_dev(rows(c), cuda))
        params.copy_(_dev(np.stack([s, m], -1), cuda))
        out.append((c, s, m))
    return out


def _gather(plain, table, b, n, head, d, page):
    c, s, m = plain
    pos = np.arange(n)
    at = table[b][pos // page], head, pos % page
    return ref.values(c[at], s[at], m[at])[:, :d]


# ---- writing and reading -----------------------------------------------------------------------

def _awkward(rng, shape):
    """Values on borders between codes, constant groups, tiny ranges, and the type's ends."""
    x = rng.normal(0, 1, shape)
    kind = rng.integers(0, 7, shape[0])
    x[kind == 1] = rng.integers(-8, 8, x[kind == 1].shape) * 0.5     # halves: many exact ties
    x[kind == 2] = 0.75                                              # constant
    x[kind == 3] = rng.integers(-40, 40, x[kind == 3].shape) * 2.0 ** -24   # subnormal numbers
    x[kind == 4] *= 30000.0
    x[kind == 5] += 900.0                                            # a range of few steps of the type
    x = x.clip(-65504, 65504).astype(np.float16)
    x[kind == 6, ::7] = -65504.0
    x[kind == 6, 1::7] = 65504.0
    return x


CACHE_CASES = [  # batch, seq, nkv, dh_qk, dh_v, page, start
    (1, 1, 1, 16, 16, 16, [0]), (2, 5, 3, 64, 64, 16, [0, 13]), (3, 33, 2, 48, 64, 32, [7, 0, 100]),
    (2, 70, 4, 128, 128, 64, [1, 63]), (1, 17, 2, 80, 112, 16, [15]), (2, 9, 1, 96, 32, 128, [120, 0]),
    (1, 40, 5, 16, 128, 16, [3]), (64, 1, 12, 64, 64, 16, None),
]


@pytest.mark.parametrize("case", CACHE_CASES, ids=str)
def test_write_and_read_are_exact(et, cuda, case):
    """Codes, scales and minima are those of the exact quotient, whatever the values; nothing else is
    touched; reading back gives fp16(c s + m) to the bit."""
    import torch
    batch, seq, nkv, dk, dv, page, start = case
    rng = _rng(batch * 1000 + seq)
    start = np.array(start if start is not None else rng.integers(0, 200, batch), np.int32)
    n = rng.integers(0, seq + 1, batch).astype(np.int32)
    n[0] = seq
    per = int((start.max() + seq + page - 1) // page)
    pages = batch * per + 2
    cache = et.KV4Cache(pages, page, nkv, dk, dv, device=cuda)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0xA5)
    for t in (cache.k_params, cache.v_params):
        t.fill_(-3.0)
    table = _table(rng, batch, per, pages)
    T = batch * seq
    fused = _awkward(rng, (T, nkv * (dk + dv) + 24))  # K and V as views of a wider buffer
    fused[rng.random(T) < 0.05, 5] = np.nan
    fused[rng.random(T) < 0.05, nkv * dk + 18] = np.inf
    f = _dev(fused, cuda)
    k, v = f[:, 8: 8 + nkv * dk], f[:, 16 + nkv * dk: 16 + nkv * (dk + dv)]
    tb, st, nl = _dev(table, cuda), _dev(start, cuda), _dev(n, cuda)
    et.kv4_write(cache, k, v, tb, st, batch, seq, new_len=nl)
    assert et.device_error() == 0
    ng = (max(dk, dv) + 31) // 32
    want = {}
    for name, x, d, rows in (("k", fused[:, 8: 8 + nkv * dk], dk, ref.k_rows),
                             ("v", fused[:, 16 + nkv * dk: 16 + nkv * (dk + dv)], dv, ref.v_rows)):
        c, s, m = ref.quantise(x.reshape(T, nkv, d), 32)
        pad = ng - s.shape[-1]
        c = np.pad(c, ((0, 0), (0, 0), (0, 32 * pad)))
        s, m = (np.pad(a, ((0, 0), (0, 0), (0, pad))) for a in (s, m))
        codes = np.full((pages, nkv, page, 16 * ng), 0xA5, np.uint8)
        params = np.full((pages, nkv, page, ng, 2), -3.0, np.float16)
        r = rows(c)
        for b in range(batch):
            for i in range(n[b]):
                p = start[b] + i
                codes[table[b][p // page], :, p % page] = r[b * seq + i]
                params[table[b][p // page], :, p % page] = np.stack([s[b * seq + i], m[b * seq + i]], -1)
        got_c = getattr(cache, name + "_codes").cpu().numpy()
        got_p = getattr(cache, name + "_params").cpu().numpy()
        assert np.array_equal(got_c, codes), name
        assert np.array_equal(got_p, params, equal_nan=True), name
        want[name] = ref.to_f16(ref.values(c, s, m)[..., :d]).reshape(T, -1)
    out = tuple(torch.full((T, nkv * d), 7.0, dtype=torch.float16, device=cuda) for d in (dk, dv))
    et.kv4_read(cache, tb, batch, seq, start=st, length=nl, out=out)
    assert et.device_error() == 0
    rows = np.concatenate([np.arange(seq) < n[b] for b in range(batch)])
    for got, name in zip(out, ("k", "v")):
        g = got.cpu().numpy()
        assert np.array_equal(g[rows], want[name][rows], equal_nan=True), name
        assert (g[~rows] == 7.0).all(), name


def test_write_without_starts_or_lengths(et, cuda):
    rng = _rng(3)
    cache = et.KV4Cache(6, 16, 2, 32, 32, device=cuda)
    x = _dev(rng.normal(0, 1, (40, 64)).astype(np.float16), cuda)
    tb = _dev(np.array([[5, 0], [2, 3]], np.int32), cuda)
    et.kv4_write(cache, x, x, tb, None, 2, 20)
    k, v = et.kv4_read(cache, tb, 2, 20)
    assert et.device_error() == 0
    c, s, m = ref.quantise(x.cpu().numpy().reshape(40, 2, 32), 32)
    want = ref.to_f16(ref.values(c, s, m)).reshape(40, 64)
    assert np.array_equal(k.cpu().numpy(), want) and np.array_equal(v.cpu().numpy(), want)


def test_bad_pages_are_reported_and_not_followed(et, cuda):
    """Where the kernels would look is checked without a GPU (test_quant4_abi.py); here: the report, the
    neighbours' data, and zeros from what could not be read."""
    import torch
    rng = _rng(4)
    cache = et.KV4Cache(4, 16, 2, 64, 64, device=cuda)
    x = _dev(rng.normal(0, 1, (2 * 32, 128)).astype(np.float16), cuda)
    good = _dev(np.array([[0, 1], [2, 3]], np.int32), cuda)
    et.kv4_write(cache, x, x, good, None, 2, 32)
    kept = [t.clone() for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params)]
    bad = _dev(np.array([[0, 4], [-1, 3]], np.int32), cuda)
    start = _dev(np.array([16, 0], np.int32), cuda)
    et.kv4_write(cache, x[:32], x[:32], bad, start, 2, 16)
    assert et.device_error() == 601 and et.device_error() == 0
    for t, was in zip((cache.k_codes, cache.k_params, cache.v_codes, cache.v_params), kept):
        assert torch.equal(t, was)
    k, _ = et.kv4_read(cache, bad, 2, 32)
    assert et.device_error() == 601
    whole, _ = et.kv4_read(cache, good, 2, 32)
    k, whole = k.view(2, 32, -1), whole.view(2, 32, -1)
    assert torch.equal(k[0, :16], whole[0, :16]) and torch.equal(k[1, 16:], whole[1, 16:])
    assert not k[0, 16:].any() and not k[1, :16].any()
    # past the table: dropped, and attention cuts the sequence at max_len
    et.kv4_write(cache, x[:32], x[:32], good, _dev(np.array([32, -20], np.int32), cuda), 2, 16)
    assert et.device_error() == 601
    for t, was in zip((cache.k_codes, cache.k_params, cache.v_codes, cache.v_params), kept):
        assert torch.equal(t, was)
    q = _dev(rng.normal(0, 1, (2, 128)).astype(np.float16), cuda)
    far = et.attention_kv4(cache, q, good, _dev(np.array([1000, 32], np.int32), cuda), 2, 1, 2)
    assert et.device_error() == 601
    near = et.attention_kv4(cache, q, good, _dev(np.array([32, 32], np.int32), cuda), 2, 1, 2)
    assert et.device_error() == 0 and torch.equal(far, near)
    z = et.attention_kv4(cache, q, bad, _dev(np.array([32, 32], np.int32), cuda), 2, 1, 2)
    assert et.device_error() == 601 and bool(torch.isfinite(z).all())


# ---- attention ---------------------------------------------------------------------------------

def _check_attention(et, cuda, batch, seq, heads, nkv, dk, dv, page, lens, mask_kind=1, q_len=None, additive=None,
                     seed=0, scale=None, size=1.0, max_len=None, extra_ld=0, poison=True):
    import torch
    rng = _rng(seed)
    lens = np.array(lens, np.int32)
    most = int(max_len if max_len is not None else max(1, lens.max()))
    per = (most + page - 1) // page
    pages = batch * per + 2
    cache = et.KV4Cache(pages, page, nkv, dk, dv, device=cuda)
    table = _table(rng, batch, per, pages)
    unused = np.ones((pages, nkv, page), bool)
    for b in range(batch):
        pos = np.arange(lens[b])
        unused[table[b][pos // page], :, pos % page] = False
    plain = _fill(et, cache, rng, cuda, size, unused if poison else None)
    T = batch * seq
    qh = rng.normal(0, 1, (T, heads * dk + extra_ld)).astype(np.float16)
    q = _dev(qh, cuda)[:, extra_ld:]
    qn = np.full(batch, seq, np.int32) if q_len is None else np.array(q_len, np.int32)
    out = torch.full((T, heads * dv + extra_ld), 5.0, dtype=torch.float16, device=cuda)
    view = out[:, : heads * dv]
    et.attention_kv4(cache, q, _dev(table, cuda), _dev(lens, cuda), batch, seq, heads, max_len=most,
                     mask_kind=mask_kind, mask=None if additive is None else _dev(additive, cuda),
                     q_len=None if q_len is None else _dev(qn, cuda), scale=scale, out=view)
    assert et.device_error() == 0
    got = out.cpu().numpy().astype(np.float64)
    assert (got[:, heads * dv:] == 5.0).all()
    sc = dk ** -0.5 if scale is None else scale
    ratio = heads // nkv
    q64 = qh[:, extra_ld:].astype(np.float64).reshape(T, heads, dk)
    for b in range(batch):
        for h in range(heads):
            k = _gather(plain[0], table, b, lens[b], h // ratio, dk, page)
            v = _gather(plain[1], table, b, lens[b], h // ratio, dv, page)
            n = int(qn[b])
            rows = np.arange(n)
            limit = lens[b] - n + rows + 1 if mask_kind == 1 else np.full(n, lens[b])
            add = None if additive is None else additive.astype(np.float64)
            qq = q64[b * seq: b * seq + n, h]
            want = ref.attention(qq, k, v, limit, sc, add)
            have = got[b * seq: (b + 1) * seq, h * dv: (h + 1) * dv]
            assert (have[n:] == 5.0).all(), (b, h)
            # a score's error: its fp32 sums (c s and m apart: at most 16 s |q| + |m| |q| per feature), times
            # scale; it enters the weights as a factor e^error on either side of the quotient.  The weights'
            # own roundings (exponential 2^-22, two fp16 parts 2^-22 of the largest) and the sums: 32 + len
            # halvings of 2^-23 of the largest |16 s| + |m| are more than enough
            sk = 16 * plain[0][1].astype(np.float32), plain[0][2].astype(np.float32)
            big_k = float(np.nanmax(sk[0]) + np.nanmax(np.abs(sk[1])))
            sv = 16 * plain[1][1].astype(np.float32), plain[1][2].astype(np.float32)
            big_v = float(np.nanmax(sv[0]) + np.nanmax(np.abs(sv[1])))
            err = sc * (dk + 8) * U32 * big_k * np.abs(qq).sum(-1, keepdims=True)
            if add is not None:
                err = err + U32 * 4 * np.where(np.isfinite(add), np.abs(add), 0).max()
            tol = HALF * np.abs(want) + 2.0 ** -25 + big_v * (2 * err + 64 * U32 + max(lens[b], 1) ** 0.5 * 8 * U32)
            bad = ~(np.abs(have[:n] - want) <= tol)
            assert not bad.any(), (b, h, np.argwhere(bad)[:4], np.abs(have[:n] - want).max(), tol.max())


ATT_CASES = [  # batch, seq, heads, nkv, dk, dv, page, lens
    (1, 1, 1, 1, 16, 16, 16, [1]), (1, 1, 12, 12, 64, 64, 16, [128]), (2, 1, 4, 4, 64, 64, 16, [0, 33]),
    (3, 1, 8, 2, 128, 128, 64, [1, 64, 257]), (2, 3, 12, 4, 48, 64, 16, [100, 3]), (1, 8, 2, 2, 96, 96, 32, [250]),
    (1, 9, 2, 2, 64, 64, 32, [250]), (2, 17, 6, 3, 80, 112, 16, [63, 65]), (1, 5, 8, 1, 128, 64, 32, [97]),
    (2, 64, 4, 4, 64, 64, 128, [64, 300]), (1, 1, 16, 1, 32, 32, 64, [3000]), (1, 2, 3, 1, 16, 128, 16, [1025]),
    (1, 1, 2, 2, 128, 128, 256, [4097]), (5, 1, 6, 6, 112, 16, 16, [31, 32, 33, 48, 1]),
    (1, 33, 5, 1, 32, 96, 32, [200]),
]


@pytest.mark.parametrize("kind", [0, 1], ids=["none", "causal"])
@pytest.mark.parametrize("case", ATT_CASES, ids=str)
def test_attention(et, cuda, case, kind):
    _check_attention(et, cuda, *case, mask_kind=kind, seed=len(str(case)))


@pytest.mark.parametrize("size", [1e-5, 2e-3, 300.0])
def test_attention_over_small_and_large_values(et, cuda, size):
    _check_attention(et, cuda, 2, 2, 4, 2, 64, 64, 16, [70, 200], seed=5, size=size, scale=0.125 / size)


def test_attention_padded_queries_and_strides(et, cuda):
    """Rows behind a sequence's last query stay as they were; sequences with fewer keys than queries leave
    their first rows empty (zeros)."""
    _check_attention(et, cuda, 4, 6, 6, 3, 64, 48, 16, [50, 6, 3, 0], q_len=[6, 2, 5, 0], seed=6, extra_ld=16)
    _check_attention(et, cuda, 2, 40, 2, 1, 32, 64, 16, [20, 41], q_len=[40, 39], seed=7, extra_ld=8)
    _check_attention(et, cuda, 2, 5, 4, 4, 64, 64, 32, [4000, 4001], q_len=[1, 5], seed=8)


def test_attention_max_len_beyond_the_lengths(et, cuda):
    _check_attention(et, cuda, 3, 1, 4, 2, 64, 64, 16, [1, 700, 31], seed=9, max_len=9000)
    _check_attention(et, cuda, 3, 2, 4, 2, 64, 64, 16, [0, 700, 31], mask_kind=0, seed=9, max_len=9000)


@pytest.mark.parametrize("seq,length,ratio", [(1, 40, 1), (3, 77, 2), (20, 300, 2), (2, 5000, 4)])
def test_attention_additive_mask(et, cuda, seq, length, ratio):
    """-inf hides, the type's lowest value keeps its softmax (a row of nothing else is an even one), and a row of
    -inf alone yields zeros."""
    rng = _rng(seq)
    mask = rng.normal(0, 2, (seq, length + 3)).astype(np.float16)
    mask[rng.random(mask.shape) < 0.3] = -np.inf
    mask[rng.random(mask.shape) < 0.1] = -65504.0
    mask[0] = -65504.0 if seq > 2 else mask[0]
    mask[-1] = -np.inf if seq > 1 else mask[-1]
    mask[:, length:] = np.nan
    _check_attention(et, cuda, 2, seq, 2 * ratio, 2, 64, 64, 16, [length, length // 2], mask_kind=3, additive=mask, seed=seq)


def test_attention_masked_nan_does_not_reach_the_output(et, cuda):
    """Tokens that the causal or additive mask hides hold infinities and NaN; a NaN that is seen does reach its
    row (K: the whole row, V: the group's features), and no other row."""
    import torch
    rng = _rng(11)
    cache = et.KV4Cache(8, 16, 2, 64, 64, device=cuda)
    table = _dev(np.arange(8, dtype=np.int32)[None], cuda)
    x = rng.normal(0, 1, (100, 128)).astype(np.float16)
    et.kv4_write(cache, _dev(x, cuda), _dev(x, cuda), table, None, 1, 100)
    q = _dev(rng.normal(0, 1, (4, 128)).astype(np.float16), cuda)
    n = _dev(np.array([100], np.int32), cuda)
    clean = et.attention_kv4(cache, q, table, n, 1, 4, 2)
    bad = x.copy()
    bad[98, 3] = np.nan    # head 0, group 0, position 98: seen by queries 2 and 3
    bad[99, 100] = np.inf  # head 1, group 1, position 99: seen by query 3
    et.kv4_write(cache, _dev(x, cuda), _dev(bad, cuda), table, None, 1, 100)
    z = et.attention_kv4(cache, q, table, n, 1, 4, 2)
    nan = torch.isnan(z)
    want = torch.zeros_like(nan)
    want[2:, 0:32] = True
    want[3, 96:128] = True
    assert torch.equal(nan, want)
    assert torch.equal(z[~want], clean[~want])
    et.kv4_write(cache, _dev(bad, cuda), _dev(x, cuda), table, None, 1, 100)
    z = et.attention_kv4(cache, q, table, n, 1, 4, 2)
    want = torch.zeros_like(nan)
    want[2:, 0:64] = True
    want[3, 64:128] = True
    assert torch.equal(torch.isnan(z), want) and torch.equal(z[~want], clean[~want])
    mask = torch.zeros((4, 128), dtype=torch.float16, device=cuda)
    mask[:, 98:] = float("-inf")
    et.kv4_write(cache, _dev(bad, cuda), _dev(bad, cuda), table, None, 1, 100)
    z = et.attention_kv4(cache, q, table, n, 1, 4, 2, mask_kind=et.MASK_ADDITIVE, mask=mask)
    assert bool(torch.isfinite(z).all())
    # every visible score NaN: the row is NaN, not empty
    one = _dev(np.array([1], np.int32), cuda)
    bad[0, 0] = np.nan
    et.kv4_write(cache, _dev(bad, cuda), _dev(x, cuda), table, None, 1, 100)
    z = et.attention_kv4(cache, q[:1], table, one, 1, 1, 2)
    assert bool(torch.isnan(z[0, :64]).all()) and bool(torch.isfinite(z[0, 64:]).all())


@pytest.mark.parametrize("mask_kind", [1, 3], ids=["causal", "additive"])
@pytest.mark.parametrize("dh", [32, 64, 128])
def test_attention_hidden_giants_cost_nothing(et, cuda, dh, mask_kind):
    """Tokens with huge V that a row does not see, or whose weight is next to nothing, leave the row's precision
    alone.  The output's own rounding is at most 2^-11 of each value, so of the norm, and 0.42 of that on the
    whole; the remaining half covers the sums (2^-22 and less of the largest term each)."""
    import torch
    rng = _rng(dh + mask_kind)
    seq, length, heads = 8, 300, 2
    cache = et.KV4Cache(20, 16, heads, dh, dh, device=cuda)
    table = _dev(np.arange(20, dtype=np.int32)[None], cuda)
    k = rng.normal(0, 1, (length, heads * dh)).astype(np.float16)
    v = rng.normal(0, 1, (length, heads * dh)).astype(np.float16)
    giants = np.zeros(length, bool)
    mask = np.zeros((seq, 304), np.float16)
    if mask_kind == 1:
        giants[-seq + 1:] = True  # the first query sees none of them
        rows = [0]
    else:
        giants[rng.permutation(length)[:40]] = True
        mask[:, :length][:, giants] = -np.inf
        unlikely = np.flatnonzero(giants)[:20]
        mask[:4, unlikely] = -60.0  # seen, with e^-60 of the weight
        rows = list(range(seq))
    v = np.clip(v.astype(np.float32) * np.where(giants, 15000, 1)[:, None], -60000, 60000).astype(np.float16)
    q = rng.normal(0, 1, (seq, heads * dh)).astype(np.float16)
    et.kv4_write(cache, _dev(k, cuda), _dev(v, cuda), table, None, 1, length)
    z = et.attention_kv4(cache, _dev(q, cuda), table, _dev(np.array([length], np.int32), cuda), 1, seq, heads,
                         max_len=length, mask_kind=mask_kind, mask=_dev(mask, cuda) if mask_kind == 3 else None)
    assert et.device_error() == 0
    z = z.cpu().numpy().astype(np.float64)
    plain = [ref.values(*ref.quantise(x.reshape(length, heads, dh), 32)) for x in (k, v)]
    limit = length - seq + 1 + np.arange(seq) if mask_kind == 1 else np.full(seq, length)
    for h in range(heads):
        at = slice(h * dh, (h + 1) * dh)
        want = ref.attention(q[:, at].astype(np.float64), plain[0][:, h], plain[1][:, h], limit, dh ** -0.5,
                             mask[:, :length].astype(np.float64) if mask_kind == 3 else None)
        for r in rows:
            off = np.linalg.norm(z[r, at] - want[r]) / np.linalg.norm(want[r])
            assert off <= 2.0 ** -11, (h, r, off)


@pytest.mark.parametrize("case", [(1, 40, 64, 1, 64, 64, 1024, [500]), (3, 1, 96, 3, 32, 128, 2048, [2049, 1, 4096]),
                                  (1, 200, 2, 2, 128, 128, 16, [201]), (2, 2, 4, 4, 16, 16, 16, [513, 1024]),
                                  (200, 1, 2, 1, 64, 64, 16, list(range(1, 201))),
                                  (1, 100000, 8, 8, 16, 16, 16, [40])], ids=lambda c: str(c)[:40])
def test_attention_many_rows_large_pages_large_batches(et, cuda, case):
    _check_attention(et, cuda, *case, seed=17)


def test_calls_that_share_a_position_or_a_scratch(et, cuda):
    """A position named by several rows keeps the codes of one of them or a mixture (nothing else is touched); a
    given workspace is used, and one on the host, or a page table with gaps between its rows, is refused."""
    import torch
    rng = _rng(18)
    cache = et.KV4Cache(40, 16, 1, 64, 64, device=cuda)
    twice = _dev(np.array([[3, 4], [3, 5]], np.int32), cuda)
    same = rng.normal(0, 1, (32, 64)).astype(np.float16)
    x = _dev(np.concatenate([same, same]), cuda)
    for t in (cache.k_codes, cache.k_params, cache.v_codes, cache.v_params):
        t.zero_()
    et.kv4_write(cache, x, x, twice, None, 2, 32)
    k, _ = et.kv4_read(cache, twice, 2, 32)
    assert torch.equal(k[:32], k[32:])
    assert not cache.k_codes[:3].any() and not cache.k_codes[6:].any()
    table = _dev(np.arange(36, dtype=np.int32)[None], cuda)
    x = _dev(rng.normal(0, 1, (576, 64)).astype(np.float16), cuda)
    et.kv4_write(cache, x, x, table, None, 1, 576)
    q = x[:8]
    n = _dev(np.array([576], np.int32), cuda)
    need = cache.workspace_bytes(1, 8, 1, 576)
    want = et.attention_kv4(cache, q, table, n, 1, 8, 1)
    ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device=cuda)
    assert torch.equal(et.attention_kv4(cache, q, table, n, 1, 8, 1, workspace=ws), want)
    gaps = torch.zeros((2, 40), dtype=torch.int32, device=cuda)[:, 4:20]
    two = _dev(np.array([10, 10], np.int32), cuda)
    xx = x[:16]
    layer = et.EncoderLayer({k: np.asarray(v, np.float16) for k, v in _weights(et, 3, 64, 64).items()}, 1, et.ACT_GELU)
    scratch = torch.empty(layer.cached_workspace_bytes(cache, 2, 1, 32), dtype=torch.uint8, device=cuda)
    out = torch.empty_like(x[:2])
    for f in (lambda: et.attention_kv4(cache, q, table, n, 1, 8, 1, workspace=ws.cpu()),
              lambda: et.attention_kv4(cache, q[:2], gaps, two, 2, 1, 1),
              lambda: et.kv4_write(cache, xx, xx, gaps, None, 2, 8),
              lambda: et.kv4_read(cache, gaps, 2, 8),
              lambda: layer.forward_cached(x[:2], out, cache, gaps, two, two, 2, 1, 32, scratch),
              lambda: layer.forward_cached(x[:2], out, cache, twice, two, two, 2, 1, 32, scratch.cpu()),
              lambda: layer.forward_cached(x[:2], out, cache, twice, two, two, 2, 1, 32, scratch[:256])):
        with pytest.raises(et.EtError):
            f()
    assert et.device_error() == 0


def test_workspace_sizes_do_not_pile_up(et, cuda):
    cache = et.KV4Cache(4, 16, 2, 64, 64, device=cuda)
    for n in range(1, 2000):
        cache.workspace_bytes(1, 1, 2, n)
    assert len(cache._workspace_bytes) <= 256


@pytest.mark.parametrize("length", [60, 3000])
def test_attention_query_that_is_not_finite_stays_in_its_row(et, cuda, length):
    import torch
    rng = _rng(23)
    cache = et.KV4Cache(200, 16, 2, 64, 64, device=cuda)
    table = _dev(np.arange(200, dtype=np.int32)[None], cuda)
    x = _dev(rng.normal(0, 1, (length, 128)).astype(np.float16), cuda)
    et.kv4_write(cache, x, x, table, None, 1, length)
    q = rng.normal(0, 1, (3, 256)).astype(np.float16)
    n = _dev(np.array([length], np.int32), cuda)
    clean = et.attention_kv4(cache, _dev(q, cuda), table, n, 1, 3, 4)
    q[1, 70], q[2, 3] = np.nan, np.inf  # heads 1 and 0
    z = et.attention_kv4(cache, _dev(q, cuda), table, n, 1, 3, 4)
    want = torch.zeros_like(z, dtype=torch.bool)
    want[1, 64:128] = want[2, :64] = True
    assert torch.equal(torch.isnan(z), want) and torch.equal(z[~want], clean[~want])


def test_two_graphs_of_the_same_call(et, cuda):
    """Each captured call has partial results of its own: replayed at once on two streams they do not meet."""
    import torch
    rng = _rng(24)
    cache = et.KV4Cache(300, 16, 2, 64, 64, device=cuda)
    table = _dev(np.arange(300, dtype=np.int32)[None], cuda)
    x = _dev(rng.normal(0, 1, (4800, 128)).astype(np.float16), cuda)
    et.kv4_write(cache, x, x, table, None, 1, 4800)
    n = _dev(np.array([4700], np.int32), cuda)
    assert cache.workspace_bytes(1, 1, 4, 4800) > 0
    qs = [_dev(rng.normal(0, 1, (1, 256)).astype(np.float16), cuda) for _ in range(2)]
    want = [et.attention_kv4(cache, q, table, n, 1, 1, 4).clone() for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(et.attention_kv4(cache, q, table, n, 1, 1, 4))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want)) and et.device_error() == 0


def test_attention_shared_pages_streams_and_replays(et, cuda):
    """A prefix shared by all sequences; two streams at once; a captured call replayed with other lengths, beside
    eager ones."""
    import torch
    rng = _rng(12)
    cache = et.KV4Cache(140, 16, 2, 64, 64, device=cuda)
    tab = np.arange(128, dtype=np.int32)[None].repeat(3, 0)
    tab[:, 100:] = 100 + np.arange(28) + np.array([[0], [4], [8]])
    table = _dev(tab, cuda)
    x = _dev(rng.normal(0, 1, (2048 * 1, 128)).astype(np.float16), cuda)
    et.kv4_write(cache, x, x, table[:1].contiguous(), None, 1, 2048)
    et.kv4_write(cache, x, x, table[2:].contiguous(), None, 1, 2048)
    q = _dev(rng.normal(0, 1, (3, 256)).astype(np.float16), cuda)
    lens = [_dev(np.array(n, np.int32), cuda) for n in ([2048, 5, 1700], [1, 900, 1999], [0, 2048, 16])]
    eager = [et.attention_kv4(cache, q, table, n, 3, 1, 4).clone() for n in lens]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            for _ in range(5):
                o += [et.attention_kv4(cache, q, table, n, 3, 1, 4) for n in lens]
    torch.cuda.synchronize()
    for o in outs:
        for i, z in enumerate(o):
            assert torch.equal(z, eager[i % 3])
    live = lens[0].clone()
    out = torch.empty_like(eager[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        et.attention_kv4(cache, q, table, live, 3, 1, 4, out=out)
    for n, want in zip(lens, eager):
        live.copy_(n)
        g.replay()
        other = et.attention_kv4(cache, q, table, lens[1], 3, 1, 4)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, eager[1])
    assert et.device_error() == 0


def test_cache_past_four_gigabytes(et, cuda):
    """Rows whose byte offsets pass 32 bits."""
    import torch
    pages, page, nkv = 17500, 1024, 16  # 287 M rows of 16 bytes
    cache = et.KV4Cache(pages, page, nkv, 32, 32, device=cuda)
    assert cache.k_codes.numel() > 2 ** 32
    rng = _rng(13)
    tab = np.array([[pages - 1, 0, 16900], [5, pages - 2, 6]], np.int32)
    x = rng.normal(0, 1, (2 * 2500, nkv * 32)).astype(np.float16)
    xd = _dev(x, cuda)
    et.kv4_write(cache, xd, xd, _dev(tab, cuda), None, 2, 2500)
    k, v = et.kv4_read(cache, _dev(tab, cuda), 2, 2500)
    c, s, m = ref.quantise(x.reshape(5000, nkv, 32), 32)
    want = ref.values(c, s, m)
    assert np.array_equal(k.cpu().numpy(), ref.to_f16(want).reshape(5000, -1)) and torch.equal(k, v)
    qh = rng.normal(0, 1, (2, nkv * 32)).astype(np.float16)
    z = et.attention_kv4(cache, _dev(qh, cuda), _dev(tab, cuda), _dev(np.array([2500, 2111], np.int32), cuda), 2, 1,
                         nkv, max_len=2500).cpu().numpy().astype(np.float64)
    assert et.device_error() == 0
    for b, n in enumerate((2500, 2111)):
        for h in range(nkv):
            kv = want[b * 2500: b * 2500 + n, h]
            w = ref.attention(qh[b: b + 1, h * 32: h * 32 + 32].astype(np.float64), kv, kv, [n], 32 ** -0.5)
            # scores off by 40 2^-23 of sum |q| 10, times two sides, times |v| < 10
            tol = HALF * np.abs(w) + 10 * (2 * 40 * U32 * 10 * np.abs(qh[b, h * 32: h * 32 + 32]).sum() * 32 ** -0.5 + 512 * U32)
            assert (np.abs(z[b, h * 32: h * 32 + 32] - w[0]) <= tol[0]).all()


# ---- Linear --------------------------------------------------------------------------------------

@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("out,inn", [(16, 16), (32, 128), (48, 272), (16, 1000 + 24), (64, 144)])
def test_w4_pack_is_exact(et, cuda, out, inn, group):
    rng = _rng(out + inn + group)
    w = _awkward(rng, (out, inn))
    w[3, 7] = np.nan
    w[5, inn - 1] = -np.inf
    q = et.W4Weight(_dev(w, cuda), group)
    c, s, m = ref.quantise(w, group)
    c = np.pad(c, ((0, 0), (0, -(-inn // 128) * 128 - c.shape[1])))
    codes, params = ref.w4_arrays(c, s, m, group)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(q.params.cpu().numpy(), params, equal_nan=True)
    dense = q.densify().cpu().numpy()
    s2 = np.pad(s, ((0, 0), (0, c.shape[1] // group - s.shape[1])))
    m2 = np.pad(m, ((0, 0), (0, c.shape[1] // group - m.shape[1])))
    assert np.array_equal(dense, ref.to_f16(ref.values(c, s2, m2)[:, :inn]), equal_nan=True)


def _gelu(x):
    return x * (0.5 + 0.5 * np.tanh(x * (0.035677408136300125 * x * x + 0.7978845608028654)))


def _check_linear(et, cuda, T, inn, out, group, act=0, bias=True, seed=0, size=1.0, small=None):
    import torch
    rng = _rng(seed + T + inn)
    w = rng.normal(0, 0.03, (out, inn)) + rng.normal(0, 0.01, (out, 1))
    q = et.W4Weight(_dev(w.astype(np.float16), cuda), group)
    c, s, m = ref.quantise(w.astype(np.float16), group)
    w64 = ref.values(c, s, m)[:, :inn]
    x = (rng.normal(0, 1, (T, inn)) * size).astype(np.float16)
    b = rng.normal(0, 0.5, out).astype(np.float16) if bias else None
    if small is not None:
        et.lib().et_debug_set_w4_few(small)
    try:
        y = et.linear_w4(_dev(x, cuda), q, None if b is None else _dev(b, cuda), act).cpu().numpy().astype(np.float64)
    finally:
        if small is not None:
            et.lib().et_debug_set_w4_few(-1)
    assert et.device_error() == 0
    lin = x.astype(np.float64) @ w64.T + (0 if b is None else b.astype(np.float64))
    want = lin if act == 0 else np.maximum(lin, 0) if act == 1 else _gelu(lin)
    few = et.lib().et_debug_w4_few_pay(T, inn, out) if small is None else small == 1
    ax = np.abs(x.astype(np.float64))
    # fp32 sums: of c s x and m x apart, each in blocks of 128
    parts = ref.values(c, s, np.zeros_like(m))[:, :inn] + np.abs(ref.values(np.zeros_like(c), s, m)[:, :inn])
    err = (inn + 16) * U32 * (ax @ parts.T) + U32 * np.abs(lin)
    if not few:
        err = err + HALF * (ax @ np.abs(w64).T)  # weights rounded to fp16
    if act == 2:
        # slope at most 1.13; tanh.approx is off by 2^-10.9 relative in the tensor-core epilogue
        err = 1.13 * err + np.abs(lin) * (2.0 ** -22 if few else 2.0 ** -11)
    tol = HALF * np.abs(want) + 2.0 ** -25 + err
    bad = ~(np.abs(y - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(y - want).max(), tol.min())
    # and on the whole no worse than the roundings' own spread
    # (results below 2^-14 lie on a grid of 2^-24: off by up to 2^-25 each, whatever their size)
    share = (2.0 ** -12 if few else 2.0 ** -11.2) + (2.0 ** -12 if act == 2 and not few else 0)
    off = np.linalg.norm(y - want)
    assert off <= share * np.linalg.norm(want) + 2.0 ** -25 * want.size ** 0.5, off


LIN_CASES = [  # T, in, out, group
    (1, 16, 16, 32), (1, 768, 2304, 32), (1, 768, 768, 128), (2, 144, 48, 64), (3, 1024, 4096, 128),
    (7, 4096, 1024, 64), (8, 272, 80, 32), (9, 528, 32, 128), (16, 4096, 528, 128), (17, 2064, 64, 64),
    (31, 256, 304, 32), (32, 6144, 16, 128), (33, 768, 768, 64), (64, 208, 144, 32), (130, 1040, 272, 128),
    (300, 4096, 768, 64), (1, 12304, 32, 128), (8, 12304, 16, 64), (25, 10256, 16, 32),
]


@pytest.mark.parametrize("case", LIN_CASES, ids=str)
def test_linear_w4(et, cuda, case):
    _check_linear(et, cuda, *case, act=0, bias=case[0] % 2 == 1)


@pytest.mark.parametrize("act", [1, 2])
@pytest.mark.parametrize("case", [(1, 768, 304, 64), (12, 400, 48, 32), (200, 512, 256, 128)], ids=str)
def test_linear_w4_activations(et, cuda, case, act):
    _check_linear(et, cuda, *case, act=act)


@pytest.mark.parametrize("small", [0, 1])
@pytest.mark.parametrize("case", [(1, 256, 64, 32), (20, 1040, 528, 64), (70, 784, 272, 128), (129, 512, 48, 32)],
                         ids=str)
def test_linear_w4_both_kernels(et, cuda, case, small):
    _check_linear(et, cuda, *case, small=small)


def test_linear_w4_small_and_large_activations(et, cuda):
    _check_linear(et, cuda, 3, 528, 64, 32, size=1e-4, bias=False)
    _check_linear(et, cuda, 3, 528, 64, 32, size=2000.0)


def test_linear_w4_nan_stays_in_its_token(et, cuda):
    import torch
    rng = _rng(21)
    for T in (5, 40):
        q = et.W4Weight(_dev(rng.normal(0, 0.05, (64, 256)).astype(np.float16), cuda), 64)
        x = _dev(rng.normal(0, 1, (T, 256)).astype(np.float16), cuda)
        clean = et.linear_w4(x, q)
        x[1, 77], x[3, 200] = float("nan"), float("inf")
        y = et.linear_w4(x, q)
        rows = torch.ones(T, dtype=torch.bool, device=cuda)
        rows[[1, 3]] = False
        assert torch.equal(y[rows], clean[rows]) and not bool(torch.isfinite(y[~rows]).any())


def test_linear_w4_captured_and_on_two_streams(et, cuda):
    import torch
    rng = _rng(22)
    q = et.W4Weight(_dev(rng.normal(0, 0.05, (512, 1024)).astype(np.float16), cuda), 128)
    x = [_dev(rng.normal(0, 1, (4, 1024)).astype(np.float16), cuda) for _ in range(3)]
    want = [et.linear_w4(v, q).clone() for v in x]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            outs += [[et.linear_w4(v, q) for v in x] for _ in range(4)]
    live, out = x[0].clone(), torch.empty_like(want[0])
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        et.linear_w4(live, q, out=out)
    for v, w in zip(x, want):
        live.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)


def test_wrappers_refuse(et, cuda):
    import torch
    cache = et.KV4Cache(4, 16, 2, 64, 64, device=cuda)
    t = torch.zeros((1, 2), dtype=torch.int32, device=cuda)
    n = torch.zeros(1, dtype=torch.int32, device=cuda)
    q = torch.zeros((1, 128), dtype=torch.float16, device=cuda)
    bad = [
        lambda: et.attention_kv4(cache, q.float(), t, n, 1, 1, 2),
        lambda: et.attention_kv4(cache, q.cpu(), t, n, 1, 1, 2),
        lambda: et.attention_kv4(cache, q, t.long(), n, 1, 1, 2),
        lambda: et.attention_kv4(cache, q, t, n.float(), 1, 1, 2),
        lambda: et.attention_kv4(cache, q, t, n, 2, 1, 2),
        lambda: et.attention_kv4(cache, q, t, n, 1, 1, 3),
        lambda: et.attention_kv4(cache, q, t, n, 1, 1, 2, max_len=33),
        lambda: et.attention_kv4(cache, q, t, n, 1, 1, 2, mask_kind=et.MASK_ADDITIVE),
        lambda: et.attention_kv4(cache, q, t, n, 1, 1, 2, mask_kind=et.MASK_ADDITIVE, mask=q[:, :31]),
        lambda: et.attention_kv4(cache, q, t, n, 1, 1, 2, mask_kind=et.MASK_PADDING),
        lambda: et.kv4_write(cache, q, q[:, :64], t, n, 1, 1),
        lambda: et.kv4_write(cache, q.t(), q, t, n, 1, 1),
        lambda: et.kv4_read(cache, t[0], 1, 1),
        lambda: et.kv4_read(cache, t, 1, 1, start=n[:0]),
        lambda: et.KV4Cache(4, 24, 2, 64, 64, device=cuda),
        lambda: et.W4Weight(torch.zeros((16, 128), dtype=torch.float32, device=cuda)),
        lambda: et.W4Weight(torch.zeros((16, 128), dtype=torch.float16, device=cuda), 48),
        lambda: et.W4Weight(torch.zeros((128, 16), dtype=torch.float16, device=cuda).t()),
        lambda: et.linear_w4(q, et.W4Weight(torch.zeros((16, 64), dtype=torch.float16, device=cuda))),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(et.EtError):
            f()
            pytest.fail(f"call {i} was taken")
    assert et.device_error() == 0


# ---- a layer and a stack over the cache ---------------------------------------------------------

def _weights(et, seed, hidden, ff, qk=None):
    qk = hidden if qk is None else qk
    r = lambda n, shape, std: et.synth.normal(seed, n, shape, std)
    return {"wqkv": r(1, (2 * qk + hidden, hidden), 0.04), "bqkv": r(2, (2 * qk + hidden,), 0.1),
            "wo": r(3, (hidden, hidden), 0.04), "bo": r(4, (hidden,), 0.1), "w1": r(5, (ff, hidden), 0.04),
            "b1": r(6, (ff,), 0.1), "w2": r(7, (hidden, ff), 0.04), "b2": r(8, (hidden,), 0.1),
            "ln1_g": 1 + r(9, (hidden,), 0.1), "ln1_b": r(10, (hidden,), 0.1), "ln2_g": 1 + r(11, (hidden,), 0.1),
            "ln2_b": r(12, (hidden,), 0.1)}


@pytest.mark.parametrize("fmt", ["dense", "w4", ("w4", 32)], ids=str)
@pytest.mark.parametrize("batch,seq,qk", [(1, 1, None), (3, 5, 192), (2, 50, None)])
def test_cached_layer_is_its_operators(et, cuda, fmt, batch, seq, qk):
    """et_encoder_layer_cached_fwd against the same operators called one by one (the projection, and with it the
    cache, to the bit; what follows to the path's tolerance: fused forms round elsewhere)."""
    import torch
    from conftest import assert_close
    hidden, ff, nhead, most = 256, 512, 4, 96
    w = {k: np.asarray(v, np.float16) for k, v in _weights(et, 31, hidden, ff, qk).items()}
    qk = hidden if qk is None else qk
    formats = {n: fmt for n in ("wqkv", "wo", "w1", "w2")}
    layer = et.EncoderLayer(w, nhead, et.ACT_GELU, formats=formats)
    dev = {k: _dev(v, cuda) for k, v in w.items()}
    lin = {n: (lambda x, act, q=et.W4Weight(dev[n], 128 if isinstance(fmt, str) else fmt[1]), b=dev[b]:
               et.linear_w4(x, q, b, act)) if fmt != "dense" else
           (lambda x, act, n=n, b=b: et.linear_dense(x, dev[n], dev[b], act))
           for n, b in (("wqkv", "bqkv"), ("wo", "bo"), ("w1", "b1"), ("w2", "b2"))}
    caches = [et.KV4Cache(batch * 6, 16, nhead, qk // nhead, hidden // nhead, device=cuda) for _ in range(2)]
    table = _dev(_rng(1).permutation(batch * 6).reshape(batch, 6).astype(np.int32), cuda)
    kv = torch.zeros(batch, dtype=torch.int32, device=cuda)
    new = None if batch == 1 else _dev(np.array([seq, seq - 1, seq][:batch], np.int32), cuda)
    ws = torch.empty(layer.cached_workspace_bytes(caches[0], batch, seq, most), dtype=torch.uint8, device=cuda)
    live = np.concatenate([np.arange(seq) < (seq if new is None else int(new[b])) for b in range(batch)])
    for step in range(2 if seq > 40 else 3):
        x = _dev(_rng(step).normal(0, 1, (batch * seq, hidden)).astype(np.float16), cuda)
        start = kv.clone()
        kv += seq if new is None else new
        if int(kv.max()) > most:
            break
        out = torch.empty_like(x)
        layer.forward_cached(x, out, caches[0], table, start, kv, batch, seq, most, ws, new)
        qkv = lin["wqkv"](x, 0)
        et.kv4_write(caches[1], qkv[:, qk: 2 * qk], qkv[:, 2 * qk:], table, start, batch, seq, new_len=new)
        for a in ("k_codes", "k_params", "v_codes", "v_params"):
            assert torch.equal(getattr(caches[0], a), getattr(caches[1], a)), (step, a)
        z = et.attention_kv4(caches[1], qkv[:, :qk], table, kv, batch, seq, nhead, max_len=most, q_len=new)
        y = et.skip_layernorm(lin["wo"](z, 0), x, dev["ln1_g"], dev["ln1_b"])
        want = et.skip_layernorm(lin["w2"](lin["w1"](y, et.ACT_GELU), 0), y, dev["ln2_g"], dev["ln2_b"])
        assert et.device_error() == 0
        assert_close(out.cpu().numpy()[live], want.cpu().numpy()[live], f"step {step}")


def test_cached_stack_answers_token_by_token(et, cuda):
    """A prompt, then single tokens (eager and replayed from a graph), against the stack over the whole sequences.
    The cache rounds keys and values to 4 bits, half a step of a fifteenth of a group's range each: random errors of
    1/15 of its 4.1 sigma / sqrt(12) = 0.08 of sigma, which the softmax averages over the tokens and the
    residual path dilutes; a wrong position or page would be off by the order of the output itself."""
    import torch
    hidden, ff, nhead, batch, prompt, steps = 256, 512, 4, 3, 40, 12
    layers = [et.EncoderLayer({k: np.asarray(v, np.float16) for k, v in _weights(et, 41 + i, hidden, ff).items()},
                              nhead, et.ACT_GELU) for i in range(2)]
    total = prompt + steps
    x = _dev(_rng(5).normal(0, 1, (batch, total, hidden)).astype(np.float16), cuda)
    whole = et.EncoderStack(layers, batch, total, device=cuda)
    want = whole.forward(x.reshape(batch * total, hidden), et.MASK_CAUSAL).view(batch, total, hidden).clone()
    stack = et.CachedStack(layers, batch, total, page=16, device=cuda)
    for attempt in range(2):
        stack.reset()
        got = [stack.forward(x[:, :prompt].reshape(-1, hidden), prompt).view(batch, prompt, hidden).clone()]
        step = x[:, prompt].contiguous()
        if attempt == 0:
            for t in range(prompt, total):
                step.copy_(x[:, t])
                got.append(stack.forward(step, 1).view(batch, 1, hidden).clone())
            first = torch.cat(got, 1)
        else:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = stack.forward(step, 1)
            for t in range(prompt, total):
                step.copy_(x[:, t])
                g.replay()
                got.append(out.view(batch, 1, hidden).clone())
            assert torch.equal(torch.cat(got, 1), first)
    assert et.device_error() == 0
    err = (first.float() - want.float()).norm() / want.float().norm()
    assert float(err) < 0.1, float(err)
    with pytest.raises(et.EtError):
        stack.used = total
        stack.forward(step, 1)


def test_cached_stack_refuses_before_its_lengths_move(et, cuda):
    import torch
    hidden, batch = 128, 2
    layers = [et.EncoderLayer({k: np.asarray(v, np.float16) for k, v in _weights(et, 51, hidden, 256).items()}, 2,
                              et.ACT_GELU)]
    stack = et.CachedStack(layers, batch, 33, page=16, device=cuda)
    x = _dev(_rng(19).normal(0, 1, (batch * 6, hidden)).astype(np.float16), cuda)
    want = stack.forward(x, 6).clone()
    stack.reset()
    n = _dev(np.array([6, 6], np.int32), cuda)
    for f in (lambda: stack.forward(x.float(), 6), lambda: stack.forward(x, 5), lambda: stack.forward(x[:, :64], 6),
              lambda: stack.forward(x, 6, new_len=n.long()), lambda: stack.forward(x, 6, new_len=n[:1]),
              lambda: stack.forward(x.cpu(), 6), lambda: stack.forward(x, 6, longest=7), lambda: stack.forward(x, 0),
              lambda: stack.forward(x.t().contiguous().t(), 6)):
        with pytest.raises(et.EtError):
            f()
        assert not bool(stack.kv_len.any()) and stack.used == 0
    assert torch.equal(stack.forward(x, 6), want)
    # lengths past the rows count the rows; the result may be the next call's input
    stack.reset()
    got = stack.forward(x, 6, new_len=n + 100)
    assert torch.equal(got, want) and stack.kv_len.tolist() == [6, 6]
    again = stack.forward(got, 6).clone()
    stack.reset()
    stack.forward(x, 6)
    assert torch.equal(stack.forward(want.clone(), 6), again)
    # padded rows do not use up the host's count where `longest` tells it
    stack.reset()
    short = _dev(np.array([2, 1], np.int32), cuda)
    for _ in range(16):
        stack.forward(x, 6, new_len=short, longest=2)
    assert stack.used == 32 and stack.kv_len.tolist() == [32, 16] and et.device_error() == 0
    with pytest.raises(et.EtError):
        stack.forward(x, 6, new_len=short, longest=2)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("batch,seq", [(1, 5), (2, 100)])
def test_layer_and_stack_of_4_bit_weights(et, cuda, group, batch, seq):
    """The whole-sequence layer with 4-bit weights against the dense layer of the weights that they stand for (which
    differ from them by their rounding to fp16)."""
    from conftest import assert_close
    hidden, ff, nhead = 256, 512, 4
    names = ("wqkv", "wo", "w1", "w2")
    w = {k: np.asarray(v, np.float16) for k, v in _weights(et, 61, hidden, ff).items()}
    plain = dict(w)
    for n in names:
        plain[n] = et.W4Weight(_dev(w[n], cuda), group).densify().cpu().numpy()
    x = _dev(_rng(20).normal(0, 1, (batch * seq, hidden)).astype(np.float16), cuda)
    stacks = [et.EncoderStack([et.EncoderLayer(a, nhead, et.ACT_GELU, formats=f) for _ in range(2)], batch, seq,
                              device=cuda) for a, f in ((w, {n: ("w4", group) for n in names}), (plain, None))]
    got, want = (s.forward(x, et.MASK_CAUSAL).cpu().numpy() for s in stacks)
    assert et.device_error() == 0
    assert_close(got, want, "stack")
