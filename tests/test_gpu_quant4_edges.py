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
