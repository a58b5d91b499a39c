"""CPU checks of the serving operators: the oracle's integers against what they stand for, and the
refusals that need no device."""
import ctypes

import numpy as np
import pytest

from oracle import forward as ofw
from oracle import serving as osv


def test_four_bit_rows_are_within_half_a_step():
    rng = np.random.default_rng(1)
    rows = [rng.integers(-32768, 32768, 64), np.full(64, 77), np.r_[np.full(63, -32768), 32767],
            rng.normal(0, 900, 64).round().astype(np.int64), np.arange(64) // 32]
    for x in rows:
        n, m, z = osv.quantise(np.asarray(x, np.int64))
        assert n.min() >= 0 and n.max() <= 15 and 1 <= m <= 4369 and -32768 <= z <= 32767
        assert (2 * np.abs(z + m * n - x) <= m).all()
        data = np.zeros(16 * 36, np.uint8)
        pool = osv.Pool(data, 1, 64, 16, 4)
        assert np.array_equal(pool.put(0, 0, 5, x), z + m * n) and np.array_equal(pool.get(0, 0, 5), z + m * n)


@pytest.mark.parametrize("prob_bits", [16, 19])
def test_attention_oracle_is_the_forward_pass_at_16_bits(prob_bits):
    import _eii
    rng = np.random.default_rng(2)
    T, page = 37, 16
    q, k, v = (rng.normal(0, 1500, (T, h, 64)).round().clip(-32768, 32767).astype(np.int64) for h in (9, 3, 3))
    E = _eii.table_exp()
    kp, vp = (osv.Pool(np.zeros(3 * 3 * 16 * 128, np.uint8), 3, 64, page, 16) for _ in range(2))
    table = np.array([[2, 0, 1]])
    one = (np.full((T, 32), 1 << 30), np.zeros((T, 32), np.int64))
    qo, kvo = np.empty_like(q), np.empty((T, 2, 3, 64), np.int64)
    osv.append(q, k, v, np.zeros(T, int), np.arange(T), table, kp, vp, one, 30, 30, qo, kvo)
    assert np.array_equal(qo, q) and np.array_equal(kvo[:, 0], k) and np.array_equal(kvo[:, 1], v)
    out = np.empty_like(q)
    osv.attention(q, np.zeros(T, int), np.arange(1, T + 1), table, kp, vp, E, 17, prob_bits, prob_bits, 16, out)
    want = ofw.attention(q, k, v, E, 10, 11, 0, 0, 16, 16, 16, 16)
    if prob_bits == 16:
        assert np.array_equal(out.reshape(T, -1), want)
    else:
        # each of <= 37 probabilities is off by at most half of 2^-16 (2^-19), |v| < 2^13; one rounding each
        assert np.abs(out.reshape(T, -1) - want).max() <= 37 * 8192 * (2.0 ** -17 + 2.0 ** -20) + 1


@pytest.mark.parametrize("inv_temp", [1, 6554, 65536, 131072, 1 << 22])
def test_weights_are_exponentials(inv_temp):
    """w against 2^30 exp(-d / T): the fit is within 3.4e-6, the 24-bit fraction and the Q24 factor
    move the exponent by 2^-24 and 31 / (2 b2) octaves at most, floors of the four products and the last
    rounding add less than 4 + 0.5 units."""
    rng = np.random.default_rng(inv_temp)
    scale = 65536 * 65536 / inv_temp
    d = np.unique(np.r_[0, 1, 2, rng.uniform(0, 23, 400) * scale].round().clip(0, (1 << 32) - 2).astype(np.int64))
    w = osv.weights((1 << 31) - 1 - d, inv_temp)
    b2 = (inv_temp * osv.LOG2E_Q24 + (1 << 15)) >> 16
    want = 2.0 ** 30 * np.exp(-d.astype(np.float64) / scale)
    rel = 3.4e-6 + np.log(2) * (2.0 ** -24 + 31 / (2 * b2))
    assert (np.abs(w - want) <= want * rel * 1.01 + 4.5).all()
    assert (np.diff(w) <= 0).all() and w[0] == 1 << 30


def test_draw_follows_its_distribution():
    row = np.round(np.log([8, 1, 4, 2, 1]) * 65536).astype(np.int64)
    us = (np.arange(4096, dtype=np.uint64) << np.uint64(20)) + np.uint64(1 << 19)
    got = np.bincount([osv.draw(row, u)[0] for u in us], minlength=5)
    assert np.abs(got - np.array([8, 1, 4, 2, 1]) * 256).max() <= 1
    assert {osv.draw(row, u, top_k=2)[0] for u in us[::64]} == {0, 2}
    assert {osv.draw(row, u, top_p=int(.7 * 65536))[0] for u in us[::64]} == {0, 2}
    assert {osv.draw(row, u, min_p=int(.2 * 65536))[0] for u in us[::64]} == {0, 2, 3}
    assert {osv.draw(row, u, top_k=4)[0] for u in us[::16]} == {0, 1, 2, 3}  # the tie at weight 1: lowest index
    assert osv.draw(np.full(4, osv.MASKED), 5) == (-1, 0, 0)


def test_refusals_without_a_device():
    import _eii
    L = _eii.lib()
    h = ctypes.c_void_p()

    def opened(heads=9, kv=3, hd=64, page=16, bits=16, n_pos=512, cos=None, sin=None):
        rc = L.eii_paged_open(0, heads, kv, hd, page, bits, n_pos, cos, sin, ctypes.byref(h))
        return rc, L.eii_last_error().decode()
    t = np.zeros((4, 64), np.int64)
    for kw, text in ((dict(heads=10), "multiple of n_kv"), (dict(heads=0), "multiple"), (dict(kv=0), "multiple"),
                     (dict(hd=96), "head_dim"), (dict(page=8), "page_size"), (dict(page=48), "page_size"),
                     (dict(page=2048), "page_size"), (dict(bits=8), "cache_bits"), (dict(n_pos=0), "n_pos"),
                     (dict(n_pos=131073), "n_pos"), (dict(hd=128), "rope tables"),
                     (dict(cos=t.ctypes.data), "together"),
                     (dict(n_pos=4, cos=(t + (1 << 30) + 1).ctypes.data, sin=t.ctypes.data), "outside")):
        if "outside" in text:
            big = t + (1 << 30) + 1
            kw["cos"] = big.ctypes.data
        rc, msg = opened(**kw)
        assert rc == _eii.EII_ERR_ARG and text in msg and not h.value, (kw, msg)
    assert L.eii_paged_open(0, 9, 3, 64, 16, 16, 8, None, None, None) == _eii.EII_ERR_ARG
    pg = _eii.Pages()
    assert L.eii_paged_append(None, ctypes.byref(pg), None, 0, None, 0, None, 0, 16, 1, None, None, 1, 1, None, 0, None,
                              None) == _eii.EII_ERR_ARG
    assert L.eii_paged_attention(None, ctypes.byref(pg), None, 0, 1, None, None, 1, 1, 16, 1, 16, None, 0, None) == _eii.EII_ERR_ARG
    assert L.eii_paged_pool_bytes(None, 1) == -_eii.EII_ERR_ARG
    assert L.eii_paged_sync(None, None) == _eii.EII_ERR_ARG
    assert b"cache is null" in L.eii_last_error()
    assert L.eii_sampler_open(0, None) == _eii.EII_ERR_ARG
    assert L.eii_sample(None, None, 0, 1, 1, None, None, None, None, None, None, None, None, None) == _eii.EII_ERR_ARG
    assert L.eii_sampler_sync(None, None) == _eii.EII_ERR_ARG
    assert b"sampler is null" in L.eii_last_error()
    L.eii_paged_close(None)
    L.eii_sampler_close(None)
    with pytest.raises(_eii.EiiError):
        _eii.Paged(9, 3, 64, 16, 16, rope=(np.zeros((4, 64), np.int64), np.zeros((4, 64), np.int64)))
