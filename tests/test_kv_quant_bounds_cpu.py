"""CPU tests of the bound that tests/test_kv_quant_range_gpu.py holds attention to: the 64-bit oracle with mistakes
planted in it has to leave the bound, and with the kernels' own roundings it has to stay inside."""
import numpy as np
import pytest

from oracle import kv_quant as oracle
from tests import test_kv_quant_range_gpu as bounds


def _attend(q, k, v, scale, round_weight, unit=None):
    """Attention whose weights (of largest 1) pass through `round_weight`, in units of `unit` per token."""
    m, h_q, d = q.shape
    n, rep = len(k), h_q // k.shape[1]
    out = np.zeros(q.shape)
    for i in range(m):
        see = np.arange(n) <= n - m + i
        for h in range(h_q):
            s = k[see, h // rep] @ q[i, h] * scale
            p = np.exp(s - s.max())
            w = round_weight(p) if unit is None else round_weight(p * unit[see]) / unit[see]
            out[i, h] = w @ v[see, h // rep] / p.sum()
    return out


def _fp16(x):
    return x.astype(np.float16).astype(np.float64)


def _two_parts(p):
    x = p * 2.0 ** 11
    hi = _fp16(x)
    return (hi + _fp16(x - hi)) * 2.0 ** -11


def _stored(x):
    return oracle.dequantise(*oracle.quantise(x))


@pytest.mark.parametrize("d,new,n", [(64, 1, 16), (128, 1, 32), (64, 40, 60), (128, 40, 64)])
def test_bound_tells_one_part_of_an_fp16_weight_from_two(d, new, n):
    k, v = (_stored(x) for x in bounds._cancelling(n, 1, d, seed=d))
    q = _fp16(np.random.default_rng(1).standard_normal((new, 2, d)) * 0.25)
    ref, _, tol, _ = bounds._bounds(q, k, v, np.ones(n, bool), d ** -0.5, True, 2.0 ** -22)
    tol = tol + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25  # the result's own rounding
    assert (np.abs(_fp16(_attend(q, k, v, d ** -0.5, _two_parts)) - ref) <= tol).all()
    one = _attend(q, k, v, d ** -0.5, lambda p: _fp16(p * 2.0 ** 11) * 2.0 ** -11)
    assert (np.abs(_fp16(one) - ref) > tol).any()


@pytest.mark.parametrize("v_log", [25, 45])
def test_bound_tells_weights_relative_to_a_hidden_value(v_log):
    """Weights in units of the largest value scale of all tokens, hidden ones too, leave the bound."""
    n, new, d = 100, 4, 64
    k, v = (_stored(x) for x in bounds._huge_rows(n, 1, d, [n - 1], None, v_log, seed=3))
    q = np.random.default_rng(2).standard_normal((new, 2, d))
    ref, _, tol, _ = bounds._bounds(q, k, v, np.ones(n, bool), d ** -0.5, True, 2.0 ** -22)
    tol = tol + 2.0 ** -11 * np.abs(ref)
    byte = oracle.quantise(v)[1][:, 0].astype(float)
    unit = 2.0 ** (byte - byte.max() + 12)
    assert (np.abs(_attend(q, k, v, d ** -0.5, _fp16, unit) - ref) > tol)[:-1].any()
    own = 2.0 ** np.where(byte < byte.max() - 8, 12.0, byte - byte.max() + 12)
    assert (np.abs(_attend(q, k, v, d ** -0.5, lambda p: _two_parts(p * 2.0 ** -11) * 2.0 ** 11, own) - ref) <= tol).all()
