"""GPU tests of the 8-bit paged KV cache against the 64-bit oracle (oracle/kv_quant.py).

Writing and reading back are exact: the scales are powers of two, so the codes are the
same in any precision.  Attention is compared on the values that the pages hold.

Bounds of an output element, with A = sum p |v| / sum p:
  * its rounding to bf16 / fp16: half a step, eps / 2 of the value;
  * a weight p rounded to fp16 (half a step: eps / 2 = 2^-11 of it) moves the output by at
    most 2^-11 A; a chunk kernel may round weights to bf16 (eps / 2 = 2^-8 of them: 2^-8 A);
  * a score x (log2 units) summed in fp32 over d products is off by at most
    dx = (d + 8) 2^-24 X, X = log2(e) scale sum |q_i k_i|, and exp2 by 2^-22 of its value:
    numerator and denominator each move by ln2 dx + 2^-22, the output by twice that of A;
  * sums of n weights in fp32 lose at most a further 2^-24 per addition on a chain; the
    longest chain of one lane is n / 16 pages long, merged pairwise: n 2^-28 A at most twice;
  * fp16 ends at 2^-25 (half a step of its subnormals).  A weight is held in units of 2^-11
    of a reference at or below the row's largest weight, so it is off by 2^-36 of that at
    most; where the value's scale is in the weight too (units of 2^-12 of the largest scale,
    codes up to 448, that scale at most vmax / 224) by 2^-37 448 / 224 vmax = 2^-36 vmax; a
    value held as 2^-6 of the largest scale and up by 2^-25 2^-6 / 224 vmax < 2^-38 vmax: n
    tokens move the output by (n + 1) 2^-36 vmax, vmax the request's largest |v|;
  * likewise keys relative to the largest scale of a tile are off by 2^-25 kmax / 224, and q
    after scaling its row to [2^14, 2^15) by 2^-25 2^-14 of the row's largest: d products
    move x by d 2^-32 log2(e) scale qmax kmax at most.
The log-sum-exp moves by ln2 dx + 2^-22, and is rounded to fp32 a few times.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv_quant as oracle

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _np(kv):
    return [t.view(torch.uint8).cpu().numpy() for t in kv]


def _fill(device, n_pages, h_kv, d, seed, spread=0.5, v_spread=None):
    """A cache full of random rows (by the oracle, so that attention does not lean on the writer)."""
    from unifiedkv_b200.kv_quant import QuantPagedKV
    rng = np.random.default_rng(seed)
    out = []
    for s in (spread, spread if v_spread is None else v_spread):
        x = rng.standard_normal((n_pages, 16, h_kv, d)) * 2.0 ** (rng.standard_normal((n_pages, 16, h_kv, 1)) * s)
        codes, byte = oracle.quantise(x)
        out.append((torch.from_numpy(codes).to(device).view(torch.float8_e4m3fn),
                    torch.from_numpy(np.ascontiguousarray(byte.transpose(0, 2, 1))).to(device)))
    return QuantPagedKV(out[0][0], out[1][0], out[0][1], out[1][1])


def _table(device, lens, n_pages, seed, width=None):
    rng = np.random.default_rng(seed)
    need = [-(-n // 16) for n in lens]
    ids = rng.permutation(n_pages)[:sum(need)]
    bt = np.zeros((len(lens), width or max(max(need), 1)), np.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[at:at + n]
        at += n
    return torch.from_numpy(bt).to(device)


def _i32(device, x):
    return torch.tensor(list(x), dtype=torch.int32, device=device)


def _cu(device, lens):
    return _i32(device, np.concatenate([[0], np.cumsum(lens)]))


def _check(got, lse, q, kv, bt, lens, new, scale, causal=True, empty=0.0, weight=2.0 ** -11):
    """got [total, hq, d] and lse against the oracle."""
    kc, vc, ks, vs = _np(kv)
    bt, qn = bt.cpu().numpy(), q.double().cpu().numpy()
    g = got.double().cpu().numpy()
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0  # half a step of its subnormals
    d, at = q.shape[2], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        k, there = oracle.request_rows(kc, ks, bt[b], n)
        v, _ = oracle.request_rows(vc, vs, bt[b], n)
        ref, ref_lse, mean_abs, size = oracle.attention(qn[at:at + m], k, v, there, m, scale, causal)
        o, l = g[at:at + m], None if lse is None else lse[at:at + m].double().cpu().numpy()
        at += m
        none = np.isneginf(ref_lse)
        if math.isnan(empty):
            assert np.isnan(o[none]).all()
        else:
            assert (o[none] == empty).all()
        qmax = np.abs(np.where(np.isfinite(qn[at - m:at]), qn[at - m:at], 0)).max(-1)
        kmax, vmax = (np.nanmax(np.abs(x), initial=0.0) for x in (k, v))
        dx = (d + 8) * 2.0 ** -24 * size + d * 2.0 ** -32 * scale * qmax * kmax
        move = dx + 2.0 ** -21 + n * 2.0 ** -27
        floor = (n + 1) * 2.0 ** -36 * vmax
        tol = half * np.abs(ref) + ((weight + 2 * move)[..., None] * mean_abs + floor) * (1 + half) + tiny
        with np.errstate(invalid="ignore"):
            near = np.abs(o - ref) <= tol
        # what lies half a step or more above the type's largest number rounds to an infinity
        top = torch.finfo(got.dtype).max * (1 + half / 2)
        near |= (np.abs(ref) + tol >= top) & np.isinf(o) & (np.sign(o) == np.sign(ref))
        bad = ~none[..., None] & ~near
        assert not bad.any(), (b, n, m, np.argwhere(bad)[:5], o[bad][:5], ref[bad][:5], tol[bad][:5])
        if l is not None:
            assert np.isneginf(l[none]).all()
            ok = ~none
            assert (np.abs(l[ok] - ref_lse[ok]) <= move[ok] + 2.0 ** -22 * (1 + np.abs(ref_lse[ok]))).all(), b


# ---- write and read back -------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("h_kv,d", [(8, 128), (2, 64), (3, 256), (1, 128)])
def test_append_is_bit_exact(cuda, dtype, h_kv, d):
    from unifiedkv_b200.kv_quant import quantize_append
    new, past = [1, 0, 37, 16, 5], [0, 9, 3, 16, 1000]
    lens = [p + n for p, n in zip(past, new)]
    n_pages = 90
    kv = _fill(cuda, n_pages, h_kv, d, seed=d)
    before = _np(kv)
    bt = _table(cuda, lens, n_pages, seed=1, width=70)
    total = sum(new)
    g = torch.Generator(device=cuda).manual_seed(5)
    # K and V inside one fused projection's rows, with rows behind the last sequence
    qkv = torch.randn(total + 3, 2 * h_kv * d + 64, generator=g, device=cuda).to(DT[dtype])
    k_new, v_new = (qkv[:, i * h_kv * d:(i + 1) * h_kv * d].unflatten(1, (h_kv, d)) for i in (0, 1))
    quantize_append(kv, k_new, v_new, bt, _i32(cuda, lens), cu_seqlens_q=_cu(cuda, new))
    after, table = _np(kv), bt.cpu().numpy()
    for src, ci, si in ((k_new, 0, 2), (v_new, 1, 3)):
        codes, byte = oracle.quantise(src.double().cpu().numpy())
        want_c, want_s = before[ci].copy(), before[si].copy()
        i = 0
        for b, n in enumerate(new):
            for j in range(n):
                pos = past[b] + j
                want_c[table[b, pos // 16], pos % 16] = codes[i]
                want_s[table[b, pos // 16], :, pos % 16] = byte[i]
                i += 1
        np.testing.assert_array_equal(after[si], want_s)
        np.testing.assert_array_equal(after[ci], want_c)  # every other slot as it was


def test_append_of_rows_at_the_borders(cuda):
    """Zeros, one huge or tiny element, powers of two and 448 times them, infinities, NaN, the largest and the
    smallest floats."""
    from unifiedkv_b200.kv_quant import dequantize_pages, quantize_append
    d = 64
    x = torch.zeros(16, 1, d)
    x[1] = 1.0
    x[2] = torch.linspace(-448, 448, d)
    x[3] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    x[4, 0, 3] = 3.4e38
    x[5] = 3.4028234e38
    x[6, 0, ::2] = 1e-45
    x[7] = 2.0 ** -126
    x[8, 0, 5] = float("inf")
    x[9, 0, 63] = float("nan")
    x[10, 0, 0] = -float("inf")
    x[11] = torch.arange(d) * 2.0 ** -9
    x[12] = -0.0
    x[13] = torch.exp2(torch.arange(d).float() - 40)
    x[14] = (torch.arange(d) + 0.5) / 64  # ties
    x[15] = 448 * 2.0 ** 119
    kv = _fill(cuda, 2, 1, d, seed=2)
    bt = _i32(cuda, [1])[None]
    y = torch.flip(x, [0])
    quantize_append(kv, x.to(cuda), y.to(cuda), bt, _i32(cuda, [16]), cu_seqlens_q=_i32(cuda, [0, 16]))
    kc, vc, ks, vs = _np(kv)
    for rows, c, s in ((x, kc, ks), (y, vc, vs)):
        codes, byte = oracle.quantise(rows.double().numpy())
        np.testing.assert_array_equal(s[1, 0], byte[:, 0])
        np.testing.assert_array_equal(c[1], codes)
    k, _ = dequantize_pages(kv, bt, _i32(cuda, [0, 16]), 16, dtype=torch.float32)
    np.testing.assert_array_equal(k.double().cpu().numpy(), oracle.dequantise(kc[1], ks[1].T))
    assert torch.isnan(k[8:11]).all() and torch.isfinite(k[:8]).all() and torch.isfinite(k[11:]).all()


def test_append_skips_what_has_no_slot(cuda):
    """Pages that are not there (-1, past the pool), positions past the table or before its start."""
    from unifiedkv_b200.kv_quant import quantize_append
    kv = _fill(cuda, 4, 2, 64, seed=3)
    before = _np(kv)
    bt = torch.tensor([[-1, 1], [4, 1 << 30], [2, 2], [3, 0], [0, 1]], dtype=torch.int32, device=cuda)
    lens = _i32(cuda, [3, 17, 33, 0, -5])  # -1, past the pool, past the table, before the start (twice)
    x = torch.randn(5, 2, 64, device=cuda).bfloat16()
    quantize_append(kv, x, x, bt, lens)
    for a, b in zip(before, _np(kv)):
        np.testing.assert_array_equal(a, b)
    quantize_append(kv, x, x, bt, _i32(cuda, [17, 17, 16, 32, 1]))  # page 1 slot 0, none, page 2 slot 15, page 0 slot 15, page 0 slot 0
    codes, byte = oracle.quantise(x.double().cpu().numpy())
    kc, _, ks, _ = _np(kv)
    for i, page, slot in ((0, 1, 0), (2, 2, 15), (3, 0, 15), (4, 0, 0)):
        np.testing.assert_array_equal(kc[page, slot], codes[i])
        np.testing.assert_array_equal(ks[page, :, slot], byte[i])
    np.testing.assert_array_equal(kc[3], before[0][3])


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("h_kv,d", [(8, 128), (2, 64), (1, 256), (5, 64)])
def test_readback_is_exact(cuda, dtype, h_kv, d):
    from unifiedkv_b200.kv_quant import dequantize_pages
    kv = _fill(cuda, 60, h_kv, d, seed=d + 1, spread=6.0)
    lens, starts = [1, 0, 300, 33, 16], [5, 0, 7, 16, 0]
    bt = _table(cuda, [n + s for n, s in zip(lens, starts)], 60, seed=4)
    bt[3, 1] = -1  # tokens 16..31 of request 3 are not in the pool
    total = sum(lens)
    out = [torch.full((h_kv, total + 2, d), 7.0, dtype=DT[dtype], device=cuda) for _ in (0, 1)]
    got = dequantize_pages(kv, bt, _cu(cuda, lens), total + 2, starts=_i32(cuda, starts),
                           out=tuple(o.transpose(0, 1) for o in out))
    packed = dequantize_pages(kv, bt, _cu(cuda, lens), total, dtype=DT[dtype], starts=_i32(cuda, starts))
    np_kv, table = _np(kv), bt.cpu().numpy()
    for which in (0, 1):
        want = []
        for b, (n, s) in enumerate(zip(lens, starts)):
            v, there = oracle.request_rows(np_kv[which], np_kv[2 + which], table[b], n + s)
            v[~there] = 0
            want.append(v[s:])
        want = torch.from_numpy(np.concatenate(want)).to(DT[dtype])
        assert torch.equal(packed[which].cpu(), want)
        assert torch.equal(got[which][:total].cpu(), want)
        assert (out[which][:, total:] == 7).all()  # rows behind the last sequence


def test_readback_past_the_table_and_before_its_start(cuda):
    from unifiedkv_b200.kv_quant import dequantize_pages
    kv = _fill(cuda, 3, 1, 64, seed=6)
    bt = _i32(cuda, [2])[None]
    k, v = dequantize_pages(kv, bt, _i32(cuda, [0, 20]), 20, starts=_i32(cuda, [-2]))
    np_kv = _np(kv)
    want = oracle.dequantise(np_kv[0][2], np_kv[2][2].T)
    assert (k[:2] == 0).all() and (k[18:] == 0).all() and (v[18:] == 0).all()
    np.testing.assert_array_equal(k[2:18].double().cpu().numpy(), want)


# ---- decode ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,h_kv,d", [(32, 8, 128), (8, 8, 256), (16, 2, 64), (8, 1, 128), (6, 3, 64), (25, 5, 128),
                                       (32, 2, 128), (40, 1, 64), (12, 12, 64), (20, 1, 256), (27, 9, 128)])
def test_decode(cuda, dtype, hq, h_kv, d):
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    lens = [1, 15, 16, 17, 333, 2049, 0, 40]
    kv = _fill(cuda, 200, h_kv, d, seed=hq + d)
    bt = _table(cuda, lens, 200, seed=7, width=150)
    g = torch.Generator(device=cuda).manual_seed(hq)
    q = torch.randn(len(lens), hq, d, generator=g, device=cuda).to(DT[dtype])
    lse = torch.full((len(lens), hq), 9.0, device=cuda)
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=d ** -0.5, n_rep=hq // h_kv, lse_out=lse)
    again = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=d ** -0.5, n_rep=hq // h_kv)
    assert out.dtype == q.dtype and out.is_contiguous()
    torch.testing.assert_close(out, again, rtol=0, atol=0, equal_nan=True)  # fixed order of every sum
    _check(out, lse, q, kv, bt, lens, [1] * len(lens), d ** -0.5, empty=float("nan"))


@pytest.mark.parametrize("lens", [[5], [16 * 148 * 2 + 3], [40000], [9000, 1, 1, 700] + [100] * 60])
def test_decode_splits(cuda, lens):
    """One long request over all workers, requests shared by neighbours, more workers than pages."""
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    hq, h_kv, d = 8, 2, 128
    n_pages = sum(-(-n // 16) for n in lens) + 1
    kv = _fill(cuda, n_pages, h_kv, d, seed=len(lens))
    bt = _table(cuda, lens, n_pages, seed=8)
    q = torch.randn(len(lens), hq, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).bfloat16()
    lse = torch.empty(len(lens), hq, device=cuda)
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=0.2, n_rep=4, lse_out=lse)
    _check(out, lse, q, kv, bt, lens, [1] * len(lens), 0.2, empty=float("nan"))


def test_decode_of_more_requests_than_the_flat_list_holds(cuda):
    """Above 4096 items no item is split between workers."""
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    rng = np.random.default_rng(2)
    lens = [int(x) for x in rng.integers(0, 60, 4200)]
    kv = _fill(cuda, 300, 1, 64, seed=9)
    bt = torch.from_numpy(rng.integers(0, 300, (4200, 4)).astype(np.int32)).to(cuda)  # pages may be shared by readers
    q = torch.randn(4200, 2, 64, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1)).half()
    lse = torch.empty(4200, 2, device=cuda)
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=0.125, n_rep=2, lse_out=lse)
    _check(out, lse, q, kv, bt, lens, [1] * 4200, 0.125, empty=float("nan"))


def test_decode_of_strided_views(cuda):
    """q inside a fused projection; one layer of a pool; a table with padding columns and an int64 length."""
    from unifiedkv_b200.kv_quant import QuantPagedKV, page16_decode_attention_q8
    hq, h_kv, d, lens = 8, 2, 128, [100, 31]
    kv = _fill(cuda, 20, h_kv, d, seed=10)
    big = [torch.zeros((3,) + t.shape, dtype=torch.uint8, device=cuda) for t in kv]
    for b, t in zip(big, kv):
        b[1] = t.view(torch.uint8)
    layer = QuantPagedKV(big[0][1].view(torch.float8_e4m3fn), big[1][1].view(torch.float8_e4m3fn), big[2][1], big[3][1])
    # pages further apart than they are long
    wide = [torch.zeros((20, 2) + t.shape[1:], dtype=torch.uint8, device=cuda) for t in kv]
    for w, t in zip(wide, kv):
        w[:, 0] = t.view(torch.uint8)
    apart = QuantPagedKV(wide[0][:, 0].view(torch.float8_e4m3fn), wide[1][:, 0].view(torch.float8_e4m3fn), wide[2][:, 0], wide[3][:, 0])
    bt = torch.zeros(2, 40, dtype=torch.int32, device=cuda)
    bt[:, :7] = _table(cuda, lens, 20, seed=11)
    qkv = torch.randn(2, 12 * d, device=cuda).bfloat16()
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    want = page16_decode_attention_q8(q.contiguous(), kv, bt, _i32(cuda, lens), softmax_scale=0.1, n_rep=4)
    for c in (layer, apart):
        got = page16_decode_attention_q8(q, c, bt[:, :9], torch.tensor(lens, device=cuda), softmax_scale=0.1, n_rep=4)
        assert torch.equal(got, want)
    odd = torch.randn(2, hq * d + 1, device=cuda).bfloat16()[:, 1:].unflatten(1, (hq, d))  # not 16-byte aligned: copied
    got = page16_decode_attention_q8(odd, kv, bt, _i32(cuda, lens), softmax_scale=0.1, n_rep=4)
    assert torch.equal(got, page16_decode_attention_q8(odd.contiguous(), kv, bt, _i32(cuda, lens), softmax_scale=0.1, n_rep=4))
    _check(got, None, odd, kv, bt, lens, [1, 1], 0.1)


@pytest.mark.parametrize("spread", [0.0, 4.0])
def test_decode_with_scales_far_apart(cuda, spread):
    """Rows of very unequal norm: key scales move the maximum, value scales the weights' unit."""
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    lens = [700, 64]
    kv = _fill(cuda, 60, 2, 128, seed=12, spread=1.0, v_spread=spread)
    bt = _table(cuda, lens, 60, seed=13)
    q = torch.randn(2, 8, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).bfloat16()
    q[0, 1] *= 2.0 ** -60
    q[0, 2] = 0
    q[1, 3] *= 16
    lse = torch.empty(2, 8, device=cuda)
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=128 ** -0.5, n_rep=4, lse_out=lse)
    _check(out, lse, q, kv, bt, lens, [1, 1], 128 ** -0.5)


def test_pages_that_are_not_there_and_tables_too_short(cuda):
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    lens = [100, 50, 500, 20]
    kv = _fill(cuda, 40, 2, 64, seed=14)
    bt = _table(cuda, [100, 50, 112, 20], 40, seed=15, width=7)
    bt[0, 2] = -1
    bt[0, 6] = 40
    bt[3] = -7
    q = torch.randn(4, 4, 64, device=cuda).half()
    lse = torch.empty(4, 4, device=cuda)
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=0.125, n_rep=2, lse_out=lse)
    _check(out, lse, q, kv, bt, [100, 50, 112, 20], [1] * 4, 0.125, empty=float("nan"))


def test_offsets_past_32_bits(cuda):
    """Pages whose first byte lies beyond 2^32 in the pool."""
    from unifiedkv_b200.kv_quant import QuantPagedKV, dequantize_pages, page16_decode_attention_q8, quantize_append
    h_kv, d = 8, 256
    n_pages = (1 << 32) // (16 * h_kv * d) + 40
    codes = [torch.empty(n_pages, 16, h_kv, d, dtype=torch.uint8, device=cuda) for _ in (0, 1)]
    scales = [torch.empty(n_pages, h_kv, 16, dtype=torch.uint8, device=cuda) for _ in (0, 1)]
    kv = QuantPagedKV(codes[0].view(torch.float8_e4m3fn), codes[1].view(torch.float8_e4m3fn), *scales)
    bt = (n_pages - 1 - torch.arange(20, device=cuda, dtype=torch.int32))[None]
    g = torch.Generator(device=cuda).manual_seed(3)
    k, v = (torch.randn(300, h_kv, d, generator=g, device=cuda).bfloat16() for _ in (0, 1))
    quantize_append(kv, k, v, bt, _i32(cuda, [300]), cu_seqlens_q=_i32(cuda, [0, 300]))
    got, _ = dequantize_pages(kv, bt, _i32(cuda, [0, 300]), 300)
    c, e = oracle.quantise(k.double().cpu().numpy())
    np.testing.assert_array_equal(got.double().cpu().numpy(), oracle.dequantise(c, e))
    q = torch.randn(1, 16, d, generator=g, device=cuda).bfloat16()
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, [300]), softmax_scale=d ** -0.5, n_rep=2)
    tail = QuantPagedKV(*(t[-20:] for t in kv))
    _check(out, None, q, tail, bt - (n_pages - 20), [300], [1], d ** -0.5)


# ---- chunks ----------------------------------------------------------------------
CHUNKS = [
    # new tokens and lengths of the requests: drafts, ragged chunks, no past, an empty request, an empty chunk
    ([4, 4, 1], [100, 4, 17]),
    ([37, 1, 0, 100, 16], [40, 500, 12, 100, 1000]),
    ([200], [200]),
    ([130, 3], [131, 2049]),
    ([2, 0, 5], [0, 0, 3]),  # fewer tokens than queries: the first queries see none
]


@pytest.mark.parametrize("new,lens", CHUNKS)
@pytest.mark.parametrize("hq,h_kv,d,dtype", [(8, 2, 128, "bf16"), (4, 2, 64, "fp16"), (5, 1, 128, "bf16"), (2, 2, 256, "bf16"),
                                             (12, 1, 64, "bf16"), (3, 3, 128, "fp16")])
def test_chunk(cuda, new, lens, hq, h_kv, d, dtype):
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    kv = _fill(cuda, 250, h_kv, d, seed=sum(new) + d)
    bt = _table(cuda, lens, 250, seed=16, width=140)
    g = torch.Generator(device=cuda).manual_seed(hq)
    total = sum(new)
    q = torch.randn(total, hq, d, generator=g, device=cuda).to(DT[dtype])
    lse = torch.full((total, hq), 9.0, device=cuda)
    out = paged_chunk_prefill_q8(q, kv, bt, softmax_scale=d ** -0.5, n_rep=hq // h_kv, cu_seqlens_q=_cu(cuda, new),
                                 seqlens_k=_i32(cuda, lens), max_seqlen_q=max(new), lse_out=lse)
    _check(out, lse, q, kv, bt, lens, new, d ** -0.5, weight=2.0 ** -8)
    if all(n >= m for n, m in zip(lens, new)):
        listed = paged_chunk_prefill_q8(q, kv, bt, [n - m for n, m in zip(lens, new)], new, n_rep=hq // h_kv)
        assert torch.equal(listed, out)


@pytest.mark.parametrize("d", [64, 128])
def test_chunk_without_a_causal_mask(cuda, d):
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    new, lens = [50, 1, 9], [60, 33, 5]
    kv = _fill(cuda, 20, 2, d, seed=17)
    bt = _table(cuda, lens, 20, seed=18)
    q = torch.randn(60, 4, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(4)).bfloat16()
    out = paged_chunk_prefill_q8(q, kv, bt, [max(0, n - m) for n, m in zip(lens, new)], new, n_rep=2, causal=False,
                                 cu_seqlens_q=_cu(cuda, new), seqlens_k=_i32(cuda, lens), max_seqlen_q=50)
    _check(out, None, q, kv, bt, lens, new, d ** -0.5, causal=False, weight=2.0 ** -8)


@pytest.mark.parametrize("d,new", [(64, 9), (128, 9), (128, 200), (256, 40)])
def test_rows_that_are_not_finite_stay_out_of_queries_that_do_not_see_them(cuda, d, new):
    """A NaN key or value poisons the queries that see it and no other; what lies behind the last token
    (or on pages of nobody) is never looked at."""
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    n = new + 21
    kv = _fill(cuda, 30, 1, d, seed=19)
    bt = _table(cuda, [n], 30, seed=20)
    table = bt.cpu().numpy()[0]
    mine = set(int(x) for x in table)
    for page in range(30):  # the other pages, and the slots behind the last token, hold NaN
        slots = range(16) if page not in mine else range((n - 1) % 16 + 1, 16) if page == table[-1] else ()
        for s in slots:
            for t, b in ((kv.k_codes, kv.k_scales), (kv.v_codes, kv.v_scales)):
                t.view(torch.uint8)[page, s] = 0x7F
                b[page, :, s] = 255
    q = torch.randn(new, 2, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(5)).bfloat16()
    call = dict(softmax_scale=d ** -0.5, n_rep=2, cu_seqlens_q=_i32(cuda, [0, new]), seqlens_k=_i32(cuda, [n]), max_seqlen_q=new)
    clean = paged_chunk_prefill_q8(q, kv, bt, **call)
    _check(clean, None, q, kv, bt, [n], [new], d ** -0.5, weight=2.0 ** -8)
    for codes, scales in ((kv.k_codes, kv.k_scales), (kv.v_codes, kv.v_scales)):
        pos = n - 4  # seen by the last four queries
        page, slot = int(table[pos // 16]), pos % 16
        keep = codes.view(torch.uint8)[page, slot].clone(), scales[page, :, slot].clone()
        codes.view(torch.uint8)[page, slot] = 0x7F
        scales[page, :, slot] = 255
        got = paged_chunk_prefill_q8(q, kv, bt, **call)
        assert torch.isnan(got[-4:]).all()
        torch.testing.assert_close(got[:-4].float(), clean[:-4].float(), rtol=2.0 ** -7, atol=2.0 ** -8)
        codes.view(torch.uint8)[page, slot], scales[page, :, slot] = keep


def test_rows_behind_the_last_sequence_are_left_alone(cuda):
    """A padded batch: q has more rows than the sequences; those rows of lse keep what they held."""
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    for d, new in ((64, [3, 2]), (128, [150, 60])):
        lens = [n + 10 for n in new]
        kv = _fill(cuda, 40, 1, d, seed=21)
        bt = _table(cuda, lens, 40, seed=22)
        total = sum(new)
        q = torch.randn(total + 50, 2, d, device=cuda).bfloat16()
        lse = torch.full((total + 50, 2), 5.0, device=cuda)
        out = paged_chunk_prefill_q8(q, kv, bt, softmax_scale=0.1, n_rep=2, cu_seqlens_q=_cu(cuda, new),
                                     seqlens_k=_i32(cuda, lens), lse_out=lse)
        assert out.shape == q.shape and (lse[total:] == 5).all()
        _check(out[:total], lse[:total], q[:total], kv, bt, lens, new, 0.1, weight=2.0 ** -8)


# ---- together --------------------------------------------------------------------
def test_serving_run_over_a_pool(cuda):
    """Prompts in chunks, then decode steps, over one layer of a pool: write, attend, read back, each step
    checked against the oracle on what the pool should hold."""
    from unifiedkv_b200.kv_quant import QuantPagedKVPool, page16_decode_attention_q8, paged_chunk_prefill_q8, quantize_append
    hq, h_kv, d = 8, 2, 128
    pool = QuantPagedKVPool(16, 2, h_kv, d, device=cuda, n_total=60)
    kv = pool.layer(1)
    pages = [pool.allocate_blocks(20), pool.allocate_blocks(9)]
    _, _, bt = pool.build_block_table(1, pages)
    g = torch.Generator(device=cuda).manual_seed(6)
    rows = [[[], []], [[], []]]  # per request, K and V values the pool holds
    lens = [0, 0]
    for new in ([40, 16], [130, 3], [1, 1], [1, 1], [4, 4], [100, 0]):
        lens = [a + b for a, b in zip(lens, new)]
        total = sum(new)
        q, k, v = (torch.randn(total, h, d, generator=g, device=cuda).bfloat16() for h in (hq, h_kv, h_kv))
        cu, sk = _cu(cuda, new), _i32(cuda, lens)
        quantize_append(kv, k, v, bt, sk, cu_seqlens_q=cu)
        if new == [1, 1]:
            out = page16_decode_attention_q8(q, kv, bt, sk, softmax_scale=d ** -0.5, n_rep=4)
        else:
            out = paged_chunk_prefill_q8(q, kv, bt, n_rep=4, cu_seqlens_q=cu, seqlens_k=sk, max_seqlen_q=max(new))
        _check(out, None, q, kv, bt, lens, new, d ** -0.5, weight=2.0 ** -8)
        at = 0
        for b, n in enumerate(new):
            for x, keep in ((k, rows[b][0]), (v, rows[b][1])):
                keep.append(oracle.dequantise(*oracle.quantise(x[at:at + n].double().cpu().numpy())))
            at += n
    for b in (0, 1):
        K, V = pool.read_kv_from_blocks(1, pages[b], lens[b])
        assert K.shape == (h_kv, lens[b], d) and K.is_contiguous()
        np.testing.assert_array_equal(K.double().cpu().numpy().transpose(1, 0, 2), np.concatenate(rows[b][0]))
        np.testing.assert_array_equal(V.double().cpu().numpy().transpose(1, 0, 2), np.concatenate(rows[b][1]))
    assert torch.count_nonzero(pool.k_cache[0].view(torch.uint8)) == 0  # the other layer is untouched
    pool.write_kv_to_blocks(0, pages[1], torch.ones(h_kv, 20, d, device=cuda), torch.ones(h_kv, 20, d, device=cuda) * 2)
    pool.write_one_token(0, pages[1][1], 4, torch.full((h_kv, 1, d), 3.0, device=cuda), torch.full((h_kv, 1, d), 5.0, device=cuda))
    K, V = pool.read_kv_from_blocks(0, pages[1], 22)
    assert (K[:, :20] == 1).all() and (V[:, :20] == 2).all() and (K[:, 20] == 3).all() and (V[:, 20] == 5).all()
    assert (K[:, 21] == 0).all()


def test_side_stream_and_graphs(cuda):
    """A captured step (write, attend, read back) replayed after its inputs changed gives the eager bits; two
    graphs replayed at once on two streams do not share scratch."""
    from unifiedkv_b200.kv_quant import dequantize_pages, page16_decode_attention_q8, paged_chunk_prefill_q8, quantize_append
    hq, h_kv, d = 8, 2, 128
    lens, new = [400, 900, 33], [3, 7, 1]
    steps = []
    for i in (0, 1):
        kv = _fill(cuda, 100, h_kv, d, seed=30 + i)
        bt, sk, cu = _table(cuda, lens, 100, seed=31), _i32(cuda, lens), _cu(cuda, new)
        g = torch.Generator(device=cuda).manual_seed(7 + i)
        q, k, v = (torch.randn(11, h, d, generator=g, device=cuda).bfloat16() for h in (hq, h_kv, h_kv))

        def step(kv=kv, bt=bt, sk=sk, cu=cu, q=q, k=k, v=v):
            quantize_append(kv, k, v, bt, sk, cu_seqlens_q=cu)
            a = page16_decode_attention_q8(q[:3], kv, bt, sk, softmax_scale=0.1, n_rep=4)
            b = paged_chunk_prefill_q8(q, kv, bt, n_rep=4, cu_seqlens_q=cu, seqlens_k=sk, max_seqlen_q=7)
            return (a, b) + dequantize_pages(kv, bt, cu, 11, starts=sk - torch.diff(cu))

        steps.append((step, sk, q, k))
    eager = [[t.clone() for t in s[0]()] for s in steps]
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        on_side = [t.clone() for t in steps[0][0]()]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager[0], on_side))
    graphs = []
    for step, *_ in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(cuda) for _ in graphs]
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), want in zip(graphs, eager):
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    for (step, sk, q, k), (graph, out) in zip(steps, graphs):
        sk.copy_(_i32(cuda, [390, 16, 12]))
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_first_call_of_a_process_inside_a_capture():
    """Nothing has to have run before: kernels are loaded and set up while the stream is being captured."""
    import subprocess
    import sys
    from pathlib import Path
    code = r'''
import torch
from unifiedkv_b200.kv_quant import QuantPagedKVPool, dequantize_pages, page16_decode_attention_q8, paged_chunk_prefill_q8, quantize_append
dev = torch.device("cuda:0")
pool = QuantPagedKVPool(16, 1, 2, 128, device=dev, n_total=30)
kv = pool.layer(0)
bt = torch.arange(30, dtype=torch.int32, device=dev).view(1, 30)
n, cu = torch.tensor([200], dtype=torch.int32, device=dev), torch.tensor([0, 200], dtype=torch.int32, device=dev)
q, k = torch.randn(200, 4, 128, device=dev).bfloat16(), torch.randn(200, 2, 128, device=dev).bfloat16()
torch.cuda.synchronize()

def step():
    quantize_append(kv, k, k, bt, n, cu_seqlens_q=cu)
    a = paged_chunk_prefill_q8(q, kv, bt, n_rep=2, cu_seqlens_q=cu, seqlens_k=n, max_seqlen_q=200)
    b = paged_chunk_prefill_q8(q[:5], kv, bt, n_rep=2, cu_seqlens_q=cu.clamp(max=5), seqlens_k=n, max_seqlen_q=5)
    return a, b, page16_decode_attention_q8(q[:1], kv, bt, n, softmax_scale=0.1, n_rep=2), *dequantize_pages(kv, bt, cu, 200)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in out]
assert all(torch.equal(x, y) for x, y in zip(got, step()))
print("ok")
'''
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-3000:]


def test_sequence_bounds_past_the_rows_of_q(cuda):
    """cu_seqlens that claim more rows than q has: the rows that are there are computed, none other is touched."""
    for d, new in ((64, 5), (128, 60)):
        kv = _fill(cuda, 12, 1, d, seed=60)
        bt = _table(cuda, [100], 12, seed=61)
        q = torch.randn(new, 2, d, device=cuda).bfloat16()
        from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
        whole = torch.cat([q, torch.zeros(20, 2, d, device=cuda, dtype=q.dtype)])
        call = dict(softmax_scale=0.1, n_rep=2, cu_seqlens_q=_i32(cuda, [0, new + 20]), seqlens_k=_i32(cuda, [100]))
        want = paged_chunk_prefill_q8(whole, kv, bt, max_seqlen_q=new + 20, **call)
        got = paged_chunk_prefill_q8(q, kv, bt, max_seqlen_q=new + 20, **call)
        torch.testing.assert_close(got.float(), want[:new].float(), rtol=2.0 ** -7, atol=2.0 ** -8)


def test_tensors_of_another_device_are_refused(cuda):
    from unifiedkv_b200.kv_quant import dequantize_pages, page16_decode_attention_q8, quantize_append
    kv = _fill(cuda, 3, 2, 64, seed=62)
    bt, n = torch.zeros(1, 2, dtype=torch.int32, device=cuda), _i32(cuda, [3])
    x = torch.randn(1, 2, 64, device=cuda).bfloat16()
    for call in (lambda: quantize_append(kv, x, x.cpu(), bt, n), lambda: quantize_append(kv, x, x, bt.cpu(), n),
                 lambda: quantize_append(kv._replace(k_scales=kv.k_scales.cpu()), x, x, bt, n),
                 lambda: dequantize_pages(kv, bt, torch.tensor([0, 2]), 2),
                 lambda: page16_decode_attention_q8(x, kv, bt, n.cpu(), softmax_scale=0.1, n_rep=1)):
        with pytest.raises(RuntimeError, match="shape_unsupported:device_cpu"):
            call()


@pytest.mark.parametrize("h_kv,n_rep,d", [(16, 2, 64), (33, 1, 128), (1, 32, 128)])
def test_many_heads(cuda, h_kv, n_rep, d):
    """More KV heads than a CTA's warps, one KV head for all: decode and chunks."""
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    lens, new = [70, 300], [1, 1]
    kv = _fill(cuda, 30, h_kv, d, seed=63)
    bt = _table(cuda, lens, 30, seed=64)
    q = torch.randn(2, h_kv * n_rep, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(10)).bfloat16()
    out = page16_decode_attention_q8(q, kv, bt, _i32(cuda, lens), softmax_scale=d ** -0.5, n_rep=n_rep)
    _check(out, None, q, kv, bt, lens, new, d ** -0.5)
    q = torch.randn(43, h_kv * n_rep, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(11)).bfloat16()
    out, lse = _chunk(cuda, q, kv, bt, lens, [3, 40], n_rep, d ** -0.5)
    _check(out, lse, q, kv, bt, lens, [3, 40], d ** -0.5)


def test_no_synchronisation_and_no_empty_launch(cuda):
    """Empty batches are answered without a launch; nothing waits for the device."""
    from unifiedkv_b200.kv_quant import dequantize_pages, paged_chunk_prefill_q8, quantize_append
    kv = _fill(cuda, 4, 2, 64, seed=40)
    bt = torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    zero = torch.zeros(1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda)
    torch.cuda.set_sync_debug_mode("error")
    try:
        quantize_append(kv, none, none, bt, lens)
        quantize_append(kv, none, none, bt, lens, cu_seqlens_q=zero)
        k, v = dequantize_pages(kv, bt, zero, 0)
        out = paged_chunk_prefill_q8(none, kv, bt, n_rep=1, cu_seqlens_q=zero, seqlens_k=lens, max_seqlen_q=0)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert k.shape == (0, 2, 64) and v.shape == (0, 2, 64) and out.shape == (0, 2, 64)


# ---- the tensor-core chunk kernel --------------------------------------------------
def _chunk(cuda, q, kv, bt, lens, new, n_rep, scale, causal=True):
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    lse = torch.full(q.shape[:2], 9.0, device=cuda)
    out = paged_chunk_prefill_q8(q, kv, bt, softmax_scale=scale, n_rep=n_rep, causal=causal, cu_seqlens_q=_cu(cuda, new),
                                 seqlens_k=_i32(cuda, lens), max_seqlen_q=max(new), lse_out=lse)
    return out, lse


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,lens", [
    ([40], [5000]),                 # 120 rows: alternating groups, the tokens split over CTAs
    ([100, 90], [130, 3000]),       # two row tiles, one of them partly empty
    ([43, 1, 20], [43, 4000, 129]),
    ([171], [4096]),                # 513 rows: a tile of one row
])
def test_long_caches(cuda, dtype, d, new, lens):
    n_pages = sum(-(-n // 16) for n in lens) + 2
    kv = _fill(cuda, n_pages, 1, d, seed=d + sum(new), spread=1.0)
    bt = _table(cuda, lens, n_pages, seed=50)
    g = torch.Generator(device=cuda).manual_seed(8)
    q = torch.randn(sum(new), 3, d, generator=g, device=cuda).to(DT[dtype])
    out, lse = _chunk(cuda, q, kv, bt, lens, new, 3, d ** -0.5)
    again, _ = _chunk(cuda, q, kv, bt, lens, new, 3, d ** -0.5)
    assert torch.equal(out, again)
    _check(out, lse, q, kv, bt, lens, new, d ** -0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("k_spread,v_spread", [(0.0, 0.0), (1.0, 4.0)])
def test_chunk_with_scales_far_apart(cuda, dtype, k_spread, v_spread):
    """Scales that move the values' reference from tile to tile, and rows of q of very unequal norm."""
    lens, new = [900, 300], [70, 30]
    kv = _fill(cuda, 90, 1, 128, seed=51, spread=k_spread, v_spread=v_spread)
    bt = _table(cuda, lens, 90, seed=52)
    table = bt.cpu().numpy()
    kv.v_scales[int(table[0, 40])] += 30  # one page's values 2^30 above the rest: the reference jumps late
    q = torch.randn(100, 2, 128, device=cuda, generator=torch.Generator(device=cuda).manual_seed(9)).to(DT[dtype])
    q[::7] = 0
    q[1::7] *= 8
    q[2::7] *= 2.0 ** -12
    out, lse = _chunk(cuda, q, kv, bt, lens, new, 2, 0.05)
    _check(out, lse, q, kv, bt, lens, new, 0.05)


def test_chunk_over_pages_that_are_not_there(cuda):
    lens, new = [600, 150, 64], [64, 50, 50]
    kv = _fill(cuda, 60, 2, 128, seed=53)
    bt = _table(cuda, lens, 60, seed=54)
    bt[0, 0] = -1
    bt[0, 9:30] = 60
    bt[0, 36] = -5
    bt[2] = -1  # nothing of request 2 is there
    q = torch.randn(sum(new), 4, 128, device=cuda).bfloat16()
    out, lse = _chunk(cuda, q, kv, bt, lens, new, 2, 0.1)
    _check(out, lse, q, kv, bt, lens, new, 0.1)


@pytest.mark.parametrize("hq,h_kv,d,new", [(4, 2, 128, 60), (4, 2, 64, 3), (4, 1, 256, 20)])
def test_negative_and_zero_softmax_scales(cuda, hq, h_kv, d, new):
    lens = [new + 100]
    kv = _fill(cuda, 20, h_kv, d, seed=55)
    bt = _table(cuda, lens, 20, seed=56)
    q = torch.randn(new, hq, d, device=cuda).bfloat16()
    for scale in (-0.1, 0.0):
        out, lse = _chunk(cuda, q, kv, bt, lens, [new], hq // h_kv, scale)
        dx = max(abs(scale), 1e-30)
        assert torch.isfinite(lse).all()
        kc, vc, ks, vs = _np(kv)
        k, there = oracle.request_rows(kc, ks, bt.cpu().numpy()[0], lens[0])
        v, _ = oracle.request_rows(vc, vs, bt.cpu().numpy()[0], lens[0])
        ref, ref_lse, mean_abs, size = oracle.attention(q.double().cpu().numpy(), k, v, there, new, scale)
        move = (d + 8) * 2.0 ** -24 * np.abs(size) + 2.0 ** -21 + lens[0] * 2.0 ** -27
        tol = 2.0 ** -8 * np.abs(ref) + (2.0 ** -11 + 2 * move)[..., None] * mean_abs * (1 + 2.0 ** -8)
        assert (np.abs(out.double().cpu().numpy() - ref) <= tol).all(), (scale, dx)


def test_chunks_of_values_that_are_not_finite(cuda):
    """NaN keys and values in several tiles, rows of q that are not finite: only who sees them is NaN."""
    lens, new = [700], [150]
    kv = _fill(cuda, 50, 1, 128, seed=57)
    bt = _table(cuda, lens, 50, seed=58)
    table = bt.cpu().numpy()[0]
    q = torch.randn(150, 2, 128, device=cuda).bfloat16()
    clean, _ = _chunk(cuda, q, kv, bt, lens, new, 2, 0.1)
    for pos, (codes, scales) in ((600, (kv.v_codes, kv.v_scales)), (640, (kv.k_codes, kv.k_scales))):
        codes.view(torch.uint8)[int(table[pos // 16]), pos % 16] = 0x7F
        scales[int(table[pos // 16]), :, pos % 16] = 255
    q[3, 1, 5] = float("inf")
    q[4, 0, 7] = float("nan")
    out, lse = _chunk(cuda, q, kv, bt, lens, new, 2, 0.1)
    first = 600 - 550  # query i sees tokens up to 550 + i
    assert torch.isnan(out[first:]).all() and torch.isnan(out[3, 1]).all() and torch.isnan(out[4, 0]).all()
    keep = torch.ones(150, 2, dtype=torch.bool, device=cuda)
    keep[first:] = False
    keep[3, 1] = keep[4, 0] = False
    assert torch.equal(out[keep], clean[keep])


# ---- row tiles cut into shares: one request by the host, a batch by the device ------
def _heads(kv, heads):
    from unifiedkv_b200.kv_quant import QuantPagedKV
    return QuantPagedKV(kv.k_codes[:, :, heads], kv.v_codes[:, :, heads], kv.k_scales[:, heads], kv.v_scales[:, heads])


def _shared_pages(device, lens, n_pages, seed):
    """A block table that comes back to the same few pages: long requests over a small cache."""
    rng = np.random.default_rng(seed)
    return torch.from_numpy(rng.integers(0, n_pages, (len(lens), -(-max(lens) // 16)), dtype=np.int32)).to(device)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_one_request_with_row_tiles_whole_and_cut(cuda, dtype):
    """150 row tiles and KV heads, a little over the SMs: one row tile of each head whole, the other cut."""
    h_kv, new, n, d = 75, 300, 5000, 64
    kv = _fill(cuda, 20, h_kv, d, seed=60)
    bt = _shared_pages(cuda, [n], 20, seed=61)
    q = torch.randn(new, h_kv, d, device=cuda, generator=torch.Generator(device=cuda).manual_seed(10)).to(DT[dtype])
    out, lse = _chunk(cuda, q, kv, bt, [n], [new], 1, 0.125)
    heads = [0, 37, 74]
    _check(out[:, heads], lse[:, heads], q[:, heads], _heads(kv, heads), bt, [n], [new], 0.125)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h_kv,n_rep,new,lens", [
    (2, 4, [12, 8, 12, 1, 10, 0, 9], [5000, 300, 4100, 1, 4, 700, 0]),  # up to 48 rows; requests and rows that see nothing
    (2, 3, [150, 90, 64], [5000, 200, 4200]),                           # two row tiles a request, the second not always there
    (40, 1, [60, 60, 33, 60], [4200, 4200, 700, 4200]),                 # more CTAs than SMs
])
def test_batches_cut_by_their_lengths(cuda, dtype, d, h_kv, n_rep, new, lens):
    kv = _fill(cuda, 20, h_kv, d, seed=62)
    bt = _shared_pages(cuda, lens, 20, seed=63)
    g = torch.Generator(device=cuda).manual_seed(11)
    q = torch.randn(sum(new), h_kv * n_rep, d, generator=g, device=cuda).to(DT[dtype])
    out, lse = _chunk(cuda, q, kv, bt, lens, new, n_rep, d ** -0.5)
    again, _ = _chunk(cuda, q, kv, bt, lens, new, n_rep, d ** -0.5)
    assert torch.equal(out, again)
    heads = sorted({0, h_kv // 2, h_kv - 1})
    rows = [h * n_rep + r for h in heads for r in range(n_rep)]
    _check(out[:, rows], lse[:, rows], q[:, rows], _heads(kv, heads), bt, lens, new, d ** -0.5)


@pytest.mark.parametrize("n_rep,new", [(4, [12, 9, 12]), (8, [40, 3, 64])])
def test_a_captured_batch_is_cut_by_the_lengths_of_its_replay(cuda, n_rep, new):
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    width = [6000, 6000, 6000]
    kv = _fill(cuda, 20, 2, 128, seed=64)
    bt = _shared_pages(cuda, width, 20, seed=65)
    q = torch.randn(sum(new), 2 * n_rep, 128, device=cuda).bfloat16()
    sk, cu = _i32(cuda, width), _cu(cuda, new)

    def step():
        lse = torch.full(q.shape[:2], 9.0, device=cuda)
        return paged_chunk_prefill_q8(q, kv, bt, softmax_scale=0.1, n_rep=n_rep, cu_seqlens_q=cu, seqlens_k=sk,
                                      max_seqlen_q=max(new), lse_out=lse), lse
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lens in ([6000, 40, 700], [12, 0, 5999], [64, 64, 64], [2500, 2500, 6000]):
        sk.copy_(_i32(cuda, lens))
        graph.replay()
        torch.cuda.synchronize()
        out, lse = (t.clone() for t in captured)
        want = step()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        _check(out, lse, q, kv, bt, lens, new, 0.1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("h_kv,n_rep,new,lens", [
    (8, 4, [60, 45, 70], [600, 1500, 70]),  # several items a worker, its pairs of warps at different ones
    (1, 8, [130, 131], [400, 131]),
    (8, 1, [1] * 300, list(range(1, 301))),  # 8-row items
    (4, 2, [90] * 60, [90] * 60),            # more items than are split: pairs run on by themselves
])
def test_pairs_of_warps_at_different_items(cuda, dtype, h_kv, n_rep, new, lens):
    """head_dim 256: two warps share a head, and pairs do not wait for one another."""
    kv = _fill(cuda, 20, h_kv, 256, seed=66)
    bt = _shared_pages(cuda, lens, 20, seed=67)
    g = torch.Generator(device=cuda).manual_seed(12)
    q = torch.randn(sum(new), h_kv * n_rep, 256, generator=g, device=cuda) * torch.exp2(
        3 * torch.randn(sum(new), h_kv * n_rep, 1, generator=g, device=cuda))
    q = q.to(DT[dtype])
    out, lse = _chunk(cuda, q, kv, bt, lens, new, n_rep, 0.02)
    for _ in range(10):
        again = _chunk(cuda, q, kv, bt, lens, new, n_rep, 0.02)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    _check(out, lse, q, kv, bt, lens, new, 0.02)


@pytest.mark.parametrize("new,lens", [
    ([9 + i % 4 for i in range(600)], [12 + i % 50 for i in range(600)]),        # 36 to 48 rows
    ([30 + i % 121 for i in range(200)], [150 + i % 31 for i in range(200)]),    # one to three row tiles
])
def test_more_row_tiles_than_are_put_in_order(cuda, new, lens):
    kv = _fill(cuda, 20, 1, 64, seed=68)
    bt = _shared_pages(cuda, lens, 20, seed=69)
    q = torch.randn(sum(new), 4, 64, device=cuda, generator=torch.Generator(device=cuda).manual_seed(13)).bfloat16()
    out, lse = _chunk(cuda, q, kv, bt, lens, new, 4, 0.125)
    _check(out, lse, q, kv, bt, lens, new, 0.125)


def test_two_batches_at_once_on_two_streams(cuda):
    """Batches cut on the device, each with its own plan and parts, side by side."""
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    runs = []
    for i, lens in enumerate(([5000, 300, 4500], [100, 5100, 64])):
        new = [40, 33, 50]
        kv = _fill(cuda, 20, 2, 128, seed=70 + i)
        bt, sk, cu = _shared_pages(cuda, lens, 20, seed=72), _i32(cuda, lens), _cu(cuda, new)
        q = torch.randn(sum(new), 4, 128, device=cuda).bfloat16()

        def step(q=q, kv=kv, bt=bt, sk=sk, cu=cu):
            return paged_chunk_prefill_q8(q, kv, bt, softmax_scale=0.1, n_rep=2, cu_seqlens_q=cu, seqlens_k=sk, max_seqlen_q=50)
        runs.append((step, step()))
    streams = [torch.cuda.Stream(cuda) for _ in runs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(runs[i][0]())
    torch.cuda.synchronize()
    for (_, want), got in zip(runs, outs):
        assert all(torch.equal(want, g) for g in got)
