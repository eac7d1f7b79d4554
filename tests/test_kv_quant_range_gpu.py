"""GPU tests of attention over 8-bit pages at the edges of the number range, against the 64-bit oracle.

Here a row's bound is made of the tokens that the row sees and of nothing else: what a causal mask hides, or
what a row gives no weight to, may not move it however large it is.  With weights p (largest 1), l = sum p, and
for each token t that the row sees

  * dx_t = (d + 8) 2^-24 X_t + d 2^-38 log2(e) |scale| max|q| max|k_t|, X_t = log2(e) |scale| sum |q_i k_t,i|:
    a score summed in fp32 over d products of q (rounded to fp16 after its row was scaled to [2^14, 2^15): off by
    2^-25 of 2^14) and exact keys;
  * mv_t = ln2 dx_t + 2^-21 + n 2^-27: with two exponentials of 2^-22 and sums of n weights, 16 a step, in fp32
    (a step of the tensor cores' sums may be cut off rather than rounded: 2^-23);
  * 2^-11 of a weight for bf16 results (half a step of fp16), 2^-22 for fp16 ones (two parts);
  * weights end at half a step of fp16's subnormals, 2^-25, in units of 2^-11 of the row's reference (chunk kernel:
    2^-36 of the largest weight) or of 2^-12 2^(vunit - vbyte_t) of it, vunit < vbyte_t + 8 (2^-30): both of |v_t|;

an element of the result is off by at most
  sum_t (p_t (exp(mv_t) - 1 + weight) + 2^-30) |v_t| / l + |out| sum_t p_t (exp(mv_t) - 1) / l
and its rounding to bf16 / fp16, half a step.  The log-sum-exp moves by sum_t p_t (exp(mv_t) - 1) / l and is rounded
to fp32 a few times.
"""
import numpy as np
import pytest
import torch

from oracle import kv_quant as oracle

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _i32(device, x):
    return torch.tensor(list(x), dtype=torch.int32, device=device)


def _cache(device, k, v, seed):
    """Requests' rows (lists of [n, h_kv, d]) in pages of no order -> cache, table."""
    from unifiedkv_b200.kv_quant import QuantPagedKV
    need = [-(-len(x) // 16) for x in k]
    rng = np.random.default_rng(seed)
    ids = rng.permutation(sum(need) + 2)
    h_kv, d = k[0].shape[1:]
    out, table = [], np.zeros((len(k), max(max(need), 1)), np.int32)
    for rows in (k, v):
        codes = np.zeros((len(ids), 16, h_kv, d), np.uint8)
        scales = np.zeros((len(ids), h_kv, 16), np.uint8)
        at = 0
        for b, x in enumerate(rows):
            c, e = oracle.quantise(x)
            for j in range(need[b]):
                m = min(16, len(x) - 16 * j)
                table[b, j] = ids[at]
                codes[ids[at], :m] = c[16 * j:16 * j + m]
                scales[ids[at], :, :m] = e[16 * j:16 * j + m].T
                at += 1
        out.append((torch.from_numpy(codes).to(device).view(torch.float8_e4m3fn), torch.from_numpy(scales).to(device)))
    return QuantPagedKV(out[0][0], out[1][0], out[0][1], out[1][1]), torch.from_numpy(table).to(device)


def _bounds(q, k, v, there, scale, causal, weight):
    """q [m, h_q, d], k and v [n, h_kv, d] in 64 bits -> out, lse, and how far each may be off."""
    m, h_q, d = q.shape
    n, h_kv = k.shape[:2]
    rep = h_q // h_kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, ltol = np.full((m, h_q), -np.inf), np.zeros((m, h_q))
    for i in range(m):
        see = there & (np.arange(n) <= (n - m + i if causal else n - 1))
        if not see.any():
            continue
        for h in range(h_q):
            kk, vv, qq = k[see, h // rep], v[see, h // rep], q[i, h]
            s = kk @ qq * scale
            top = s.max()
            p = np.exp(s - top)
            l = p.sum()
            size = np.log2(np.e) * abs(scale) * (np.abs(kk) @ np.abs(qq))
            most = d * np.log2(np.e) * abs(scale) * np.abs(qq).max() * np.abs(kk).max(-1)
            mv = np.log(2) * ((d + 8) * 2.0 ** -24 * size + 2.0 ** -38 * most) + 2.0 ** -21 + n * 2.0 ** -27
            off = np.exp(np.minimum(s - top + mv, 700)) - p
            out[i, h] = p @ vv / l
            tol[i, h] = (off + weight * p + 2.0 ** -30) @ np.abs(vv) / l + np.abs(out[i, h]) * off.sum() / l
            lse[i, h] = top + np.log(l)
            ltol[i, h] = off.sum() / l + 2.0 ** -22 * (1 + abs(lse[i, h]))
    return out, lse, tol, ltol


def _check(got, lse, q, kv, bt, lens, new, scale, causal=True, empty=0.0):
    kc, vc, ks, vs = (t.view(torch.uint8).cpu().numpy() for t in kv)
    table, qn, g = bt.cpu().numpy(), q.double().cpu().numpy(), got.double().cpu().numpy()
    info, at = torch.finfo(got.dtype), 0
    weight = 2.0 ** -22 if got.dtype == torch.float16 else 2.0 ** -11
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134  # half a step of the subnormals
    for b, (n, m) in enumerate(zip(lens, new)):
        k, there = oracle.request_rows(kc, ks, table[b], n)
        v, _ = oracle.request_rows(vc, vs, table[b], n)
        ref, ref_lse, tol, ltol = _bounds(qn[at:at + m], k, v, there, scale, causal, weight)
        o, l = g[at:at + m], lse[at:at + m].double().cpu().numpy()
        at += m
        tol = tol * (1 + info.eps) + info.eps / 2 * np.abs(ref) + tiny
        none = np.isneginf(ref_lse)
        assert np.isnan(o[none]).all() if np.isnan(empty) else (o[none] == empty).all()
        with np.errstate(invalid="ignore"):
            near = np.abs(o - ref) <= tol
        # half a step or more above the type's largest number rounds to an infinity
        near |= (np.abs(ref) + tol >= info.max * (1 + info.eps / 4)) & np.isinf(o) & (np.sign(o) == np.sign(ref))
        bad = ~none[..., None] & ~near
        assert not bad.any(), (b, n, m, int(bad.sum()), np.argwhere(bad)[:4], o[bad][:4], ref[bad][:4], tol[bad][:4])
        assert np.isneginf(l[none]).all()
        wrong = ~none & ~(np.abs(l - np.where(none, 0, ref_lse)) <= ltol)
        assert not wrong.any(), (b, np.argwhere(wrong)[:4], l[wrong][:4], ref_lse[wrong][:4], ltol[wrong][:4])


def _chunk(device, q, kv, bt, lens, new, scale, causal=True):
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    lse = torch.full(q.shape[:2], 9.0, device=device)
    out = paged_chunk_prefill_q8(q, kv, bt, softmax_scale=scale, n_rep=q.shape[1] // kv.k_codes.shape[2], causal=causal,
                                 cu_seqlens_q=_i32(device, np.concatenate([[0], np.cumsum(new)])),
                                 seqlens_k=_i32(device, lens), max_seqlen_q=max(new), lse_out=lse)
    return out, lse


def _decode(device, q, kv, bt, lens, scale):
    from unifiedkv_b200.kv_quant import page16_decode_attention_q8
    lse = torch.full(q.shape[:2], 9.0, device=device)
    return page16_decode_attention_q8(q, kv, bt, _i32(device, lens), softmax_scale=scale,
                                      n_rep=q.shape[1] // kv.k_codes.shape[2], lse_out=lse), lse


def _q(device, total, hq, d, dtype, seed, size=1.0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(total, hq, d, generator=g, device=device) * size).to(DT[dtype])


# ---- small queries over tiles without keys, or with keys of zeros ------------------
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [40, 150])  # 80 rows (alternating groups), 300 (two row tiles)
def test_small_queries_over_absent_tiles_and_zero_keys(cuda, d, new):
    rng = np.random.default_rng(d + new)
    n = 700
    k, v = (rng.standard_normal((n, 1, d)) for _ in (0, 1))
    k[400:] = 0  # zeros up to and under the causal border
    kv, bt = _cache(cuda, [k], [v], 1)
    gone = bt.clone()
    gone[0, 8:17] = -1  # a whole 128-token tile, and a page of the next
    for size in (1.0, 2.0 ** -8, 2.0 ** -20, 2.0 ** -40):
        q = _q(cuda, new, 2, d, "bf16", 3, size)
        for table in (bt, gone):
            _check(*_chunk(cuda, q, kv, table, [n], [new], d ** -0.5), q, kv, table, [n], [new], d ** -0.5)
    q = _q(cuda, new, 2, d, "bf16", 4)
    for scale in (1e-20, 1e-37):
        _check(*_chunk(cuda, q, kv, gone, [n], [new], scale), q, kv, gone, [n], [new], scale)


# ---- one huge row: hidden from a query, or of no weight to it ----------------------
def _huge_rows(n, h_kv, d, where, k_log, v_log, seed):
    """Unit rows, but for rows `where`: keys -2^k_log along the first dimension, values of 2^v_log."""
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((n, h_kv, d)) for _ in (0, 1))
    for t in where:
        if k_log is not None:
            k[t] = 0
            k[t, :, 0] = -2.0 ** k_log
        v[t] *= 2.0 ** v_log
    return k, v


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,d", [(2, 64), (4, 128), (2, 256)])
@pytest.mark.parametrize("v_log", [9, 25, 45, 68, -20, -68])
def test_few_rows_beside_a_huge_value(cuda, dtype, hq, d, v_log):
    """Drafted tokens: the last token's value is huge (or every other one tiny), and only the last query sees it."""
    for n, new in ((5, 2), (100, 4), (700, 3)):
        k, v = _huge_rows(n, 1, d, [n - 1], None, v_log, seed=n)
        kv, bt = _cache(cuda, [k], [v], 2)
        q = _q(cuda, new, hq, d, dtype, 5)
        _check(*_chunk(cuda, q, kv, bt, [n], [new], d ** -0.5), q, kv, bt, [n], [new], d ** -0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,d", [(2, 64), (4, 128), (2, 256)])
@pytest.mark.parametrize("v_log", [12, 30, 60])
def test_decode_beside_a_huge_value_of_no_weight(cuda, dtype, hq, d, v_log):
    lens = [5, 40, 333, 6000]
    rows = [_huge_rows(n, 1, d, {0, n // 2, n - 2}, 13, v_log, seed=n) for n in lens]
    kv, bt = _cache(cuda, [r[0] for r in rows], [r[1] for r in rows], 3)
    q = _q(cuda, len(lens), hq, d, dtype, 6)
    q[:, :, 0] = 4
    _check(*_decode(cuda, q, kv, bt, lens, d ** -0.5), q, kv, bt, lens, [1] * 4, d ** -0.5, empty=float("nan"))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,d", [(2, 64), (4, 128), (2, 256)])
@pytest.mark.parametrize("spread", [6.0, 14.0])
def test_few_rows_over_values_of_every_size(cuda, dtype, hq, d, spread):
    rng = np.random.default_rng(d)
    lens = [3, 16, 200, 2500]
    k = [rng.standard_normal((n, 1, d)) for n in lens]
    v = [rng.standard_normal((n, 1, d)) * 2.0 ** np.clip(rng.standard_normal((n, 1, 1)) * spread, -33, 33) for n in lens]
    for x in v:
        x[::5] = 0
    kv, bt = _cache(cuda, k, v, 4)
    q = _q(cuda, len(lens), hq, d, dtype, 7)
    _check(*_decode(cuda, q, kv, bt, lens, d ** -0.5), q, kv, bt, lens, [1] * 4, d ** -0.5, empty=float("nan"))
    new = [2, 3, 4, 3]
    q = _q(cuda, sum(new), hq, d, dtype, 8)
    _check(*_chunk(cuda, q, kv, bt, lens, new, d ** -0.5), q, kv, bt, lens, new, d ** -0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [40, 150])
@pytest.mark.parametrize("k_log,v_log,at", [
    (None, 20, -3), (None, 45, -3),  # hidden from all but the last three queries
    (13, 18, 0), (13, 45, 0),        # seen by all, of no weight
    (30, 0, -3), (28, 45, -60),
    (None, -40, 3),                  # tiny beside its tile
])
def test_chunks_beside_a_huge_row(cuda, dtype, d, new, k_log, v_log, at):
    n = 300
    k, v = _huge_rows(n, 1, d, [at % n], k_log, v_log, seed=9)
    kv, bt = _cache(cuda, [k], [v], 5)
    q = _q(cuda, new, 2, d, dtype, 10)
    q[:, :, 0] = 4
    _check(*_chunk(cuda, q, kv, bt, [n], [new], d ** -0.5), q, kv, bt, [n], [new], d ** -0.5)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_cut_into_shares_beside_a_huge_row(cuda, dtype, d):
    """Some CTAs of a row tile meet the huge rows, others do not; pages that are not there, NaN rows."""
    lens, new = [5000, 300, 4100], [40, 3, 50]
    rows = [_huge_rows(n, 2, d, [n // 3, n - 2], 13, 40, seed=n) for n in lens]
    kv, bt = _cache(cuda, [r[0] for r in rows], [r[1] for r in rows], 6)
    bt[0, 100:120] = -1
    bt[0, 104] = 1 << 20
    q = _q(cuda, sum(new), 8, d, dtype, 11)
    q[:, :, 0] = 4
    out, lse = _chunk(cuda, q, kv, bt, lens, new, d ** -0.5)
    _check(out, lse, q, kv, bt, lens, new, d ** -0.5)
    page, slot = int(bt[2, (4100 - 20) // 16]), (4100 - 20) % 16  # a NaN value row that the last 20 queries see
    kv.v_codes.view(torch.uint8)[page, slot] = 0x7F
    kv.v_scales[page, :, slot] = 255
    got, _ = _chunk(cuda, q, kv, bt, lens, new, d ** -0.5)
    assert torch.isnan(got[-20:]).all() and torch.equal(got[:-20], out[:-20])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_over_scales_that_move(cuda, dtype, d):
    """Values that grow and shrink from tile to tile by less than the span that fp16 holds exactly."""
    rng = np.random.default_rng(d)
    n, new = 900, 150
    log = np.concatenate([np.full(128, x) for x in (0, 5, 9, 2, -1, 8, 9, 3)])[:n, None, None]
    k, v = rng.standard_normal((n, 1, d)) * 2.0 ** (log / 4), rng.standard_normal((n, 1, d)) * 2.0 ** log
    kv, bt = _cache(cuda, [k], [v], 7)
    q = _q(cuda, new, 2, d, dtype, 12)
    _check(*_chunk(cuda, q, kv, bt, [n], [new], 0.05), q, kv, bt, [n], [new], 0.05)


# ---- queries that are not finite ----------------------------------------------------
@pytest.mark.parametrize("d,new", [(64, 3), (128, 3), (256, 3), (64, 60), (128, 60), (128, 200)])
def test_infinite_queries_give_nan(cuda, d, new):
    """A score of inf or -inf in every token is no softmax: NaN, also where all of them are -inf."""
    rng = np.random.default_rng(d)
    n = new + 30
    k, v = np.abs(rng.standard_normal((n, 1, d))) + 0.5, rng.standard_normal((n, 1, d))
    kv, bt = _cache(cuda, [k], [v], 8)
    q = _q(cuda, new, 2, d, "bf16", 13)
    clean, clean_lse = _chunk(cuda, q, kv, bt, [n], [new], 0.1)
    q[0, 0, 3], q[1, 1, 5], q[2, 0, 7] = -float("inf"), float("inf"), float("nan")
    out, lse = _chunk(cuda, q, kv, bt, [n], [new], 0.1)
    for i, h in ((0, 0), (1, 1), (2, 0)):
        assert torch.isnan(out[i, h]).all(), (i, h)
        out[i, h], lse[i, h] = clean[i, h], clean_lse[i, h]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


# ---- values at the top of the range --------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_largest_values_do_not_overflow(cuda, d):
    """Every value the largest that the format holds: so is the mean, however many parts it is joined from."""
    n, top = 3000, 448 * 2.0 ** 119
    rng = np.random.default_rng(d)
    kv, bt = _cache(cuda, [rng.standard_normal((n, 2, d))], [np.full((n, 2, d), top)], 9)
    q = _q(cuda, 1, 4, d, "bf16", 14)
    _check(*_decode(cuda, q, kv, bt, [n], 0.1), q, kv, bt, [n], [1], 0.1)
    for new in (3, 60, 200):
        q = _q(cuda, new, 4, d, "bf16", 15)
        _check(*_chunk(cuda, q, kv, bt, [n], [new], 0.1), q, kv, bt, [n], [new], 0.1)


# ---- the second part of fp16 weights -------------------------------------------------
def _cancelling(n, h_kv, d, seed):
    """Values in pairs of opposite sign, keys small: the result is small beside the values, and a weight that was
    rounded to 11 bits shows."""
    rng = np.random.default_rng(seed)
    k, v = rng.standard_normal((n, h_kv, d)) * 0.25, rng.standard_normal((n, h_kv, d))
    v[1::2] = -v[:n // 2 * 2:2]
    return k, v


@pytest.mark.parametrize("d,new,n", [(64, 1, 16), (128, 1, 32), (256, 1, 16), (64, 3, 40), (64, 40, 60), (128, 40, 64),
                                     (128, 150, 160)])
def test_weights_of_fp16_results_keep_both_parts(cuda, d, new, n):
    k, v = _cancelling(n, 1, d, seed=d)
    kv, bt = _cache(cuda, [k], [v], 10)
    q = _q(cuda, new, 2, d, "fp16", 16, 0.25)
    _check(*_chunk(cuda, q, kv, bt, [n], [new], d ** -0.5), q, kv, bt, [n], [new], d ** -0.5)


# ---- softmax scales of zero and below -------------------------------------------------
@pytest.mark.parametrize("hq,h_kv,d,new,lens", [(4, 2, 128, [60, 9], [160, 30]), (4, 2, 64, [3, 1], [20, 500]),
                                                (4, 1, 256, [20, 5], [90, 5]), (1, 1, 64, [1] * 4200, [3] * 4200)])
def test_log_sums_of_scales_of_zero_and_below(cuda, hq, h_kv, d, new, lens):
    rng = np.random.default_rng(d)
    if len(lens) > 100:  # more requests than are split between workers, over two pages
        kv, bt = _cache(cuda, [rng.standard_normal((32, h_kv, d))], [rng.standard_normal((32, h_kv, d))], 11)
        bt = bt[0][torch.arange(len(lens), device=cuda) % 2][:, None].contiguous()
    else:
        kv, bt = _cache(cuda, *([rng.standard_normal((n, h_kv, d)) for n in lens] for _ in (0, 1)), 11)
        bt[0, 1] = -1  # a page that is not there
    q = _q(cuda, sum(new), hq, d, "bf16", 17)
    for scale in (-0.1, 0.0):
        _check(*_chunk(cuda, q, kv, bt, lens, new, scale), q, kv, bt, lens, new, scale)


# ---- 64-bit page ids and lengths -------------------------------------------------------
def test_ids_and_lengths_past_32_bits(cuda):
    """Page ids of a 64-bit table that lie outside the pool stay outside it when they are narrowed."""
    from unifiedkv_b200.kv_quant import dequantize_pages, quantize_append
    rng = np.random.default_rng(0)
    kv, bt = _cache(cuda, [rng.standard_normal((48, 2, 64))], [rng.standard_normal((48, 2, 64))], 12)
    before = [t.view(torch.uint8).clone() for t in kv]
    x = torch.ones(2, 2, 64, device=cuda, dtype=torch.bfloat16)
    far = torch.tensor([[2 ** 32 + 1], [-2 ** 32]], device=cuda)
    quantize_append(kv, x, x, far, _i32(cuda, [1, 1]))
    quantize_append(kv, x, x, torch.zeros(2, 1, dtype=torch.int64, device=cuda),
                    torch.tensor([2 ** 32 + 1, 2 - 2 ** 32], device=cuda))
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, kv))
    k, v = dequantize_pages(kv, far, _i32(cuda, [0, 4, 8]), 8)
    assert (k == 0).all() and (v == 0).all()
    out, lse = _decode(cuda, x, kv, far, [4, 4], 0.1)
    assert torch.isnan(out).all() and torch.isneginf(lse).all()


# ---- lengths that the host holds --------------------------------------------------------
def test_calls_with_numbers_of_the_host_refuse_a_capture(cuda):
    """Their copies to the device could not be replayed; the capture around them goes on."""
    from unifiedkv_b200.kv_quant import QuantPagedKVPool, paged_chunk_prefill_q8
    pool = QuantPagedKVPool(16, 1, 2, 64, device=cuda, n_total=4)
    kv = pool.layer(0)
    bt = torch.arange(4, dtype=torch.int32, device=cuda)[None]
    q = _q(cuda, 5, 4, 64, "bf16", 18)
    x = torch.ones(2, 20, 64, device=cuda, dtype=torch.bfloat16)
    calls = [lambda: paged_chunk_prefill_q8(q, kv, bt, [9], [5], n_rep=2), lambda: pool.write_kv_to_blocks(0, [0, 1], x, x),
             lambda: pool.write_one_token(0, 1, 4, x[:, :1], x[:, :1]), lambda: pool.read_kv_from_blocks(0, [0, 1], 20)]
    for call in calls[1:] + calls[:1]:
        call()
    want = calls[0]()
    torch.cuda.synchronize()
    cu, lens = _i32(cuda, [0, 5]), _i32(cuda, [14])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            with pytest.raises(RuntimeError, match="_unavailable:host_numbers_in_capture$"):
                call()
        out = paged_chunk_prefill_q8(q, kv, bt, n_rep=2, cu_seqlens_q=cu, seqlens_k=lens, max_seqlen_q=5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ---- the exact path of the chunk kernel in other calls ------------------------------------
@pytest.mark.parametrize("d,new", [(64, 40), (128, 40), (128, 150)])
def test_huge_rows_without_a_causal_mask_and_in_a_replayed_graph(cuda, d, new):
    """Every query sees every token; the huge rows come and go between replays, as do the lengths."""
    from unifiedkv_b200.kv_quant import paged_chunk_prefill_q8
    lens, start = [300, new + 5], [300, 260]
    rows = [_huge_rows(n, 1, d, [n // 2], 13, 40, seed=n) for n in start]
    kv, bt = _cache(cuda, [r[0] for r in rows], [r[1] for r in rows], 13)
    calm, _ = _cache(cuda, *([np.random.default_rng(i).standard_normal((n, 1, d)) for n in start] for i in (0, 1)), 13)
    q = _q(cuda, 2 * new, 2, d, "bf16", 19)
    q[:, :, 0] = 4
    for b in (kv, calm):
        _check(*_chunk(cuda, q, b, bt, lens, [new, new], 0.1, causal=False), q, b, bt, lens, [new, new], 0.1, causal=False)
    live = type(kv)(*(t.clone() for t in kv))
    sk, cu, lse = _i32(cuda, start), _i32(cuda, [0, new, 2 * new]), torch.zeros(2 * new, 2, device=cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_chunk_prefill_q8(q, live, bt, softmax_scale=0.1, n_rep=2, cu_seqlens_q=cu, seqlens_k=sk,
                                     max_seqlen_q=new, lse_out=lse)
    for source, n in ((kv, start), (calm, lens), (kv, lens), (calm, start)):
        for a, b in zip(live, source):
            a.copy_(b)
        sk.copy_(_i32(cuda, n))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, lse, q, live, bt, n, [new, new], 0.1)
