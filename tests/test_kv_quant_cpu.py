"""CPU tests of the 8-bit paged KV cache: the oracle's format against torch's own e4m3
cast, the pool's bookkeeping, and every refusal of the operators (all run before any
device work, so CPU tensors reach them)."""
import numpy as np
import pytest
import torch

from oracle import kv_quant as oracle
from unifiedkv_b200 import _lib, kv_quant
from unifiedkv_b200.kv_quant import QuantPagedKV, QuantPagedKVPool


def _kv(n=5, h=2, d=64, device="cpu"):
    codes = torch.zeros(n, 16, h, d, dtype=torch.float8_e4m3fn, device=device)
    scales = torch.zeros(n, h, 16, dtype=torch.uint8, device=device)
    return QuantPagedKV(codes, codes.clone(), scales, scales.clone())


def test_oracle_codes_are_the_e4m3_numbers():
    codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(codes.view(torch.float8_e4m3fn).double().numpy(), oracle.E4M3)


def test_oracle_quantises_as_the_cast_does():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(200, 64, generator=g) * torch.exp2(torch.randn(200, 1, generator=g) * 20)
    x[0] = 0
    x[1] = torch.linspace(0, 448, 64)
    x[2, :] = 449.0
    x[3] = 3.4e38
    x[4] *= 1e-44
    codes, byte = oracle.quantise(x.numpy())
    e = byte.astype(int) - 127
    y = np.clip(x.double().numpy() / 2.0 ** e[:, None], -448, 448)
    want = torch.from_numpy(y).float().to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(codes & 0x7F, want & 0x7F)
    assert byte[0] == 0 and byte[1] == 127 and byte[2] == 128 and byte[3] == 246
    amax = x.abs().amax(1).double().numpy()
    ok = (e > -127) & (e < 119)
    assert (amax[ok] <= 448 * 2.0 ** e[ok]).all() and (amax[ok] > 224 * 2.0 ** e[ok]).all()
    codes, byte = oracle.quantise(np.array([[1.0, np.inf], [np.nan, 2.0]]))
    assert (byte == 255).all() and (codes == 0x7F).all()


def test_stored_elements_are_within_half_a_step():
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(500, 128, generator=g) * 3).double().numpy()
    codes, byte = oracle.quantise(x)
    e = 2.0 ** (byte.astype(np.float64) - 127)[:, None]
    off = np.abs(oracle.dequantise(codes, byte) - x)
    assert (off <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * e)).all()


def test_cache_refusals():
    kv = _kv()
    k = torch.zeros(2, 2, 64)
    bt = torch.zeros(2, 3, dtype=torch.int32)
    lens = torch.ones(2, dtype=torch.int32)

    def call(c=kv, k=k, v=None, bt=bt, lens=lens, cu=None):
        return kv_quant.quantize_append(c, k, k if v is None else v, bt, lens, cu)

    half = kv.k_codes[:, :, :1]
    cases = [
        (lambda: call(kv._replace(k_codes=kv.k_codes[0])), "cache_rank"),
        (lambda: call(kv._replace(v_codes=kv.v_codes[:3])), "cache_rank"),
        (lambda: call(QuantPagedKV(kv.k_codes[:, :8], kv.v_codes[:, :8], *kv[2:])), "block_size_8"),
        (lambda: call(_kv(d=96)), "head_dim_96"),
        (lambda: call(kv._replace(k_codes=kv.k_codes.view(torch.uint8), v_codes=kv.v_codes.view(torch.uint8))), "cache_dtype"),
        (lambda: call(kv._replace(k_scales=kv.k_scales.transpose(1, 2))), "scales"),
        (lambda: call(kv._replace(v_scales=kv.v_scales.to(torch.int32))), "scales"),
        (lambda: call(QuantPagedKV(half, half, kv.k_scales[:, :1], kv.v_scales[:, :1])), "cache_layout"),
        (lambda: call(k=k[0]), "new_token"),
        (lambda: call(k=k[:, :1]), "new_token"),
        (lambda: call(v=k[:1]), "new_token"),
        (lambda: call(v=k.half()), "dtype_mismatch"),
        (lambda: call(bt=bt[0]), "block_table_rank"),
        (lambda: call(bt=bt[:1]), "seqlens"),
        (lambda: call(lens=lens[:1]), "seqlens"),
        (lambda: call(cu=lens), "cu_seqlens"),
    ]
    for fn, token in cases:
        with pytest.raises(RuntimeError, match=f"^q8_append_shape_unsupported:{token}$"):
            fn()
    with pytest.raises(RuntimeError, match="dtype_torch.float64"):
        call(k=k.double())
    with pytest.raises(RuntimeError, match="^q8_append_unavailable:tensors_not_on_cuda$"):
        call()


def test_readback_refusals():
    kv = _kv()
    bt = torch.zeros(2, 3, dtype=torch.int32)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    out = torch.zeros(2, 2, 64)

    def call(total=2, cu=cu, bt=bt, starts=None, out=None, dtype=torch.bfloat16):
        return kv_quant.dequantize_pages(kv, bt, cu, total, dtype=dtype, starts=starts, out=out)

    wide = torch.zeros(2, 2, 65)[:, :, :64]
    cases = [
        (lambda: call(total=-1), "total_-1"),
        (lambda: call(cu=cu[:2]), "cu_seqlens"),
        (lambda: call(bt=bt[0]), "block_table_rank"),
        (lambda: call(starts=cu), "starts"),
        (lambda: call(out=(out, out[:1])), "out"),
        (lambda: call(out=(out, out.half())), "out"),
        (lambda: call(total=3, out=(out, out)), "out"),
        (lambda: call(out=(wide, wide)), "out_layout"),
        (lambda: call(out=(out, out.transpose(0, 1))), "out_layout"),
    ]
    for fn, token in cases:
        with pytest.raises(RuntimeError, match=f"^q8_dequantize_shape_unsupported:{token}$"):
            fn()
    with pytest.raises(RuntimeError, match="dtype_torch.int8"):
        call(dtype=torch.int8)
    with pytest.raises(RuntimeError, match="^q8_dequantize_unavailable:tensors_not_on_cuda$"):
        call()


def test_attention_refusals():
    kv = _kv()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    bt = torch.zeros(2, 3, dtype=torch.int32)
    lens = torch.ones(2, dtype=torch.int32)

    def decode(q=q, bt=bt, lens=lens, n_rep=2, lse=None, kv=kv):
        return kv_quant.page16_decode_attention_q8(q, kv, bt, lens, softmax_scale=0.1, n_rep=n_rep, lse_out=lse)

    cases = [
        (lambda: decode(q=q[0]), "q_dim_2"),
        (lambda: decode(q=q[:0], bt=bt[:0], lens=lens[:0]), "empty"),
        (lambda: decode(q=q[:, :, :32]), "head_dim_32"),
        (lambda: decode(q=q[:, :3]), "gqa"),
        (lambda: decode(n_rep=4), "gqa"),
        (lambda: decode(q=q.float()), "dtype_torch.float32"),
        (lambda: decode(bt=bt[0]), "block_table_rank"),
        (lambda: decode(bt=bt[:1]), "block_table_batch"),
        (lambda: decode(lens=lens[:1]), "seqlens"),
        (lambda: decode(lse=torch.zeros(2, 3)), "lse_out"),
        (lambda: decode(lse=torch.zeros(2, 4, dtype=torch.float64)), "lse_out"),
    ]
    for fn, token in cases:
        with pytest.raises(RuntimeError, match=f"^page16_native_shape_unsupported:{token}$"):
            fn()
    with pytest.raises(RuntimeError, match="^page16_native_unavailable:tensors_not_on_cuda$"):
        decode()

    def chunk(past=(0, 0), new=(1, 1), **kw):
        return kv_quant.paged_chunk_prefill_q8(q, kv, bt, past, new, n_rep=2, **kw)

    for bad in (((0,), (1, 1)), ((0, 0), (1, 2)), ((0, 0), (3, -1)), (None, None)):
        with pytest.raises(RuntimeError, match="^prefill_shape_unsupported:chunk_lens$"):
            chunk(*bad)
    with pytest.raises(RuntimeError, match="^prefill_shape_unsupported:cu_seqlens$"):
        chunk(cu_seqlens_q=lens, seqlens_k=lens)
    with pytest.raises(RuntimeError, match="^prefill_unavailable:tensors_not_on_cuda$"):
        chunk()


def test_library_checks_without_a_gpu():
    """The C entry points check their arguments before any device work."""
    L = _lib.load()
    p = torch.zeros(4096, dtype=torch.uint8)
    a = (p.data_ptr() + 15) // 16 * 16

    def append(d=64, h=2, pages=3, ps=2048, ss=32, total=1, batch=1, dtype=2, kst=128, base=a, cu=None):
        return L.bpkv_q8_append(base, a, a, a, a, a, a, cu, a, batch, total, h, d, 1, pages, kst, 64, 128, 64, ps, ss,
                                1, dtype, None)

    for kw, token in ((dict(d=96), "head_dim_96"), (dict(h=0), "empty"), (dict(ps=2047), "alignment"), (dict(ss=8), "alignment"),
                      (dict(dtype=7), "dtype_7"), (dict(total=2), "seqlens"), (dict(kst=127), "alignment"),
                      (dict(base=a + 2), "alignment"), (dict(base=None), "null_pointer"), (dict(total=-1), "empty")):
        assert append(**kw) == _lib.BPKV_ERR_SHAPE and token in _lib.last_error(), (kw, _lib.last_error())
    assert append(total=0, batch=0) == 0  # nothing to do: no launch

    def attend(hq=4, h=2, d=64, batch=1, total=1, max_q=1, cu=None, dtype=2, q=a, ws=None, ws_bytes=0, qst=256, max_blocks=1):
        return L.bpkv_q8_attention(q, a, a, a, a, a, cu, a, a, None, batch, total, hq, h, d, max_blocks, 3, max_q, qst, 64, 2048, 32, 1,
                                   0.1, 1, 0, dtype, ws, ws_bytes, None)

    for kw, token in ((dict(hq=3), "gqa"), (dict(d=80), "head_dim_80"), (dict(dtype=0), "dtype_0"), (dict(max_q=2), "max_seqlen_q"), (dict(total=2), "max_seqlen_q"),
                      (dict(q=None), "null_pointer"), (dict(q=a + 4), "alignment"), (dict(qst=100), "alignment"),
                      (dict(max_blocks=1 << 27), "max_blocks")):
        assert attend(**kw) == _lib.BPKV_ERR_SHAPE and token in _lib.last_error(), (kw, _lib.last_error())
    assert attend() == _lib.BPKV_ERR_WORKSPACE and "workspace" in _lib.last_error()
    b = (a + 31) // 32 * 32
    assert attend(ws=b + 16, ws_bytes=1 << 30) == _lib.BPKV_ERR_SHAPE and "workspace_alignment" in _lib.last_error()
    assert attend(hq=2050, h=1025) == _lib.BPKV_ERR_SHAPE and "kv_heads" in _lib.last_error()
    assert attend(batch=0, total=0) == 0
    need = L.bpkv_q8_attention_workspace_size
    assert need(1, 1, 3, 2, 64, 9, 1, 0.1) == 0 and need(1, 1, 4, 2, 96, 9, 1, 0.1) == 0
    assert need(4, 4, 32, 8, 128, 9, 1, 0.1) > 0


def test_missing_library_fails_loudly():
    """Without the library every operator raises and nothing is computed (a fresh interpreter: the real library
    is loaded in this one)."""
    import subprocess
    import sys
    from pathlib import Path
    code = r'''
import torch
from pathlib import Path
import unifiedkv_b200._lib as L
L.LIB_PATH = Path("/nonexistent/libbpkv.so")
from unifiedkv_b200 import kv_quant
c = torch.zeros(2, 16, 1, 64, dtype=torch.float8_e4m3fn)
s = torch.zeros(2, 1, 16, dtype=torch.uint8)
kv = kv_quant.QuantPagedKV(c, c, s, s)
x, bt, n = torch.zeros(1, 1, 64), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
cu = torch.tensor([0, 1], dtype=torch.int32)
calls = [lambda: kv_quant.quantize_append(kv, x, x, bt, n), lambda: kv_quant.dequantize_pages(kv, bt, cu, 1),
         lambda: kv_quant.page16_decode_attention_q8(x.half(), kv, bt, n, softmax_scale=0.1, n_rep=1),
         lambda: kv_quant.paged_chunk_prefill_q8(x.half(), kv, bt, [0], [1])]
for fn in calls:
    try:
        fn()
    except RuntimeError as exc:
        assert str(exc).startswith("page16_native_unavailable"), str(exc)
    else:
        raise AssertionError("ran without the library")
print("ok")
'''
    root = Path(__file__).resolve().parents[1]
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-3000:]


def test_pool_bookkeeping_and_layout():
    pool = QuantPagedKVPool(16, 3, 2, 64, device="cpu", n_total=10)
    assert pool.allocate_blocks(3) == [0, 1, 2] and pool.n_free == 7
    kv = pool.layer(1)
    assert kv.k_codes.dtype == torch.float8_e4m3fn and kv.k_codes.shape == (10, 16, 2, 64)
    assert kv.k_scales.shape == (10, 2, 16) and kv.k_scales.dtype == torch.uint8
    pool.free_blocks_by_ids([0, 1, 2])
    with pytest.raises(RuntimeError, match="q8_pool_shape_unsupported:head_dim_96"):
        QuantPagedKVPool(16, 1, 2, 96, device="cpu", n_total=4)


def test_sixteen_bit_paths_refuse_an_8_bit_pool():
    """Codes mean nothing without their scales: what moves or reads 16-bit pages says no."""
    from unifiedkv_b200.chunked_prefill import append_chunk_kv, paged_chunk_prefill
    from unifiedkv_b200.offload import AsyncOffloadManager
    from unifiedkv_b200.page16_native import decode_append
    from unifiedkv_b200.pool import write_pages
    pool = QuantPagedKVPool(16, 1, 2, 64, device="cpu", n_total=4)
    kc, vc = pool.k_cache[0], pool.v_cache[0]
    x = torch.zeros(2, 20, 64, dtype=torch.bfloat16)
    bt = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="dtype_mismatch"):
        write_pages(kc, vc, x, x, [0, 1], None, -1, 0, 0)
    with pytest.raises(RuntimeError, match="dtype_mismatch"):
        append_chunk_kv(kc, vc, x, x, [0, 1], 3)
    with pytest.raises(RuntimeError, match="dtype_mismatch"):
        decode_append(x[:, :1].transpose(0, 1), x[:, :1].transpose(0, 1), kc, vc, bt, torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="dtype_mismatch"):
        paged_chunk_prefill(torch.zeros(3, 4, 64, dtype=torch.bfloat16), kc, vc, bt, [0], [3], 0.1, 2)
    with pytest.raises(RuntimeError, match="dtype_torch.float8_e4m3fn"):
        AsyncOffloadManager(pool, 1)
