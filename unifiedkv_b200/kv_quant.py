"""8-bit paged KV cache: writing it, reading it back, and attention over it.

The reference's pool holds 16-bit K and V (core/pool.py:20-71); this module adds a
pool of half the size and the operators that work on it:

  ``QuantPagedKVPool``           the pool (a ``PagedKVPool``: same pages, tables, free list)
  ``quantize_append``            new tokens of a ragged batch into their pages
  ``dequantize_pages``           ranges of cached tokens as dense K and V
  ``page16_decode_attention_q8`` one-token decode, beside ``page16_decode_attention``
  ``paged_chunk_prefill_q8``     chunks of new tokens, beside ``paged_chunk_prefill``

Format.  The K (or V) row of one token and KV head is ``head_dim`` e4m3 codes and one
scale byte: value = code * 2^(byte - 127).  The exponent is the smallest e in
[-127, 119] with max|row| <= 448 * 2^e, and the codes are the row divided by 2^e rounded
to nearest even: a stored element is off by at most 2^-4 of itself, or by 2^-10 * 2^e
where it lies below 2^-6 * 2^e.  A row with an infinity or a NaN is stored as NaN (byte
255).  One layer's cache is

  k_codes, v_codes    float8_e4m3fn [pages, 16, kv_heads, head_dim], each page dense
  k_scales, v_scales  uint8 [pages, kv_heads, 16], each page dense

A token costs 2 * kv_heads * (head_dim + 1) bytes.  head_dim is 64, 128 or 256.

Attention computes on the stored values: scores, softmax and sums in fp32, the products on
fp16 operands that hold the codes exactly.  An element of q is off by at most 2^-40 of the
largest of its row, a weight is rounded to 11 bits (22 for fp16 results) and counts as zero
below 2^-30 of the largest of its row.  What a row does not see, or gives no weight to, takes
nothing from it however large it is: up to a ratio of 2^72 between the values of a request
(but rows of K or V with a largest magnitude below 2^-118 count as zeros beside larger ones).
Scales that far apart cost time: chunks of many rows, where keys of 128 tokens or values of a
request differ by 2^15 and more in scale, take up to a hundred times as long.  A query row
with an infinity or a NaN gives NaN wherever it sees a token.

A page id outside the pool (-1 as of an offloaded page, or past its end) is never
touched: tokens on such a page are not written, read back as zeros, and are left out of
attention.  Every call runs on the current stream of its tensors' device without
synchronising with the host, and takes its scratch from torch's allocator.  Calls whose
lengths and tables are device tensors can be captured in a CUDA graph, and two graphs
never share scratch.  Those that take them as Python numbers (``past_lens`` and
``chunk_lens``, the pool's page I/O) copy them to the device when they are called, which
no graph can replay: they refuse to be captured.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Tuple

import torch

from . import _lib
from .pool import PagedKVPool

HEAD_DIMS = (64, 128, 256)

# the current device and stream handle without building Python objects: a call's host time is what a short one takes
_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_stream = (torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream")
           else lambda index: torch.cuda.current_stream(index).cuda_stream)


class QuantPagedKV(NamedTuple):
    """One layer of an 8-bit paged cache (views are fine: only a page has to be dense)."""
    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def _check_kv(kv: QuantPagedKV, what: str) -> Tuple[int, int, int]:
    """Sizes (pages, kv_heads, head_dim) of a well-formed layer."""
    kc, vc, ks, vs = kv
    shape, scales = kc.shape, ks.shape
    if len(shape) != 4 or vc.shape != shape:
        raise RuntimeError(f"{what}_shape_unsupported:cache_rank")
    n, page, h_kv, d = shape
    if page != 16:
        raise RuntimeError(f"{what}_shape_unsupported:block_size_{page}")
    if d not in HEAD_DIMS:
        raise RuntimeError(f"{what}_shape_unsupported:head_dim_{d}")
    if kc.dtype is not torch.float8_e4m3fn or vc.dtype is not torch.float8_e4m3fn:
        raise RuntimeError(f"{what}_shape_unsupported:cache_dtype")
    if scales != (n, h_kv, 16) or vs.shape != scales or ks.dtype is not torch.uint8 or vs.dtype is not torch.uint8:
        raise RuntimeError(f"{what}_shape_unsupported:scales")
    s, t = kc.stride(), ks.stride()
    if s[3] != 1 or (s[2] != d and h_kv > 1) or s[1] != h_kv * d or vc.stride() != s:
        raise RuntimeError(f"{what}_shape_unsupported:cache_layout")
    if t[2] != 1 or (t[1] != 16 and h_kv > 1) or vs.stride() != t:
        raise RuntimeError(f"{what}_shape_unsupported:cache_layout")
    return n, h_kv, d


def _check_device(what: str, dev: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    if dev.type != "cuda":
        raise RuntimeError(f"{what}_unavailable:tensors_not_on_cuda")
    for t in tensors:
        if t is not None and t.device != dev:
            raise RuntimeError(f"{what}_shape_unsupported:device_{t.device}")


def _refuse_capture(what: str, dev: torch.device) -> None:
    """For calls that copy the host's numbers: a graph would copy again from memory that is gone."""
    if dev.type == "cuda":
        with torch.cuda.device(dev):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{what}_unavailable:host_numbers_in_capture")


def _narrow(t: torch.Tensor) -> torch.Tensor:
    """int32; 64-bit numbers past its range stay far out (a page id out of the pool stays out of it)."""
    if t.dtype is torch.int32:
        return t
    if t.dtype is torch.int64:
        t = t.clamp(-2 ** 30, 2 ** 31 - 1)
    return t.to(torch.int32)


def _int32(t: torch.Tensor, what: str, name: str, numel: int) -> torch.Tensor:
    if t.numel() != numel:
        raise RuntimeError(f"{what}_shape_unsupported:{name}")
    t = _narrow(t)
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor, what: str, batch: Optional[int] = None) -> torch.Tensor:
    if t.dim() != 2:
        raise RuntimeError(f"{what}_shape_unsupported:block_table_rank")
    if batch is not None and t.shape[0] != batch:
        raise RuntimeError(f"{what}_shape_unsupported:block_table_batch")
    t = _narrow(t)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """The kernels read rows [.., head_dim] in 16-byte pieces: any token and head strides that keep those aligned."""
    per = 16 // t.element_size()
    s = t.stride()
    if s[2] == 1 and s[0] % per == 0 and s[1] % per == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def quantize_append(kv: QuantPagedKV, k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor,
                    seqlens_k: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None) -> None:
    """Quantise the new tokens of every request into their pages (in place).

    k_new/v_new: [total, kv_heads, head_dim] bf16, fp16 or fp32, new tokens of all
    requests packed; slices of a fused projection are read where they are.  seqlens_k
    [B] counts a request's tokens with the new ones; cu_seqlens_q [B+1] bounds its new
    tokens in the packed rows (left out: one new token per request, a decode step).
    Token i of n goes to position seqlens_k - n + i.  Tokens whose position has no page
    (negative, past the table, a page id outside the pool) and rows behind the last
    sequence are skipped.  Two tokens of one call must not share a slot.
    """
    what = "q8_append"
    lib = _lib.lib()  # raises page16_native_unavailable when the library is missing
    n, h_kv, d = _check_kv(kv, what)
    if k_new.dim() != 3 or v_new.shape != k_new.shape or k_new.shape[1] != h_kv or k_new.shape[2] != d:
        raise RuntimeError(f"{what}_shape_unsupported:new_token")
    if v_new.dtype != k_new.dtype:
        raise RuntimeError(f"{what}_shape_unsupported:dtype_mismatch")
    code = _lib.dtype_code(k_new.dtype)
    bt = _table(block_table, what)
    B, total = bt.shape[0], k_new.shape[0]
    if cu_seqlens_q is None and total != B:
        raise RuntimeError(f"{what}_shape_unsupported:seqlens")
    lens = _int32(seqlens_k, what, "seqlens", B)
    cu = None if cu_seqlens_q is None else _int32(cu_seqlens_q, what, "cu_seqlens", B + 1)
    dev = k_new.device
    _check_device(what, dev, *kv, v_new, bt, lens, cu)
    if dev.index != _device():  # the library launches on the current device
        with torch.cuda.device(dev):
            return quantize_append(kv, k_new, v_new, bt, lens, cu)
    k, v = _aligned(k_new), _aligned(v_new)
    ks, vs = k.stride(), v.stride()
    rc = lib.bpkv_q8_append(
        k.data_ptr(), v.data_ptr(), kv.k_codes.data_ptr(), kv.v_codes.data_ptr(), kv.k_scales.data_ptr(),
        kv.v_scales.data_ptr(), bt.data_ptr(), _lib.ptr(cu), lens.data_ptr(), B, total, h_kv, d, bt.shape[1], n,
        ks[0], ks[1], vs[0], vs[1], kv.k_codes.stride(0), kv.k_scales.stride(0), bt.stride(0), code,
        _stream(dev.index))
    if rc:
        _lib.check(rc, what)


def dequantize_pages(kv: QuantPagedKV, block_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
                     dtype: torch.dtype = torch.bfloat16, starts: Optional[torch.Tensor] = None,
                     out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Ranges of cached tokens as dense K and V, [total, kv_heads, head_dim] each, packed.

    Rows cu_seqlens[b] .. cu_seqlens[b+1]-1 are tokens starts[b], starts[b]+1, ... of
    request b (starts left out: from its first token).  ``total`` is cu_seqlens[-1], known
    to the host.  The values are exact in fp32 and bf16; fp16 rounds values below its
    normal range and overflows above 65504.  Tokens without a page read as zeros.
    ``out``: a pair of equally strided tensors to fill (unit stride of head_dim, other
    strides multiples of 16 bytes; no two elements in one place); rows behind the last sequence keep what they held.
    """
    what = "q8_dequantize"
    lib = _lib.lib()  # raises page16_native_unavailable when the library is missing
    n, h_kv, d = _check_kv(kv, what)
    bt = _table(block_table, what)
    B = bt.shape[0]
    total = int(total)
    if total < 0:
        raise RuntimeError(f"{what}_shape_unsupported:total_{total}")
    cu = _int32(cu_seqlens, what, "cu_seqlens", B + 1)
    st = None if starts is None else _int32(starts, what, "starts", B)
    dev = kv.k_codes.device
    if out is None:
        code = _lib.dtype_code(dtype)
        k = torch.empty((total, h_kv, d), dtype=dtype, device=dev)
        v = torch.empty((total, h_kv, d), dtype=dtype, device=dev)
    else:
        k, v = out
        code = _lib.dtype_code(k.dtype)
        if k.shape != (total, h_kv, d) or v.shape != k.shape or v.dtype != k.dtype:
            raise RuntimeError(f"{what}_shape_unsupported:out")
        per = 16 // k.element_size()
        s = k.stride()
        if s[2] != 1 or s[0] % per or s[1] % per or v.stride() != s or k.data_ptr() % 16 or v.data_ptr() % 16:
            raise RuntimeError(f"{what}_shape_unsupported:out_layout")
        if (s[0] == 0 and total > 1) or (s[1] == 0 and h_kv > 1) or (total > 0 and k.data_ptr() == v.data_ptr()):
            raise RuntimeError(f"{what}_shape_unsupported:out_overlap")
    _check_device(what, dev, *kv, bt, cu, st, k, v)
    if dev.index != _device():  # the library launches on the current device
        with torch.cuda.device(dev):
            return dequantize_pages(kv, bt, cu, total, starts=st, out=(k, v))
    rc = lib.bpkv_q8_dequantize(
        kv.k_codes.data_ptr(), kv.v_codes.data_ptr(), kv.k_scales.data_ptr(), kv.v_scales.data_ptr(), bt.data_ptr(),
        cu.data_ptr(), _lib.ptr(st), k.data_ptr(), v.data_ptr(), B, total, h_kv, d, bt.shape[1], n,
        kv.k_codes.stride(0), kv.k_scales.stride(0), bt.stride(0), k.stride(0), k.stride(1), code,
        _stream(dev.index))
    if rc:
        _lib.check(rc, what)
    return k, v


def _attention(what: str, q: torch.Tensor, kv: QuantPagedKV, block_table: torch.Tensor, seqlens_k: torch.Tensor,
               cu_seqlens_q: Optional[torch.Tensor], max_q: int, softmax_scale: float, n_rep: int, causal: bool,
               lse_out: Optional[torch.Tensor]) -> torch.Tensor:
    lib = _lib.lib()  # raises page16_native_unavailable when the library is missing
    n, h_kv, d = _check_kv(kv, what)
    shape = q.shape
    if len(shape) != 3:
        raise RuntimeError(f"{what}_shape_unsupported:q_dim_{q.dim()}")
    total, h_q, dq = shape
    if dq != d:
        raise RuntimeError(f"{what}_shape_unsupported:head_dim_{dq}")
    if h_q == 0 or h_kv == 0 or h_q != h_kv * int(n_rep):
        raise RuntimeError(f"{what}_shape_unsupported:gqa")
    if q.dtype != torch.bfloat16 and q.dtype != torch.float16:
        raise RuntimeError(f"{what}_shape_unsupported:dtype_{q.dtype}")
    code = _lib.dtype_code(q.dtype)
    bt = _table(block_table, what, total if cu_seqlens_q is None else None)
    B = bt.shape[0]
    lens = _int32(seqlens_k, what, "seqlens", B)
    cu = None if cu_seqlens_q is None else _int32(cu_seqlens_q, what, "cu_seqlens", B + 1)
    if lse_out is not None and (lse_out.dtype != torch.float32 or lse_out.numel() != total * h_q
                                or not lse_out.is_contiguous()):
        raise RuntimeError(f"{what}_shape_unsupported:lse_out")
    dev = q.device
    _check_device(what, dev, *kv, bt, lens, cu, lse_out)
    if dev.index != _device():  # the library launches on the current device
        with torch.cuda.device(dev):
            return _attention(what, q, kv, bt, lens, cu, max_q, softmax_scale, n_rep, causal, lse_out)
    q = _aligned(q)
    out = q.new_empty(shape)
    max_blocks = bt.shape[1]
    ws_bytes = lib.bpkv_q8_attention_workspace_size(B, total, h_q, h_kv, d, max_blocks, max_q, softmax_scale)
    ws = q.new_empty(ws_bytes // 2) if ws_bytes else None
    qs = q.stride()
    rc = lib.bpkv_q8_attention(
        q.data_ptr(), kv.k_codes.data_ptr(), kv.v_codes.data_ptr(), kv.k_scales.data_ptr(), kv.v_scales.data_ptr(),
        bt.data_ptr(), _lib.ptr(cu), lens.data_ptr(), out.data_ptr(), _lib.ptr(lse_out), B, total, h_q, h_kv, d, max_blocks,
        n, max_q, qs[0], qs[1], kv.k_codes.stride(0), kv.k_scales.stride(0), bt.stride(0), float(softmax_scale),
        int(causal), int(cu is None), code, _lib.ptr(ws), ws_bytes, _stream(dev.index))
    if rc:
        _lib.check(rc, what)
    return out


def page16_decode_attention_q8(q: torch.Tensor, kv: QuantPagedKV, block_table: torch.Tensor,
                               cache_seqlens: torch.Tensor, *, softmax_scale: float, n_rep: int,
                               lse_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One-token decode attention over 8-bit pages; ``page16_decode_attention`` for a ``QuantPagedKV``.

    q: [B, q_heads, head_dim] bf16 or fp16 (token and head strides that are multiples of
    16 bytes are read in place).  block_table [B, max_blocks], cache_seqlens [B] lengths
    with the current token, whose K and V are already in the cache
    (``quantize_append(kv, k, v, block_table, cache_seqlens)``).  Returns a contiguous
    tensor like q.  As for the 16-bit pool, pages past the table are never read and a
    request without tokens gives NaN rows.  ``lse_out``: fp32 [B, q_heads], the natural
    log-sum-exp of the scaled scores (-inf for a request without tokens).
    """
    if q.dim() == 3 and q.shape[0] == 0:
        raise RuntimeError("page16_native_shape_unsupported:empty")
    return _attention("page16_native", q, kv, block_table, cache_seqlens, None, 1, softmax_scale, n_rep, True, lse_out)


def paged_chunk_prefill_q8(q_chunk: torch.Tensor, kv: QuantPagedKV, block_table: torch.Tensor, past_lens=None,
                           chunk_lens=None, softmax_scale: Optional[float] = None, n_rep: int = 1,
                           causal: bool = True, cu_seqlens_q: Optional[torch.Tensor] = None,
                           seqlens_k: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                           lse_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of chunks of new tokens over 8-bit pages; ``paged_chunk_prefill`` for a ``QuantPagedKV``.

    q_chunk: [total_q, q_heads, head_dim] bf16 or fp16, the requests' chunks packed.
    Query i of a chunk of n sees the tokens t <= len - n + i of its request (every token
    when ``causal`` is false), the chunk's own K and V being in the cache already
    (``quantize_append``).  Chunks of one or a few tokens (drafts) and long ones both
    run here.  Lengths as lists (past_lens, chunk_lens; not in a graph capture) or device tensors (cu_seqlens_q
    [B+1], seqlens_k [B] = past + chunk, with max_seqlen_q the longest chunk; of a longer
    chunk the rows past that may be left unwritten).  A query that sees no token gives
    zeros (lse -inf); rows behind the last sequence are not written.  ``softmax_scale``
    defaults to head_dim^-0.5.  A row's last bits depend on the other lengths of its
    batch, as they decide how its tokens are shared out.
    """
    what = "prefill"
    total = int(q_chunk.shape[0])
    if cu_seqlens_q is None or seqlens_k is None:
        if past_lens is None or chunk_lens is None:
            raise RuntimeError(f"{what}_shape_unsupported:chunk_lens")
        chunk_lens = [int(x) for x in chunk_lens]
        past_lens = [int(x) for x in past_lens]
        if len(chunk_lens) != len(past_lens) or sum(chunk_lens) != total or min(chunk_lens + past_lens, default=0) < 0:
            raise RuntimeError(f"{what}_shape_unsupported:chunk_lens")
        cu = [0]
        for x in chunk_lens:
            cu.append(cu[-1] + x)
        dev = q_chunk.device
        _refuse_capture(what, dev)
        cu_seqlens_q = torch.tensor(cu, dtype=torch.int32).to(dev, non_blocking=True)
        seqlens_k = torch.tensor([p + c for p, c in zip(past_lens, chunk_lens)], dtype=torch.int32).to(dev, non_blocking=True)
        max_q = max(chunk_lens, default=0)
    else:
        max_q = total if max_seqlen_q is None else min(int(max_seqlen_q), total)
    scale = q_chunk.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    return _attention(what, q_chunk, kv, block_table, seqlens_k, cu_seqlens_q, max_q, scale, n_rep, bool(causal), lse_out)


class QuantPagedKVPool(PagedKVPool):
    """A ``PagedKVPool`` whose pages are 8-bit: the same page ids, tables, free list and watermarks.

    ``k_cache``/``v_cache`` are float8_e4m3fn codes [L, N, 16, h_kv, d]; the scales are
    ``k_scales``/``v_scales``, uint8 [L, N, h_kv, 16].  ``layer(l)`` is what the operators
    above take.  ``out_dtype`` is the type of ``read_kv_from_blocks``.  The offload manager
    and the compacting writeback move 16-bit pages and refuse this pool.
    """

    def __init__(self, block_size: int, num_layers: int, num_kv_heads: int, head_dim: int,
                 out_dtype: torch.dtype = torch.bfloat16, gpu_mem_frac: float = 0.75, cpu_mem_gb: float = 48.0,
                 *, device: Optional[torch.device] = None, n_total: Optional[int] = None):
        if int(head_dim) not in HEAD_DIMS:
            raise RuntimeError(f"q8_pool_shape_unsupported:head_dim_{head_dim}")
        self.out_dtype = out_dtype
        self._k_scales: Optional[torch.Tensor] = None
        self._v_scales: Optional[torch.Tensor] = None
        super().__init__(block_size, num_layers, num_kv_heads, head_dim, torch.float8_e4m3fn, gpu_mem_frac,
                         cpu_mem_gb, device=device, n_total=n_total)
        if n_total is None:  # the base class sized the pages by their codes; the scales add 1 / head_dim
            self.N_total = max(1, self.N_total * self.head_dim // (self.head_dim + 1))
            self.free_blocks = list(range(self.N_total))
            self.N_wm_low = max(1, int(0.15 * self.N_total))
            self.N_wm_high = max(2, int(0.40 * self.N_total))

    def ensure_allocated(self) -> None:
        if self.is_allocated:
            return
        shape = (self.num_layers, self.N_total, self.num_kv_heads, self.B)
        k_scales = torch.zeros(shape, dtype=torch.uint8, device=self.device)
        v_scales = torch.zeros_like(k_scales)
        super().ensure_allocated()  # last: with its codes the pool counts as allocated
        self._k_scales, self._v_scales = k_scales, v_scales

    def release_if_empty(self) -> bool:
        if not super().release_if_empty():
            return False
        self._k_scales = None
        self._v_scales = None
        torch.cuda.empty_cache()
        return True

    @property
    def k_scales(self) -> torch.Tensor:
        self.ensure_allocated()
        return self._k_scales

    @property
    def v_scales(self) -> torch.Tensor:
        self.ensure_allocated()
        return self._v_scales

    def layer(self, layer_id: int) -> QuantPagedKV:
        return QuantPagedKV(self.k_cache[layer_id], self.v_cache[layer_id], self.k_scales[layer_id],
                            self.v_scales[layer_id])

    def _row(self, *values: int) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32).to(self.device, non_blocking=True)

    def write_kv_to_blocks(self, layer_id: int, block_ids: List[int], K: torch.Tensor, V: torch.Tensor):
        """K, V [h_kv, seq, d] -> pages ``block_ids`` in order, quantised."""
        _refuse_capture("q8_pool", self.device)
        n = min(int(K.shape[1]), len(block_ids) * self.B)
        if n == 0:
            return
        K, V = K.to(self.device)[:, :n], V.to(self.device)[:, :n]
        quantize_append(self.layer(layer_id), K.transpose(0, 1), V.transpose(0, 1), self._ids_tensor(block_ids)[None],
                        self._row(n), cu_seqlens_q=self._row(0, n))

    def write_one_token(self, layer_id: int, block_id: int, pos_in_block: int, k_tok: torch.Tensor,
                        v_tok: torch.Tensor):
        _refuse_capture("q8_pool", self.device)
        if not (0 <= int(block_id) < self.N_total and 0 <= int(pos_in_block) < self.B):
            raise RuntimeError(f"q8_pool_shape_unsupported:slot_{block_id}_{pos_in_block}")
        quantize_append(self.layer(layer_id), k_tok.to(self.device).transpose(0, 1),
                        v_tok.to(self.device).transpose(0, 1), self._row(int(block_id))[None],
                        self._row(int(pos_in_block) + 1))

    def read_kv_from_blocks(self, layer_id: int, block_ids: List[int], seq_len: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Pages -> K, V [h_kv, seq_len, d] of ``out_dtype``."""
        _refuse_capture("q8_pool", self.device)
        n = max(0, min(int(seq_len), len(block_ids) * self.B))
        K = torch.empty(self.num_kv_heads, n, self.head_dim, dtype=self.out_dtype, device=self.device)
        V = torch.empty_like(K)
        if n:
            dequantize_pages(self.layer(layer_id), self._ids_tensor(block_ids)[None], self._row(0, n), n,
                             out=(K.transpose(0, 1), V.transpose(0, 1)))
        return K, V
