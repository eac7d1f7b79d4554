"""CPU tests of how the 8-bit cache's Python side takes its arguments."""
import pytest
import torch

from unifiedkv_b200 import kv_quant


def test_64_bit_numbers_do_not_wrap():
    ids = torch.tensor([[0, 2 ** 32 + 1, -2 ** 32, 2 ** 31, -1]])
    got = kv_quant._table(ids, "x")
    assert got.dtype == torch.int32 and got[0, 0] == 0 and got[0, 1] == 2 ** 31 - 1 == got[0, 3]
    assert got[0, 2] < 0 and got[0, 4] == -1
    got = kv_quant._int32(torch.tensor([2 ** 32 + 1, 5]), "x", "seqlens", 2)
    assert got.tolist() == [2 ** 31 - 1, 5]
    same = torch.tensor([1, 2], dtype=torch.int32)
    assert kv_quant._int32(same, "x", "seqlens", 2) is same
    assert kv_quant._int32(torch.tensor([1, 2], dtype=torch.int16), "x", "seqlens", 2).tolist() == [1, 2]


def test_numbers_of_the_host_are_refused_in_a_capture(monkeypatch):
    import contextlib
    kv_quant._refuse_capture("x", torch.device("cpu"))
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    kv_quant._refuse_capture("x", torch.device("cuda:0"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="^x_unavailable:host_numbers_in_capture$"):
        kv_quant._refuse_capture("x", torch.device("cuda:0"))


@pytest.mark.parametrize("failing", [1, 2, 3, 4])
def test_pool_allocates_again_after_running_out_of_memory(monkeypatch, failing):
    """Whichever of the four tensors did not fit, the next access allocates the pool anew."""
    pool = kv_quant.QuantPagedKVPool(16, 2, 2, 64, device="cpu", n_total=3)
    made = [0]

    def once(fn):
        def make(*args, **kw):
            made[0] += 1
            if made[0] == failing:
                raise torch.OutOfMemoryError("no room")
            return fn(*args, **kw)
        return make
    monkeypatch.setattr(torch, "zeros", once(torch.zeros))
    monkeypatch.setattr(torch, "zeros_like", once(torch.zeros_like))
    with pytest.raises(torch.OutOfMemoryError):
        pool.layer(0)
    assert not pool.is_allocated
    kv = pool.layer(1)
    assert [tuple(x.shape) for x in kv] == [(3, 16, 2, 64)] * 2 + [(3, 2, 16)] * 2


def test_readback_refuses_outputs_that_overlap():
    codes, scales = torch.zeros(3, 16, 2, 64, dtype=torch.float8_e4m3fn), torch.zeros(3, 2, 16, dtype=torch.uint8)
    kv = kv_quant.QuantPagedKV(codes, codes.clone(), scales, scales.clone())
    bt, cu = torch.zeros(1, 3, dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32)
    x, y = torch.zeros(4, 2, 64), torch.zeros(4, 2, 64)
    for out in ((x, x), (x[:1].expand(4, 2, 64), y[:1].expand(4, 2, 64)), (x[:, :1].expand(4, 2, 64), y[:, :1].expand(4, 2, 64))):
        with pytest.raises(RuntimeError, match="^q8_dequantize_shape_unsupported:out_overlap$"):
            kv_quant.dequantize_pages(kv, bt, cu, 4, out=out)
    both = torch.zeros(4, 2, 2, 64)  # K and V side by side are two places
    with pytest.raises(RuntimeError, match="tensors_not_on_cuda"):
        kv_quant.dequantize_pages(kv, bt, cu, 4, out=(both[:, 0], both[:, 1]))


def test_a_token_outside_its_page_is_refused():
    """It would be skipped in silence: the 16-bit pool raises, too."""
    pool = kv_quant.QuantPagedKVPool(16, 1, 2, 64, device="cpu", n_total=3)
    x = torch.zeros(2, 1, 64)
    for block, pos in ((0, 16), (0, -1), (3, 0), (-1, 0)):
        with pytest.raises(RuntimeError, match=f"^q8_pool_shape_unsupported:slot_{block}_{pos}$"):
            pool.write_one_token(0, block, pos, x, x)
    with pytest.raises(RuntimeError, match="tensors_not_on_cuda"):
        pool.write_one_token(0, 2, 15, x, x)
