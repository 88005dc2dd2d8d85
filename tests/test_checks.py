"""CPU tests of the tensor checks the entry points share."""
import torch

from tilelang_fa_v100._checks import rows_ready


def test_rows_ready_moves_a_contiguous_tensor_at_an_odd_address():
    base = torch.arange(65, dtype=torch.float16)
    odd = base[1:].view(4, 16)
    assert odd.is_contiguous() and odd.data_ptr() % 16 != 0
    got = rows_ready(odd)
    assert got.data_ptr() % 16 == 0 and got.is_contiguous() and torch.equal(got, odd)
    even = base[:64].view(4, 16)
    assert rows_ready(even) is even
