"""The paged cache's calls as Python sees them: what they hold, take and give back."""

import pytest
import torch
from test_paged_gpu import BF16, I8, _cache, _cu, _ok, _pages

pytestmark = pytest.mark.gpu


def test_a_read_whose_second_output_does_not_fit_keeps_nothing(cuda):
    c = _cache(cuda, 4, 16, 2, 64, BF16, 1)
    table, _ = _pages([16], 16)
    table, cu = table.to(cuda), _cu([0]).to(cuda)
    rows = 1 << 19  # 128 MiB an output
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held, used = torch.cuda.memory_allocated(cuda), torch.cuda.memory_reserved(cuda)
    total = torch.cuda.get_device_properties(cuda).total_memory
    torch.cuda.set_per_process_memory_fraction((used + (200 << 20)) / total, cuda)
    try:
        for _ in range(3):
            with pytest.raises(torch.OutOfMemoryError):
                c.read(table, None, cu, rows)
            assert torch.cuda.memory_allocated(cuda) == held
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, cuda)
    k, v = c.read(table, None, _cu([16]).to(cuda), 16)
    assert k.shape == v.shape == (16, 2, 64)
    _ok()


@pytest.mark.parametrize("stride", [1, 0, 515, 1 << 33])
def test_one_row_may_have_any_stride(cuda, stride):
    c = _cache(cuda, 2, 16, 2, 64, BF16, 1)
    table, cu = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda), _cu([1]).to(cuda)
    lens = torch.tensor([20], dtype=torch.int32, device=cuda)
    one, zero = torch.ones((32, 32), device=cuda), torch.zeros((32, 32), device=cuda)
    qkv = torch.randn((1, 8 * 64), generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda)
    want = c.append(qkv, cu, lens, table, one, zero)
    assert torch.equal(want, c.append(qkv.as_strided((1, 8 * 64), (stride, 1)), cu, lens, table, one, zero))
    o = c.attend(want, cu, lens, table, 1, 20)
    assert torch.equal(o, c.attend(want.as_strided((1, 4 * 64), (stride, 1)), cu, lens, table, 1, 20))
    none = c.attend(want[:0].as_strided((0, 4 * 64), (stride, 1)), _cu([0]).to(cuda), lens, table, 1, 20)
    assert none.shape == (0, 4 * 64)
    _ok()
