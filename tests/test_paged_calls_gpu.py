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
