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


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("qs,kv", [([1], [5000]), ([2, 3], [3000, 40]), ([64, 1, 1], [3000, 2000, 5])])
def test_a_workspace_of_ones_own(cuda, qs, kv, dtype):
    """attention_workspace() sizes it, whatever it holds before; captured calls that share one in a row replay right."""
    table, n = _pages(kv, 64)
    c = _cache(cuda, n, 64, 2, 128, dtype, 3)
    cu, lens, table = _cu(qs).to(cuda), torch.tensor(kv, dtype=torch.int32, device=cuda), table.to(cuda)
    q = torch.randn((sum(qs), 8 * 128), generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda)
    want = c.attend(q, cu, lens, table, max(qs), max(kv))
    ws = c.attention_workspace(len(qs), sum(qs), max(qs), max(kv), 8)
    assert ws is not None
    ws.fill_(255)
    assert torch.equal(c.attend(q, cu, lens, table, max(qs), max(kv), workspace=ws), want)
    with pytest.raises(RuntimeError, match="invalid argument"):
        c.attend(q, cu, lens, table, max(qs), max(kv), workspace=ws[:-1])
    outs = [torch.zeros_like(q) for _ in range(2)]
    graphs = []
    for o in outs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            c.attend(q, cu, lens, table, max(qs), max(kv), out=o, workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    _ok()
