"""Linear's activation buffers: a call's own, given back when it returns, so
that calls on two streams do not write each other's and token counts that vary
keep no memory."""

import gc
import weakref

import pytest
import torch

BF16 = torch.bfloat16


def test_calls_share_and_keep_no_buffers(monkeypatch):
    from bitnet_tt import _lib
    from bitnet_tt.layers import Linear

    seen = []

    def entry(x, gamma, eps, bufs, *rest, **kw):
        seen.append(weakref.ref(bufs))

    monkeypatch.setattr(_lib, "act_quant", entry)
    monkeypatch.setattr(_lib, "bitlinear_fused", entry)
    monkeypatch.setattr(_lib, "bitlinear_q", lambda *a, **kw: None)
    lin = Linear(64, 64, "cpu")
    lin.weight = torch.zeros(1, dtype=torch.uint8)
    for m in (*range(1, 20), 5, 5):
        assert lin(torch.zeros((m, 64), dtype=BF16)).shape == (m, 64)
    gc.collect()
    assert len(seen) == 21 and all(r() is None for r in seen)


def _linear(cuda, k, n, seed):
    from bitnet_tt.layers import Linear

    lin = Linear(k, n, cuda)
    g = torch.Generator().manual_seed(seed)
    lin.load_ternary(torch.randint(-1, 2, (n, k), generator=g).to(torch.int8), 0.02)
    return lin


@pytest.mark.gpu
def test_two_streams_with_equal_shapes(cuda):
    lins = [_linear(cuda, 2560, 2560, i) for i in range(2)]
    m = 300
    xs = [torch.randn((m, 2560), generator=torch.Generator().manual_seed(i)).to(BF16).to(cuda) for i in range(2)]
    want = [lin(x) for lin, x in zip(lins, xs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(lins[i](xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.gpu
def test_many_token_counts_keep_no_memory(cuda):
    lin = _linear(cuda, 2560, 640, 3)
    x = torch.randn((2000, 2560), generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda)
    lin(x[:10])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(cuda)
    for m in range(100, 2000, 100):
        lin(x[:m])
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(cuda) == before


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [1, 0, 2563, 2560])
def test_one_row_of_any_stride(cuda, stride):
    """A row that torch counts as contiguous whatever its stride: a slice of wider rows, a transposed column."""
    lin = _linear(cuda, 2560, 640, 4)
    x = torch.randn((1, 2560), generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    assert torch.equal(lin(x.as_strided((1, 2560), (stride, 1))), lin(x.clone()))


def test_rows_that_are_apart_are_refused_where_they_cannot_be():
    from bitnet_tt import _lib

    for x in (torch.zeros((3, 80), dtype=BF16)[:, :64], torch.zeros((64, 3), dtype=BF16).t(), torch.zeros((3, 64))):
        with pytest.raises(ValueError, match="contiguous"):
            _lib.bitlinear_fused(x, None, 1e-5, None, None, 64, None, 0, None, None)
