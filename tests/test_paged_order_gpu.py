"""What one launch of a paged call may read of another's: chains of append and
attend over buffers that are rewritten in place before every call."""

import pytest
import torch
from test_paged_gpu import BF16, I8, _cache, _cu, _ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_mixed_calls_read_what_was_just_written(cuda, dtype, captured):
    """Chunks beside single tokens: the small rows' kernel runs beside the chunks' and does not wait for it, so
    offsets, lengths, table, queries and scales have to be the ones that the launches before both wrote.  Two
    groups of sequences take turns in the same buffers; the same calls one at a time, without dependent launch,
    give the bits."""
    from bitnet_tt import _lib

    hq, hk, d, page, rounds = 8, 2, 128, 16, 12
    qs = [[40] + [1] * 23, [1] * 12 + [37] + [1] * 11]
    kv0 = [[300 + (53 * i + 17 * g) % 400 for i in range(24)] for g in range(2)]
    width = -(-(720 + 41 * rounds) // page)
    order = torch.randperm(48 * width, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    tables = [order[:24 * width].view(24, width).to(cuda), order[24 * width:].view(24, width).to(cuda)]
    caches = [_cache(cuda, 48 * width, page, hk, d, dtype, 2) for _ in range(2)]
    cus = [_cu(q).to(cuda) for q in qs]
    toks = [sum(q) for q in qs]
    most = max(toks)
    one, zero = torch.ones((width * page, d // 2), device=cuda), torch.zeros((width * page, d // 2), device=cuda)
    gen = torch.Generator().manual_seed(4)
    rows = [torch.randn((most, (hq + 2 * hk) * d), generator=gen).to(BF16).to(cuda) for _ in range(rounds)]
    lens = []
    for r in range(rounds):
        g = r % 2
        lens.append(torch.tensor([k + (r // 2 + 1) * n for k, n in zip(kv0[g], qs[g])], dtype=torch.int32, device=cuda))
    qkv = torch.zeros_like(rows[0])
    cu, kv, table = torch.zeros_like(cus[0]), torch.zeros_like(lens[0]), torch.zeros_like(tables[0])
    q = torch.zeros((most, hq * d), dtype=BF16, device=cuda)
    outs = [torch.zeros((rounds, most, hq * d), dtype=BF16, device=cuda) for _ in range(2)]

    def chain(c, out, pause):
        for r in range(rounds):
            g = r % 2
            qkv.copy_(rows[r]), cu.copy_(cus[g]), kv.copy_(lens[r]), table.copy_(tables[g])
            pause()
            c.append(qkv[:toks[g]], cu, kv, table, one, zero, q[:toks[g]])
            pause()
            c.attend(q[:toks[g]], cu, kv, table, max(qs[g]), width * page, out=out[r, :toks[g]])
            pause()

    _lib.set_pdl(False)
    try:
        chain(caches[0], outs[0], torch.cuda.synchronize)
    finally:
        _lib.set_pdl(True)
    if captured:
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            chain(caches[1], outs[1], lambda: None)
        torch.cuda.synchronize()
        g.replay()
    else:
        chain(caches[1], outs[1], lambda: None)
    torch.cuda.synchronize()
    _ok()
    assert torch.equal(caches[0].key_pages, caches[1].key_pages)
    assert torch.equal(caches[0].value_pages, caches[1].value_pages)
    for r in range(rounds):
        assert torch.equal(outs[0][r], outs[1][r]), f"call {r}"
