"""Paged attention on values at the ends of their types: what a token does not see
does not reach it, and what it sees does."""

import pytest
import torch
from test_paged_gpu import BF16, I8, _cache, _cu, _ok, _pages, _rows64

pytestmark = pytest.mark.gpu


def _attend(cuda, c, table, qs, kv, q):
    out = c.attend(q.to(cuda), _cu(qs).to(cuda), torch.tensor(kv, dtype=torch.int32, device=cuda), table.to(cuda),
                   max(qs), max(kv))
    torch.cuda.synchronize()
    _ok()
    return out.double().cpu()


@pytest.mark.parametrize("qs,kv", [([3], [40]), ([120], [130]), ([600], [700]), ([200, 1], [3000, 9])])
def test_hidden_values_weigh_nothing_however_large(cuda, qs, kv):
    """The last new token's value is near bf16's largest: the tokens before it are those of any other value, bit
    for bit."""
    hq, hk, d, page = 4, 1, 128, 16
    table, n = _pages(kv, page, 3)
    c = _cache(cuda, n, page, hk, d, BF16, 3)
    q = torch.randn((sum(qs), hq * d), generator=torch.Generator().manual_seed(2)).to(BF16)
    want = _attend(cuda, c, table, qs, kv, q)
    at = kv[0] - 1
    c.value_pages[int(table[0, at // page]), :, at % page] = 3e38
    got = _attend(cuda, c, table, qs, kv, q)
    assert torch.equal(got[:qs[0] - 1], want[:qs[0] - 1]) and torch.equal(got[qs[0]:], want[qs[0]:])
    assert not torch.equal(got[qs[0] - 1], want[qs[0] - 1])


@pytest.mark.parametrize("qs,kv", [([3], [40]), ([120], [130]), ([100], [3000])])
def test_a_key_scale_of_nan_reaches_all_that_see_it_and_no_other(cuda, qs, kv):
    """What append leaves of a key with an infinity in an int8 cache, at every place of a step."""
    hq, hk, d, page = 4, 1, 64, 16
    table, n = _pages(kv, page, 3)
    q = torch.randn((sum(qs), hq * d), generator=torch.Generator().manual_seed(2)).to(BF16)
    plain = _attend(cuda, _cache(cuda, n, page, hk, d, I8, 3), table, qs, kv, q)
    past = kv[0] - qs[0]
    for at in (past, *(past + 1 + i for i in range(0, min(9, qs[0] - 1)))):
        c = _cache(cuda, n, page, hk, d, I8, 3)
        c.key_scale[int(table[0, at // page]), :, at % page] = float("nan")
        got = _attend(cuda, c, table, qs, kv, q)
        assert bool(got[at - past:].isnan().all())
        assert torch.equal(got[:at - past], plain[:at - past])


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("qs,kv", [([1], [40]), ([1], [5000]), ([6], [40]), ([120], [130]), ([60], [3000]), ([20, 1], [16, 3])])
def test_a_query_of_nan_gives_nan_and_one_without_keys_zeros(cuda, qs, kv, dtype):
    hq, hk, d, page = 4, 1, 128, 16
    table, n = _pages(kv, page, 3)
    c = _cache(cuda, n, page, hk, d, dtype, 3)
    q = torch.randn((sum(qs), hq * d), generator=torch.Generator().manual_seed(2)).to(BF16)
    want = _attend(cuda, c, table, qs, kv, q).view(-1, hq, d)
    blind = max(0, qs[0] - kv[0])  # tokens before the first key
    assert bool((want[:blind] == 0).all()) and bool((want[blind:qs[0]] != 0).any())
    for tok in sorted({0, blind, qs[0] - 1}):
        bad = q.clone()
        bad[tok, d + 5] = float("nan")  # head 1
        got = _attend(cuda, c, table, qs, kv, bad).view(-1, hq, d)
        assert bool((got[tok, 1] == 0).all() if tok < blind else got[tok, 1].isnan().all())
        got[tok, 1] = want[tok, 1]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("heads", [(4, 2), (64, 1)])
@pytest.mark.parametrize("b", [2, 40, 200])
def test_a_negative_length_is_reported_where_all_sequences_are_long(cuda, b, heads, dtype):
    """Offsets that go back, with bounds that leave no short sequence: the chunk kernel's alone to find."""
    from bitnet_tt import _lib

    hq, hk = heads
    c = _cache(cuda, b, 64, hk, 64, dtype, 1)
    table = torch.arange(b, dtype=torch.int32, device=cuda).view(b, 1)
    lens = torch.full((b,), 40, dtype=torch.int32, device=cuda)
    q = torch.zeros((40 * b, hq * 64), dtype=BF16, device=cuda)
    cu = [40 * i for i in range(b)] + [40 * (b - 1) - 20]
    for max_kv in (40, 0):
        c.attend(q, torch.tensor(cu, dtype=torch.int32, device=cuda), lens if max_kv else lens * 0, table, 40, max_kv)
        torch.cuda.synchronize()
        assert _lib.last_device_status() == (-1, 350)
        _ok()
