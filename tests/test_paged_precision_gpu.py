"""The precision that paged attention holds, by a sequence's own rows (new tokens x
query heads of a KV head), alone and among others, against the softmax in 64 bits.

Values of alternating sign cancel, so that an output is small beside A = sum_j p_j |v_j|
and errors of the weights show next to its own rounding.  The bound, with
S = max sum |q k| scale:
  * a score is a sum of D fp32 products times a factor, off by at most (D + 3) 2^-24 S; the
    weight and the sum of weights each by that share: 2 (D + 3) 2^-24 S;
  * exp2 (2 units in the last place, 2^-22), fp32 sums of at most 2^10 weights (a tree or
    256 at a time: below 2^-15), two joins: together below 2^-14;
  * the weight's own rounding, W: up to 32 rows 2^-16 as a bf16 pair, 2^-11 as f16 (int8, no
    longer sequence in the call); more rows 2^-8 as one bf16 and 7.5e-5 for the polynomial
    exponential, or, int8, three f16 roundings (the weight, the scale, code * scale),
    3 2^-11, and the polynomial;
  * f16 (int8) has a smallest step: 2^-32 of the largest p_j vs_j and code (up to 32 rows),
    2^-32 of the largest weight and value (more), summed over the keys;
  * the output's rounding, 2^-8 |o|."""

import pytest
import torch
from test_paged_gpu import BF16, I8, _cache, _cu, _ok, _pages, _rows64, _scales

pytestmark = pytest.mark.gpu


def _check(cuda, qs, kv, hq, hk, d, page, dtype, seed=0, sharp=0.1, scales=None, spread=0, lift=0, max_q=None, extra=0):
    """scales(g, shape): value scales of an int8 cache.  spread: queries' elements span 2^spread.  lift: queries are
    2^lift times what they are, and the scale 2^-lift."""
    g = torch.Generator().manual_seed(seed)
    table, n = _pages(kv, page, seed)
    c = _cache(cuda, n, page, hk, d, dtype, seed)
    sign = 1.0 - 2.0 * (torch.arange(page) % 2)
    u = 0.5 + torch.rand((n, hk, 1, d), generator=g)
    if dtype == BF16:
        c.value_pages.copy_((u * sign[:, None]).expand(n, hk, page, d))
    else:
        c.value_pages.copy_((u * 80 * sign[:, None]).round().expand(n, hk, page, d))
        if scales is not None:
            c.value_scale.copy_(scales(g, tuple(c.value_scale.shape)))
    cu = _cu(qs)
    toks = int(cu[-1]) + extra
    q = torch.randn((toks, hq * d), generator=g) * sharp
    if spread:
        q = q * 2.0 ** (-spread * torch.rand(q.shape, generator=g))
    q = q.to(BF16)
    out = c.attend((q.float() * 2.0 ** lift).to(BF16).to(cuda), cu.to(cuda), torch.tensor(kv, dtype=torch.int32).to(cuda),
                   table.to(cuda), max_q or max(qs), max(kv), d ** -0.5 * 2.0 ** -lift)
    torch.cuda.synchronize()
    _ok()
    got = out.double().cpu().view(toks, hq, d)
    grp = hq // hk
    for b, (m, k) in enumerate(zip(qs, kv)):
        if m == 0:
            continue
        kk, vv = _rows64(c, table, b, k)
        small = (m if dtype == BF16 else max(qs)) * grp <= 32
        weight = (2.0 ** -16 if dtype == BF16 else 2.0 ** -11) if small else \
            (2.0 ** -8 if dtype == BF16 else 3 * 2.0 ** -11) + 7.5e-5
        see = torch.arange(k)[None] < (k - m + torch.arange(m)[:, None] + 1)
        for h in range(hq):
            qq = q[int(cu[b]):int(cu[b + 1]), h * d:(h + 1) * d].double()
            s = (qq @ kk[:, h // grp].T * d ** -0.5).masked_fill(~see, -float("inf"))
            size = float((qq.abs() @ kk[:, h // grp].abs().T).max()) * d ** -0.5
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            p = p / p.sum(-1, keepdim=True)
            v = vv[:, h // grp]
            want, spread = p @ v, p @ v.abs()
            room = want.abs() * 2.0 ** -8 + (2 * (d + 3) * 2.0 ** -24 * size + 2.0 ** -14 + weight) * spread
            if dtype == I8:
                vs = _scales(c, table, b, k)[:, h // grp, None]
                if small:
                    codes = torch.where(vs > 0, v.abs() / vs.clamp(min=1e-300), torch.zeros_like(v)).sum(0)
                    room = room + 2.0 ** -32 * (p * vs[:, 0]).amax(-1, keepdim=True) * codes
                else:
                    room = room + 2.0 ** -32 * (p.amax(-1, keepdim=True) * v.abs().sum(0) + 128 * float(vs.max()))
            worst = float(((got[int(cu[b]):int(cu[b + 1]), h] - want).abs() - room).max())
            assert worst <= 0, f"sequence {b} ({m} tokens of {grp} rows) head {h}: {worst} over the bound"


BATCHES = [([1], [6]), ([5], [9]), ([8], [21]), ([1, 40, 40], [6, 41, 45]), ([40, 2, 0, 39], [40, 7, 9, 60]),
           ([5, 40, 8, 40, 40], [5, 40, 11, 90, 40]), ([300, 3], [333, 4])]


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 2, 64), (10, 2, 128), (12, 1, 64), (17, 1, 128)])
@pytest.mark.parametrize("qs,kv", BATCHES)
def test_a_sequences_precision_is_its_own(cuda, qs, kv, heads, dtype):
    """The same few rows alone, and among chunks that fill the batch."""
    _check(cuda, qs, kv, *heads, 16, dtype, seed=len(qs))


@pytest.mark.parametrize("dtype", [BF16, I8])
def test_precision_with_rows_behind_the_last_sequence(cuda, dtype):
    # as many rows as if every sequence had max_seqlen tokens
    _check(cuda, [40, 1], [44, 7], 8, 2, 128, 16, dtype, seed=3, extra=39)


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("qs,kv", [([3, 1], [900, 700]), ([60, 2, 1], [1000, 900, 5])])
def test_precision_over_split_contexts(cuda, qs, kv, dtype):
    _check(cuda, qs, kv, 4, 1, 128, 32, dtype, seed=7)


RANGES = [([1, 1], [90, 700]), ([6], [300]), ([60], [100]), ([100, 2], [600, 33])]


@pytest.mark.parametrize("spread", [10, 30, 60])
@pytest.mark.parametrize("qs,kv", RANGES)
def test_value_scales_of_any_spread(cuda, qs, kv, spread):
    """Scales from 1 down to 2^-spread, rows without any scale among them (a scale of 0)."""
    def scales(g, shape):
        s = 2.0 ** (-spread * torch.rand(shape, generator=g))
        return s * (torch.rand(shape, generator=g) > 0.1)

    _check(cuda, qs, kv, 4, 1, 128, 16, I8, seed=spread, scales=scales)


@pytest.mark.parametrize("qs,kv", RANGES)
def test_small_values_behind_a_large_one_that_is_not_seen(cuda, qs, kv):
    """The last key's value scale is 2^18 times the others': the tokens before it keep their own precision."""
    def scales(g, shape):
        return torch.full(shape, 2.0 ** -20)

    def with_last(g, shape):
        s = scales(g, shape)
        table, _ = _pages(kv, 16, 5)
        for b, k in enumerate(kv):
            s[int(table[b, (k - 1) // 16]), :, (k - 1) % 16] = 2.0 ** -2
        return s

    _check(cuda, qs, kv, 4, 1, 64, 16, I8, seed=5, scales=with_last)


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("qs,kv", RANGES)
def test_queries_of_any_spread_and_size(cuda, qs, kv, dtype):
    _check(cuda, qs, kv, 4, 1, 128, 16, dtype, seed=8, sharp=0.5, spread=27)
    for lift in (-60, 60):
        _check(cuda, qs, kv, 4, 1, 64, 16, dtype, seed=9, lift=lift)
