"""PagedGenerator's use of its pages, on a model that only counts: the next token
follows from the last one and its position."""

import contextlib

import pytest
import torch

VOCAB = 97


class _Model:
    device = torch.device("cpu")

    class config:
        max_position_embeddings = 256
        head_dim = 64
        rope_theta = 1e4
        vocab_size = VOCAB

    def __init__(self):
        self.rows = {}  # (page, row) -> token
        self.batches = []

    def paged_caches(self, num_pages, page_size, dtype):
        self.page_size = page_size
        return []

    def forward_paged(self, ids, batch, rope, caches, keep_logits):
        cu, kv, table = batch.cu_seqlens.tolist(), batch.kv_lens.tolist(), batch.block_table.tolist()
        assert len(set(p for row in table for p in row if p >= 0)) == sum(p >= 0 for row in table for p in row)
        out = []
        for b, n in enumerate(kv):
            new = ids[cu[b]:cu[b + 1]].tolist()
            for i, t in enumerate(new):
                pos = n - len(new) + i
                self.rows[table[b][pos // self.page_size], pos % self.page_size] = t
            out.append(_next([self.rows[table[b][p // self.page_size], p % self.page_size] for p in range(n)]))
        self.batches.append(len(kv))
        return torch.tensor(out, dtype=torch.int32), None


def _next(tokens):
    return (sum((i + 1) * t for i, t in enumerate(tokens)) + len(tokens)) % VOCAB


def _alone(prompt, n):
    tokens = list(prompt)
    for _ in range(n):
        tokens.append(_next(tokens))
    return tokens[len(prompt):]


@pytest.fixture
def make(monkeypatch):
    from bitnet_tt.inference import PagedGenerator

    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return lambda pages, **kw: PagedGenerator(_Model(), pages, 16, **kw)


def _prompt(n, seed=0):
    return [(7 * i + seed) % VOCAB for i in range(n)]


@pytest.mark.parametrize("chunk", [8192, 13])
@pytest.mark.parametrize("lens,new", [([64, 64], 5), ([60, 60, 20], 10), ([100, 3, 90, 1, 64], 20), ([17] * 9, 40), ([128], 1)])
def test_a_batch_may_be_larger_than_the_pool(make, lens, new, chunk):
    gen = make(8, chunk_tokens=chunk)
    prompts = [_prompt(n, i) for i, n in enumerate(lens)]
    assert gen.generate(prompts, new) == [_alone(p, new) for p in prompts]
    assert sorted(gen.free_pages) == list(range(8)) and not gen.sequences


def test_prompts_that_fit_together_are_read_together(make):
    gen = make(12)
    gen.generate([_prompt(20), _prompt(40), _prompt(60)], 10)
    assert gen.model.batches == [3] * 10


@pytest.mark.parametrize("chunk", [8192, 5])
def test_generate_leaves_other_sequences_alone(make, chunk):
    gen = make(8, chunk_tokens=chunk)
    a, b = gen.add(_prompt(20)), gen.add(_prompt(30, 1))
    gen.step()
    held = {i: (list(s.pages), s.length, list(s.pending), list(s.generated)) for i, s in gen.sequences.items()}
    prompts = [_prompt(40, 2), _prompt(30, 3)]
    assert gen.generate(prompts, 6) == [_alone(p, 6) for p in prompts]
    assert held == {i: (s.pages, s.length, s.pending, s.generated) for i, s in gen.sequences.items()}
    told = {a: gen.sequences[a].generated, b: gen.sequences[b].generated}
    for _ in range(12):
        gen.step()
    assert told[a] == _alone(_prompt(20), len(told[a])) and told[b] == _alone(_prompt(30, 1), len(told[b]))


def test_a_prompt_beyond_the_pool_is_refused_before_anything_runs(make):
    gen = make(4)
    for prompts, new in (([_prompt(5), _prompt(65)], 1), ([_prompt(60)], 6)):
        with pytest.raises(ValueError, match="pages"):
            gen.generate(prompts, new)
    gen.add(_prompt(20))
    gen.step()  # two pages
    with pytest.raises(ValueError, match="2 free pages"):
        gen.generate([_prompt(33)], 1)
    assert gen.model.batches == [1] and len(gen.sequences) == 1


def test_prompts_being_read_leave_decoding_sequences_their_next_page(make):
    gen = make(8, chunk_tokens=40)
    one = gen.add(_prompt(15))
    gen.step()
    two = gen.add(_prompt(130, 1))  # more than the pool
    for _ in range(20):  # beyond two page boundaries
        assert one in gen.step()
    assert gen.sequences[one].generated == _alone(_prompt(15), 21)
    assert gen.sequences[two].length == 0
    gen.release(one)
    gen.step()
    assert gen.sequences[two].length == 40


def test_prompts_begun_together_can_be_read_to_their_end(make):
    gen = make(8, chunk_tokens=48)
    a, b = gen.add(_prompt(64)), gen.add(_prompt(80, 1))
    out = {}
    while a not in out:
        out |= gen.step()
    gen.release(a)
    while b not in out:
        out |= gen.step()
    assert out[a] == _alone(_prompt(64), 1)[0] and out[b] == _alone(_prompt(80, 1), 1)[0]


def test_a_pool_that_is_full_is_an_error_that_a_release_mends(make):
    gen = make(2)
    a, b = gen.add(_prompt(16)), gen.add(_prompt(16, 1))
    assert set(gen.step()) == {a, b}
    with pytest.raises(RuntimeError, match="no pages"):
        gen.step()
    gen.release(a)
    assert set(gen.step()) == {b}
    assert gen.sequences[b].generated == _alone(_prompt(16, 1), 2)
