"""Workloads of the paged KV cache: rotating and writing new tokens into it (in
bf16, or quantised to int8 as they are written), reading rows back, and the
attention of each sequence's new tokens over its pages.

Every case is one call as a serving loop makes it for one layer:

  append  qkv rows of the new tokens -> rotated queries, and the rotated keys
          and the values in the pages.  An int8 cache is read back afterwards
          (the rows just written), which is how its contents are seen.
  attend  queries of the new tokens over all keys of their sequences, causal
          from the end: token i of a chunk of n sees the first kv_len - n + i + 1.
  read    rows 0 .. kv_len - 1 of every sequence as packed bf16 (what moves a
          sequence to another pool, or to the contiguous cache).

The lengths of a case follow from its sizes alone; values follow from the seed.
`own` False computes the plain forms, True calls the framework.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"

# (query heads, KV heads, head dimension): the 2B-4T model, the mini model, and
# the group sizes 1, 8 and 4 of the attention tests.
HEADS = {"2b4t": (20, 5, 128), "mini": (4, 2, 64), "mha": (4, 4, 128), "wide": (16, 2, 128), "small": (16, 4, 64)}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one token of each of a batch's 32 sequences, the serving loop's smallest write
        {"name": "append 32x1 bf16", "op": "append", "heads": "2b4t", "B": 32, "q": 1, "q_mode": "all", "kv": 700,
         "page": 64, "kv_type": "bf16", "table": "bf16", "interleaved": False, "rot": 128},
        # a whole prompt pass of the benchmark's size: 32 prompts of 512 tokens
        {"name": "append 32x512 bf16", "op": "append", "heads": "2b4t", "B": 32, "q": 512, "q_mode": "all", "kv": 512,
         "page": 64, "kv_type": "bf16", "table": "bf16", "interleaved": False, "rot": 128},
        # ragged chunks into an int8 cache, and the same rows read back
        {"name": "append ragged int8", "op": "append", "heads": "2b4t", "B": 24, "q": 999, "q_mode": "ragged",
         "kv": 4000, "page": 32, "kv_type": "int8", "table": "f32", "interleaved": False, "rot": 128},
        # a checkpoint with adjacent pairs and half of each head rotated, mini model, odd sizes
        {"name": "append partial interleaved", "op": "append", "heads": "mini", "B": 7, "q": 77, "q_mode": "ragged",
         "kv": 500, "page": 16, "kv_type": "int8", "table": "f32", "interleaved": True, "rot": 32},
        # contexts of 16 sequences moved out of an int8 cache
        {"name": "read 16 ragged int8", "op": "read", "heads": "2b4t", "B": 16, "q": 0, "q_mode": "all", "kv": 4096,
         "page": 64, "kv_type": "int8"},
        # one short sequence of the mini model
        {"name": "read 1 short bf16", "op": "read", "heads": "mini", "B": 1, "q": 0, "q_mode": "all", "kv": 131,
         "page": 16, "kv_type": "bf16"},
        # a chat turn: one sequence, one token, latency only
        {"name": "decode 1x300", "op": "attend", "heads": "2b4t", "B": 1, "q": 1, "q_mode": "all", "kv": 300,
         "page": 64, "kv_type": "bf16"},
        # one sequence with a long context: the keys have to be split over the GPU
        {"name": "decode 1x131072", "op": "attend", "heads": "2b4t", "B": 1, "q": 1, "q_mode": "all", "kv": 131072,
         "page": 256, "kv_type": "bf16"},
        # 256 sequences at ragged contexts up to 4K, int8 cache (the benchmark's many-context decode)
        {"name": "decode 256 ragged int8", "op": "attend", "heads": "2b4t", "B": 256, "q": 1, "q_mode": "all",
         "kv": 4096, "page": 64, "kv_type": "int8"},
        # five drafted tokens of 16 sequences verified at once
        {"name": "verify 16x5", "op": "attend", "heads": "2b4t", "B": 16, "q": 5, "q_mode": "all", "kv": 2050,
         "page": 16, "kv_type": "bf16"},
        # chunks of prompts beside decoding sequences in one batch, int8 cache
        {"name": "mixed 48 int8", "op": "attend", "heads": "2b4t", "B": 48, "q": 1024, "q_mode": "mixed", "kv": 4096,
         "page": 64, "kv_type": "int8"},
        # the last 4096-token chunks of two long prompts
        {"name": "chunk 2x4096 of 16384", "op": "attend", "heads": "2b4t", "B": 2, "q": 4096, "q_mode": "all",
         "kv": 16384, "page": 128, "kv_type": "bf16"},
    ]


# The largest listed work: no drawn case does more.
_MOST_FLOPS, _MOST_BYTES, _MOST_SCORES = 6.8e11, 6.0e8, 2.6e9


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: any operator, any of the head layouts, page sizes and
    types; batch, chunk and context spread over their logarithms."""
    while True:
        op = rng.choice(["append", "append", "attend", "attend", "attend", "read"])
        heads = rng.choice(sorted(HEADS))
        d = HEADS[heads][2]
        c = {"op": op, "heads": heads, "B": _log(rng, 1, 256), "page": rng.choice([16, 32, 64, 128, 256]),
             "kv_type": rng.choice(["bf16", "int8"]), "kv": _log(rng, 1, 32768)}
        if op == "read":
            c |= {"q": 0, "q_mode": "all"}
        else:
            c |= {"q": _log(rng, 1, 4096) if rng.random() < 0.6 else rng.randint(1, 9),
                  "q_mode": rng.choice(["all", "ragged", "mixed"])}
            c["q"] = min(c["q"], c["kv"])
        if op == "append":
            c |= {"table": rng.choice(["bf16", "f32"]), "interleaved": rng.random() < 0.5,
                  "rot": rng.choice([d, d, d // 2])}
        w = work(c)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and _padded(c) <= _MOST_SCORES:
            return c


def _frac(i, a):
    return (i + 1) * a % 1.0


def _lens(c):
    """(new tokens, keys after them) of every sequence, from the sizes alone.
    Sequence 0 has the largest of both; contexts spread evenly below it."""
    qs, kvs = [], []
    for i in range(c["B"]):
        if c["q_mode"] == "all" or i == 0:
            q = c["q"]
        elif c["q_mode"] == "mixed":  # chunks of a prompt in every 16th slot, one token elsewhere
            q = c["q"] if i % 16 == 0 else 1
        else:  # ragged, with an idle slot now and then
            q = 0 if i % 7 == 3 else 1 + int((c["q"] - 1) * _frac(i, 0.41421356))
        kv = c["kv"] if i == 0 else 1 + int((c["kv"] - 1) * _frac(i, 0.61803399))
        qs.append(q)
        kvs.append(max(kv, q))
    return qs, kvs


def _padded(c):
    """Scores (attend) or gathered values (read) that the plain form holds at once."""
    hq, hk, d = HEADS[c["heads"]]
    return c["B"] * c["kv"] * (max(1, c["q"]) * hq if c["op"] == "attend" else 2 * hk * d)


def _row_bytes(c):
    """Bytes of one KV head's key (or value) row in the cache, scale included."""
    d = HEADS[c["heads"]][2]
    return 2 * d if c["kv_type"] == "bf16" else d + 4


def work(c):
    hq, hk, d = HEADS[c["heads"]]
    qs, kvs = _lens(c)
    toks, row = sum(qs), _row_bytes(c)
    pages = sum(-(-k // c["page"]) for k in kvs)
    idx = 4 * (2 * c["B"] + 1)  # offsets and lengths
    if c["op"] == "append":
        by = toks * (hq + 2 * hk) * d * 2 + toks * hq * d * 2 + 2 * toks * hk * row + idx + 4 * toks // c["page"]
        by += max(qs) * c["rot"] * (2 if c["table"] == "bf16" else 4)  # cos and sin of the positions, rot / 2 each
        if c["kv_type"] == "int8":
            by += 2 * toks * hk * (row + 2 * d)
        return {"bytes": by, "flops": 3 * toks * (hq + hk) * c["rot"] + (4 * toks * hk * d if c["kv_type"] == "int8" else 0)}
    if c["op"] == "read":
        return {"bytes": sum(kvs) * hk * 2 * (row + 2 * d) + idx + 4 * pages,
                "flops": sum(kvs) * hk * 2 * d if c["kv_type"] == "int8" else 0}
    seen = sum(q * k - q * (q - 1) // 2 for q, k in zip(qs, kvs))
    live = [k for q, k in zip(qs, kvs) if q]
    return {"bytes": 2 * toks * hq * d * 2 + sum(live) * hk * 2 * row + idx + 4 * pages, "flops": 4 * seen * hq * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(c, seed):
    hq, hk, d = HEADS[c["heads"]]
    g = torch.Generator(device=DEV).manual_seed(seed)
    qs, kvs = _lens(c)
    per = [-(-k // c["page"]) for k in kvs]
    npages = sum(per) + 3
    # pages in the order a long-running pool hands them out: none
    order = torch.randperm(npages, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.full((c["B"], max(per) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (npages, hk, c["page"], d)
    st = {"c": dict(c), "block_table": table.to(DEV),
          "cu": torch.tensor([0] + qs, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV),
          "kv_lens": torch.tensor(kvs, dtype=torch.int32, device=DEV),
          "max_q": max(qs), "max_kv": max(kvs), "tokens": sum(qs), "rows": sum(kvs), "ks": None, "vs": None}
    if c["kv_type"] == "bf16":
        st["k"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
        st["v"] = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    else:
        # rows quantised from normal values: the largest code is +-127, the scale about 3 / 127
        for n in ("k", "v"):
            x = torch.randn(shape, generator=g, device=DEV) * (0.5 + torch.rand(shape[:3], generator=g, device=DEV))[..., None]
            top = x.abs().amax(-1)
            st[n] = torch.round(x * (127.0 / top)[..., None]).to(torch.int8)
            st[n + "s"] = top / 127.0
    if c["op"] == "append":
        st["qkv"] = torch.randn((st["tokens"], (hq + 2 * hk) * d), generator=g, device=DEV).mul_(1.5).to(torch.bfloat16)
        pos = torch.arange(max(kvs), dtype=torch.float64, device=DEV)
        ang = pos[:, None] * 500000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=DEV) / c["rot"])
        dt = torch.bfloat16 if c["table"] == "bf16" else torch.float32
        st["cos"], st["sin"] = ang.cos().to(dt), ang.sin().to(dt)
        st["q"] = torch.zeros((st["tokens"], hq * d), dtype=torch.bfloat16, device=DEV)
        st["starts"] = st["kv_lens"] - (st["cu"][1:] - st["cu"][:-1])
    elif c["op"] == "attend":
        # queries with some spread of sharpness: a score's deviation is about 2
        st["q"] = torch.randn((st["tokens"], hq * d), generator=g, device=DEV).mul_(2.0).to(torch.bfloat16)
    else:
        st["starts"] = torch.zeros(c["B"], dtype=torch.int32, device=DEV)
        st["cu_rows"] = torch.tensor([0] + kvs, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEV)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    return _run_own(st) if own else _PLAIN[st["c"]["op"]](st)


def _run_own(st):
    c = st["c"]
    cache = st.get("cache")
    if cache is None:  # the handle that a program keeps beside its pages
        if "bitnet-tt_b200" not in (os.path.basename(p) for p in sys.path):
            sys.path.insert(0, os.path.join(os.getcwd(), "bitnet-tt_b200"))
        from bitnet_tt.layers import PagedKVCache

        cache = st["cache"] = PagedKVCache.from_tensors(st["k"], st["v"], st["ks"], st["vs"])
    if c["op"] == "append":
        cache.append(st["qkv"], st["cu"], st["kv_lens"], st["block_table"], st["cos"], st["sin"], st["q"],
                     interleaved=c["interleaved"])
        if c["kv_type"] == "bf16":
            return {"q": st["q"], "k": st["k"], "v": st["v"]}
        k, v = cache.read(st["block_table"], st["starts"], st["cu"], st["tokens"])
        return {"q": st["q"], "k": k, "v": v}
    if c["op"] == "attend":
        return cache.attend(st["q"], st["cu"], st["kv_lens"], st["block_table"], st["max_q"], st["max_kv"])
    k, v = cache.read(st["block_table"], st["starts"], st["cu_rows"], st["rows"])
    return {"k": k, "v": v}


def _spread(cu, n):
    """(sequence, place in it) of each of n packed rows."""
    r = torch.arange(n, device=DEV)
    b = torch.searchsorted(cu[1:].long(), r, right=True)
    return b, r - cu.long()[b]


def _slots(st, b, pos):
    """(page, row in the page) of position pos of sequence b."""
    page = st["c"]["page"]
    return st["block_table"].long()[b, pos // page], pos % page


def _rotated(st, x, pos):
    """The first `rot` dimensions of x [tokens, heads, d] (32 bits) turned by the angles of pos."""
    c = st["c"]
    rot = c["rot"]
    cos, sin = st["cos"].float()[pos][:, None], st["sin"].float()[pos][:, None]
    t = x[..., :rot]
    a, b = (t[..., 0::2], t[..., 1::2]) if c["interleaved"] else (t[..., : rot // 2], t[..., rot // 2:])
    ra, rb = a * cos - b * sin, b * cos + a * sin
    t = torch.stack([ra, rb], -1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], -1)
    return torch.cat([t, x[..., rot:]], -1)


def _plain_append(st):
    hq, hk, d = HEADS[st["c"]["heads"]]
    b, i = _spread(st["cu"], st["tokens"])
    pos = st["starts"].long()[b] + i
    x = st["qkv"].view(st["tokens"], hq + 2 * hk, d).float()
    qk = _rotated(st, x[:, : hq + hk], pos)
    st["q"].copy_(qk[:, :hq].reshape(st["tokens"], hq * d))
    page, slot = _slots(st, b, pos)
    for n, rows in (("k", qk[:, hq:]), ("v", x[:, hq + hk:])):
        if st["c"]["kv_type"] == "int8":
            top = rows.abs().amax(-1).clamp(min=1e-5)
            st[n + "s"][page, :, slot] = top / 127.0
            rows = torch.round(rows * (127.0 / top)[..., None])
        st[n][page, :, slot] = rows.to(st[n].dtype)
    if st["c"]["kv_type"] == "bf16":
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    return {"q": st["q"], **_rows(st, page, slot)}


def _rows(st, page, slot):
    """Rows of the cache as bf16 [rows, KV heads, d]."""
    if st["c"]["kv_type"] == "bf16":
        return {n: st[n][page, :, slot] for n in ("k", "v")}
    return {n: (st[n][page, :, slot].float() * st[n + "s"][page, :, slot][..., None]).to(torch.bfloat16)
            for n in ("k", "v")}


def _plain_read(st):
    b, pos = _spread(st["cu_rows"], st["rows"])
    return _rows(st, *_slots(st, b, pos + st["starts"].long()[b]))


def _plain_attend(st):
    hq, hk, d = HEADS[st["c"]["heads"]]
    nb, n, m = st["c"]["B"], st["max_q"], st["max_kv"]
    lens = (st["cu"][1:] - st["cu"][:-1]).long()
    kv = st["kv_lens"].long()
    key = torch.arange(m, device=DEV)
    page, slot = _slots(st, torch.arange(nb, device=DEV)[:, None], key[None].expand(nb, m))
    page = page.clamp(min=0)
    k, v = (st[x][page, :, slot].float() for x in ("k", "v"))  # [B, keys, KV heads, d]
    if st["ks"] is not None:
        k, v = k * st["ks"][page, :, slot][..., None], v * st["vs"][page, :, slot][..., None]
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    b, i = _spread(st["cu"], st["tokens"])
    q = torch.zeros((nb, n, hq, d), device=DEV)
    q[b, i] = st["q"].view(-1, hq, d).float()
    q = q.view(nb, n, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(nb, hk, -1, d)  # rows: head in group, token
    s = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(nb, hk, hq // hk, n, m)
    # token i of a chunk sees the keys before kv - len + i + 1
    ends = (kv - lens)[:, None] + torch.arange(n, device=DEV)[None] + 1
    hidden = key[None, None] >= torch.minimum(ends, kv[:, None])[..., None]
    s.masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    v = v.masked_fill((key[None] >= kv[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(s.view(nb, hk, -1, m), v).view(nb, hk, hq // hk, n, d) / total.clamp(min=1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(nb, n, hq * d)[b, i].to(torch.bfloat16)


_PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(c, seed):
    st = prepare(c, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[c["op"]](st)


def _contents(st, b, lo, hi):
    """Keys and values lo .. hi - 1 of sequence b in 64 bits, [KV heads, rows, d] each."""
    page = st["c"]["page"]
    at = st["block_table"][b, : -(-hi // page)].long()
    out = []
    for n in ("k", "v"):
        x = st[n][at].double()
        if st[n + "s"] is not None:
            x = x * st[n + "s"][at].double()[..., None]
        out.append(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, lo:hi])
    return out


def _exact_read(st):
    parts = [_contents(st, b, 0, n) for b, n in enumerate(st["kv_lens"].tolist())]
    return {"k": torch.cat([p[0].transpose(0, 1) for p in parts]), "v": torch.cat([p[1].transpose(0, 1) for p in parts])}


def _exact_append(st):
    c = st["c"]
    hq, hk, d = HEADS[c["heads"]]
    half, page = c["rot"] // 2, c["page"]
    cu = st["cu"].tolist()
    out = {n: st[n].double() if c["kv_type"] == "bf16" else [] for n in ("k", "v")}
    out["q"] = torch.empty((st["tokens"], hq * d), dtype=torch.float64, device=DEV)
    j = torch.arange(half, device=DEV)
    first, second = (2 * j, 2 * j + 1) if c["interleaved"] else (j, j + half)
    for b, kv in enumerate(st["kv_lens"].tolist()):
        lo, hi = cu[b], cu[b + 1]
        if hi == lo:
            continue
        pos = torch.arange(kv - (hi - lo), kv, device=DEV)
        turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None]
        x = st["qkv"][lo:hi].double().view(hi - lo, hq + 2 * hk, d)
        z = torch.complex(x[:, : hq + hk, first], x[:, : hq + hk, second]) * turn
        y = x[:, : hq + hk].clone()
        y[..., first], y[..., second] = z.real, z.imag
        out["q"][lo:hi] = y[:, :hq].reshape(hi - lo, hq * d)
        for n, rows in (("k", y[:, hq:]), ("v", x[:, hq + hk:])):
            if c["kv_type"] == "bf16":
                out[n][st["block_table"][b].long()[pos // page], :, pos % page] = rows
            else:
                step = rows.abs().amax(-1, keepdim=True).clamp(min=1e-5) / 127.0
                out[n].append(torch.round(rows / step) * step)
    if c["kv_type"] == "int8":
        out["k"], out["v"] = torch.cat(out["k"]), torch.cat(out["v"])
    return out


def _exact_attend(st):
    hq, hk, d = HEADS[st["c"]["heads"]]
    cu = st["cu"].tolist()
    out = torch.zeros((st["tokens"], hq, d), dtype=torch.float64, device=DEV)
    for b, kv in enumerate(st["kv_lens"].tolist()):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        k, v = _contents(st, b, 0, kv)
        see = torch.arange(kv, device=DEV)[None] <= torch.arange(kv - n, kv, device=DEV)[:, None]
        for h in range(hq):
            q = st["q"][cu[b]:cu[b + 1], h * d:(h + 1) * d].double()
            s = (q @ k[h // (hq // hk)].T / math.sqrt(d)).masked_fill(~see, -math.inf)
            out[cu[b]:cu[b + 1], h] = torch.softmax(s, -1) @ v[h // (hq // hk)]
    return out.view(-1, hq * d)
