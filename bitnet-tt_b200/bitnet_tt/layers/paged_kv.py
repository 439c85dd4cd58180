"""Paged KV cache of one layer: pools of pages shared by sequences of any length.

Where KVCache (layers/attention.py) holds max_seq_len rows for every sequence
and takes one token per sequence or a prompt from position 0, a PagedKVCache
holds pages: a block table names each sequence's, a call appends or attends any
number of new tokens per sequence (a decode token, drafted tokens, a chunk of a
prompt, none), and the pages are bf16 or int8, quantised as they are written.

The arguments shared by the calls, all on the cache's device:
  block_table  int32 [B, max_pages]: the pages of sequence b, in order; only the
               entries that a sequence's length reaches are read
  cu_seqlens   int32 [B + 1]: row offsets of the sequences' new tokens
  kv_lens      int32 [B]: each sequence's keys, its new tokens included
Work is enqueued on the device's current stream.  Shapes and types are checked
here (ValueError) and in the library (RuntimeError); page ids, offsets and
lengths live on the device, where a bad one is recorded
(_lib.last_device_status) and skipped.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
_INT_MAX = 0x7fffffff


@dataclass
class PagedBatch:
    """The new tokens of one forward pass over paged caches: one per sequence of a
    decode step, any number elsewhere."""

    cu_seqlens: torch.Tensor   # int32 [B + 1]
    kv_lens: torch.Tensor      # int32 [B], the new tokens included
    block_table: torch.Tensor  # int32 [B, max_pages]
    max_seqlen: int
    max_kv_len: int

    @classmethod
    def of(cls, new_tokens: list[int], kv_lens: list[int], pages: list[list[int]], device) -> "PagedBatch":
        """From host lists: new tokens, keys after them, and pages of every sequence."""
        width = max(1, max(len(x) for x in pages))
        table = torch.full((len(pages), width), -1, dtype=torch.int32)
        for b, x in enumerate(pages):
            table[b, : len(x)] = torch.tensor(x, dtype=torch.int32)
        cu = torch.tensor([0, *new_tokens], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        return cls(cu.to(device), torch.tensor(kv_lens, dtype=torch.int32).to(device), table.to(device),
                   max(new_tokens), max(kv_lens))


def _want(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class PagedKVCache:
    """Pools [num_pages, num_kv_heads, page_size, head_dim] of keys and values;
    dtype torch.bfloat16, or torch.int8 with fp32 scales [num_pages, num_kv_heads,
    page_size]: a row's value is code * scale."""

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device=None,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        dev = torch.device(device if device is not None else "cuda")
        _want(dtype in (torch.bfloat16, torch.int8), f"paged cache of {dtype}: bfloat16 or int8 expected")
        k, v = (torch.zeros(shape, dtype=dtype, device=dev) for _ in range(2))
        ks, vs = ((torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2))
                  if dtype == torch.int8 else (None, None))
        self._bind(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, key_pages: torch.Tensor, value_pages: torch.Tensor, key_scale: torch.Tensor | None = None,
                     value_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over existing pools (nothing is copied)."""
        self = cls.__new__(cls)
        self._bind(key_pages, value_pages, key_scale, value_scale)
        return self

    def _bind(self, k: torch.Tensor, v: torch.Tensor, ks: torch.Tensor | None, vs: torch.Tensor | None) -> None:
        _want(k.dim() == 4 and k.shape == v.shape, "key and value pages must be equal [pages, heads, page_size, head_dim]")
        _want(k.dtype == v.dtype and k.dtype in (torch.bfloat16, torch.int8), "pages must be bfloat16 or int8")
        _want(k.is_contiguous() and v.is_contiguous(), "pages must be contiguous")
        _want(k.shape[2] in PAGE_SIZES, f"page_size {k.shape[2]} is not one of {PAGE_SIZES}")
        _want(k.shape[3] in (64, 128), f"head_dim {k.shape[3]} is not 64 or 128")
        _want(k.device == v.device, "key and value pages must be on one device")
        if k.dtype == torch.int8:
            for s in (ks, vs):
                _want(s is not None and s.dtype == torch.float32 and s.shape == k.shape[:3] and s.is_contiguous()
                      and s.device == k.device, "int8 pages need contiguous fp32 scales [pages, heads, page_size]")
        else:
            _want(ks is None and vs is None, "bfloat16 pages have no scales")
        self._pools = (k, v, ks, vs)
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        self.device = k.device
        self._index = k.get_device()
        self.dtype = k.dtype
        self._scale = k.shape[3] ** -0.5
        self._module = _lib.paged_module()
        self._handle = self._module.cache(
            *(_lib.ptr(t) or 0 for t in (k, v, ks, vs)), self.num_pages, self.page_size, self.num_kv_heads, self.head_dim,
            _lib.KV_INT8 if k.dtype == torch.int8 else _lib.KV_BF16, self._index)

    # The handle holds the pools' addresses: their contents may be written, the tensors not replaced.
    @property
    def key_pages(self) -> torch.Tensor:
        return self._pools[0]

    @property
    def value_pages(self) -> torch.Tensor:
        return self._pools[1]

    @property
    def key_scale(self) -> torch.Tensor | None:
        return self._pools[2]

    @property
    def value_scale(self) -> torch.Tensor | None:
        return self._pools[3]

    def nbytes(self) -> int:
        """Bytes of the pools, scales included."""
        return sum(t.numel() * t.element_size() for t in self._pools if t is not None)

    # ---- what is wrong with a call's arguments -------------------------------
    # The module tests all of them at once; these run when it says that something is
    # wrong, to say what.
    def _refuse_index(self, block_table: torch.Tensor, **vectors: torch.Tensor) -> None:
        for name, t in {"block_table": block_table, **vectors}.items():
            if t.dtype is not torch.int32 or t.get_device() != self._index or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor on {self.device}")
        if block_table.dim() != 2 or min(block_table.shape) < 1:
            raise ValueError("block_table must be [sequences, pages]")
        b = block_table.shape[0]
        for name, t in vectors.items():
            if t.numel() != b + name.startswith("cu_"):
                raise ValueError(f"{name} of shape {tuple(t.shape)} does not belong to a block_table of {b} sequences")

    def _refuse_rows(self, t: torch.Tensor, shared: int, name: str) -> int:
        if t.dtype is not torch.bfloat16 or t.get_device() != self._index or t.dim() != 2 or t.stride(1) != 1:
            raise ValueError(f"{name} must be bfloat16 rows [tokens, features] on {self.device}")
        heads, rest = divmod(t.shape[1], self.head_dim)
        heads -= shared
        if rest or heads < 1 or heads % self.num_kv_heads:
            raise ValueError(f"{name} of {t.shape[1]} features does not hold heads of {self.head_dim} for "
                             f"{self.num_kv_heads} KV heads")
        return heads

    def _refuse_out(self, t: torch.Tensor | None, shape: tuple, name: str) -> None:
        if t is not None and (t.dtype is not torch.bfloat16 or t.get_device() != self._index or t.shape != shape
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous bfloat16 {shape} on {self.device}")

    def _refuse_rest(self, status: int | None, what: str) -> None:
        if status is not None:
            _lib.check(status, what)
        raise ValueError(f"{what}: an argument is not as documented")

    # ---- calls -------------------------------------------------------------
    def append(self, qkv: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor,
               rope_cos: torch.Tensor, rope_sin: torch.Tensor, q_out: torch.Tensor | None = None,
               interleaved: bool = False, stepwise: bool = False) -> torch.Tensor:
        """Rotates the new tokens' queries and keys (qkv rows [tokens, (n_heads +
        2 n_kv) * head_dim], which may be strided), writes keys and values to their
        pages and returns the queries [tokens, n_heads * head_dim].  Token i of n
        stands at position kv_lens[b] - n + i.  rope tables: bf16 or fp32 [positions,
        rotary_dim / 2]; rotary_dim may be less than head_dim.  The rotation is
        rounded once; stepwise rounds its products and sums to bf16 too, as the bf16
        model code and the contiguous cache's kernels do."""
        r = self._module.append(self._handle, qkv, cu_seqlens, kv_lens, block_table, rope_cos, rope_sin, q_out,
                                interleaved, stepwise)
        if r is None or type(r) is int:
            self._refuse_index(block_table, cu_seqlens=cu_seqlens, kv_lens=kv_lens)
            heads = self._refuse_rows(qkv, 2 * self.num_kv_heads, "qkv")
            for t in (rope_cos, rope_sin):
                if (t.dtype not in (torch.bfloat16, torch.float32) or t.dtype != rope_cos.dtype or t.dim() != 2
                        or t.shape != rope_cos.shape or t.get_device() != self._index or not t.is_contiguous()):
                    raise ValueError("rope tables must be two equal contiguous bf16 or fp32 [positions, rotary_dim / 2]")
            self._refuse_out(q_out, (qkv.shape[0], heads * self.head_dim), "q_out")
            self._refuse_rest(r, "bitnet_paged_append")
        return r

    def attend(self, q: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor,
               max_seqlen: int, max_kv_len: int, scale: float | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """Causal grouped-head attention of the new tokens' rotated queries [tokens,
        n_heads * head_dim] over their sequences' pages.  max_seqlen and max_kv_len
        bound the new tokens and the keys of every sequence.  scale: 1 /
        sqrt(head_dim) by default.  workspace (attention_workspace): taken from the
        allocator if not given."""
        r = self._module.attend(self._handle, q, cu_seqlens, kv_lens, block_table, max_seqlen, max_kv_len,
                                self._scale if scale is None else scale, out, workspace)
        if r is None or type(r) is int:
            self._refuse_index(block_table, cu_seqlens=cu_seqlens, kv_lens=kv_lens)
            self._refuse_rows(q, 0, "q")
            if max(max_seqlen, max_kv_len) > _INT_MAX or min(max_seqlen, max_kv_len) < -_INT_MAX:
                raise ValueError("max_seqlen and max_kv_len are 32-bit bounds")
            self._refuse_out(out, tuple(q.shape), "out")
            if workspace is not None and (workspace.get_device() != self._index or not workspace.is_contiguous()):
                raise ValueError(f"workspace must be a contiguous tensor on {self.device}")
            self._refuse_rest(r, "bitnet_paged_attention")
        return r

    def attention_workspace(self, batch: int, total_tokens: int, max_seqlen: int, max_kv_len: int,
                            num_heads: int) -> torch.Tensor | None:
        """Workspace of attend() for these bounds (None when it needs none).  Calls
        that may overlap need one each."""
        _want(all(0 <= x <= _INT_MAX for x in (batch, total_tokens, max_seqlen, max_kv_len, num_heads)),
              "the workspace's bounds are out of range")
        with torch.cuda.device(self._index):
            n = _lib.paged_attention_workspace_bytes(batch, total_tokens, max_seqlen, max_kv_len, num_heads,
                                                     self.num_kv_heads, self.head_dim)
        return torch.empty(n, dtype=torch.uint8, device=self.device) if n else None

    def read(self, block_table: torch.Tensor, starts: torch.Tensor | None, cu_rows: torch.Tensor, total_rows: int,
             k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows starts[b] .. starts[b] + cu_rows[b + 1] - cu_rows[b] - 1 of every
        sequence (starts None: from row 0) as packed bf16 keys and values
        [total_rows, n_kv, head_dim]."""
        r = self._module.read(self._handle, block_table, starts, cu_rows, total_rows, k_out, v_out)
        if r is None or type(r) is int:
            self._refuse_index(block_table, cu_rows=cu_rows, **({} if starts is None else {"starts": starts}))
            if not 0 <= total_rows <= _INT_MAX:
                raise ValueError("total_rows is out of range")
            shape = (total_rows, self.num_kv_heads, self.head_dim)
            self._refuse_out(k_out, shape, "k_out")
            self._refuse_out(v_out, shape, "v_out")
            self._refuse_rest(r, "bitnet_paged_read")
        return r
