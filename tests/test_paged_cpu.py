"""The paged cache's refusals, which need no GPU: the library checks a call's
arguments before it asks for the device, and PagedKVCache checks shapes and
types before it calls the library."""

import pytest
import torch

NONE_GPU = (-3, -4)  # what a call with good arguments answers where there is no GPU


def _buffer(n=1 << 16):
    t = torch.zeros(n, dtype=torch.uint8)
    return t, (t.data_ptr() + 255) // 256 * 256


def _call(name, over_kv=None, **over):
    """Entry point `name` with good arguments but for those in `over` (by name)
    and `over_kv` (fields of the cache)."""
    from bitnet_tt import _lib

    keep, a = _buffer()
    kv = dict(k_pages=a, v_pages=a, k_scale=None, v_scale=None, num_pages=8, page_size=16, n_kv_heads=2, head_dim=64,
              kv_type=_lib.KV_BF16)
    kv |= over_kv or {}
    args = {
        "bitnet_paged_append": dict(kv=_lib.PagedKV(*kv.values()), block_table=a, B=2, max_pages=4, cu_seqlens=a,
                                    kv_lens=a, qkv=a, ld_qkv=512, total_tokens=3, n_heads=4, rope_cos=a, rope_sin=a,
                                    rope_len=64, rotary_dim=64, rope_f32=0, interleaved=0, stepwise=0, q_out=a, stream=None),
        "bitnet_paged_read": dict(kv=_lib.PagedKV(*kv.values()), block_table=a, B=2, max_pages=4, starts=None, cu_rows=a,
                                  total_rows=5, k_out=a, v_out=a, stream=None),
        "bitnet_paged_attention": dict(kv=_lib.PagedKV(*kv.values()), block_table=a, B=2, max_pages=4, cu_seqlens=a,
                                       kv_lens=a, q=a, ld_q=256, total_tokens=3, max_seqlen=2, max_kv_len=64, n_heads=4,
                                       scale=0.125, workspace=None, workspace_bytes=0, out=a, stream=None),
    }[name]
    unknown = set(over) - set(args)
    assert not unknown
    args |= over
    st = getattr(_lib.load(), name)(*args.values())
    del keep
    return st


COMMON = [({"B": 0}, -1), ({"max_pages": 0}, -1), ({"block_table": None}, -1), ({"block_table": 2}, -2),
          ({"max_pages": (1 << 31) // 16}, -1)]
COMMON_KV = [({"k_pages": None}, -1), ({"v_pages": None}, -1), ({"k_pages": 8}, -2), ({"num_pages": 0}, -1),
             ({"page_size": 8}, -1), ({"page_size": 48}, -1), ({"page_size": 512}, -1), ({"n_kv_heads": 0}, -1),
             ({"head_dim": 32}, -1), ({"head_dim": 96}, -1), ({"kv_type": 2}, -1), ({"kv_type": 1}, -1),
             ({"kv_type": 1, "k_scale": 16, "v_scale": 8}, -2), ({"kv_type": 1, "k_scale": 4, "v_scale": 16}, -2),
             ({"num_pages": 1 << 26}, -1)]
OWN = {
    "bitnet_paged_append": [({"cu_seqlens": None}, -1), ({"kv_lens": None}, -1), ({"qkv": None}, -1),
                            ({"q_out": None}, -1), ({"rope_cos": None}, -1), ({"rope_sin": None}, -1),
                            ({"qkv": 8}, -2), ({"q_out": 8}, -2), ({"rope_cos": 8}, -2), ({"cu_seqlens": 2}, -2),
                            ({"ld_qkv": 511}, -1), ({"ld_qkv": 504}, -1), ({"ld_qkv": 516}, -1),
                            ({"total_tokens": -1}, -1), ({"n_heads": 3}, -1), ({"n_heads": 0}, -1),
                            ({"rope_len": 0}, -1), ({"rotary_dim": 0}, -1), ({"rotary_dim": 24}, -1),
                            ({"rotary_dim": 80}, -1)],
    "bitnet_paged_read": [({"cu_rows": None}, -1), ({"k_out": None}, -1), ({"v_out": None}, -1), ({"k_out": 8}, -2),
                          ({"starts": 2}, -2), ({"total_rows": -1}, -1)],
    "bitnet_paged_attention": [({"cu_seqlens": None}, -1), ({"kv_lens": None}, -1), ({"q": None}, -1), ({"out": None}, -1),
                               ({"q": 8}, -2), ({"out": 8}, -2), ({"kv_lens": 2}, -2), ({"ld_q": 255}, -1),
                               ({"ld_q": 248}, -1), ({"ld_q": 260}, -1), ({"total_tokens": -1}, -1),
                               ({"max_seqlen": -1}, -1), ({"max_kv_len": -1}, -1), ({"max_kv_len": 65}, -1),
                               ({"n_heads": 3}, -1), ({"n_heads": 0}, -1), ({"n_heads": 130, "ld_q": 8320}, -1),
                               ({"scale": 0.0}, -1), ({"scale": -1.0}, -1), ({"scale": float("nan")}, -1),
                               ({"scale": float("inf")}, -1)],
}


@pytest.mark.parametrize("name", sorted(OWN))
def test_library_refuses_bad_arguments_before_it_asks_for_a_gpu(name):
    for over, want in COMMON + OWN[name]:
        assert _call(name, **over) == want, over
    for over, want in COMMON_KV:
        assert _call(name, over_kv=over) == want, over


@pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers: only where no kernel can be launched")
@pytest.mark.parametrize("name", sorted(OWN))
def test_good_arguments_get_as_far_as_the_device(name):
    assert _call(name) in NONE_GPU
    keep, a = _buffer()
    assert _call(name, over_kv=dict(kv_type=1, k_scale=a, v_scale=a)) in NONE_GPU


def test_workspace_size_follows_from_the_sizes_alone():
    from bitnet_tt import _lib

    ws = _lib.paged_attention_workspace_bytes
    assert ws(32, 32, 1, 128, 20, 5, 128) == 0            # short contexts are not split
    assert ws(1, 1, 1, 32768, 20, 5, 128) > 0             # a long one is
    assert ws(1, 1, 1, 32768, 20, 5, 128) % 16 == 0
    for bad in [(0, 1, 1, 64, 4, 2, 64), (1, -1, 1, 64, 4, 2, 64), (1, 1, 1, 64, 4, 3, 64), (1, 1, 1, 64, 4, 2, 80),
                (1, 1, -1, 64, 4, 2, 64), (1, 1, 1, -1, 4, 2, 64)]:
        assert ws(*bad) == 0


@pytest.fixture
def host_cache(monkeypatch):
    """A cache over host tensors: the module refuses them, and the checks say why.
    Good arguments but for their device are the last check's."""
    from bitnet_tt import _lib
    from bitnet_tt.layers import PagedKVCache

    monkeypatch.setattr(_lib, "ptr", lambda t: None if t is None else t.data_ptr())
    k = torch.zeros((8, 2, 16, 64), dtype=torch.bfloat16)
    return PagedKVCache.from_tensors(k, k.clone())


def _good():
    i32 = dict(dtype=torch.int32)
    return dict(table=torch.zeros((2, 4), **i32), cu=torch.zeros(3, **i32), lens=torch.zeros(2, **i32),
                qkv=torch.zeros((3, 512), dtype=torch.bfloat16), q=torch.zeros((3, 256), dtype=torch.bfloat16),
                cos=torch.zeros((64, 32)), sin=torch.zeros((64, 32)))


def test_cache_checks_its_pools():
    from bitnet_tt.layers import PagedKVCache

    def pool(*shape, dt=torch.bfloat16):
        return torch.zeros(shape, dtype=dt)

    k, i8, s = pool(8, 2, 16, 64), pool(8, 2, 16, 64, dt=torch.int8), torch.zeros((8, 2, 16))
    for args in [(k, pool(8, 2, 16, 128)), (pool(8, 2, 16), pool(8, 2, 16)), (k, i8), (k.float(), k.float()),
                 (pool(8, 2, 24, 64),) * 2, (pool(8, 2, 8, 64),) * 2, (pool(8, 2, 16, 96),) * 2,
                 (pool(8, 16, 2, 64).transpose(1, 2), k), (i8, i8), (i8, i8, s), (i8, i8, s, s.double()),
                 (i8, i8, s, s[:4]), (k, k, s, s)]:
        with pytest.raises(ValueError):
            PagedKVCache.from_tensors(*args)
    with pytest.raises(ValueError):
        PagedKVCache(8, 16, 2, 64, "cpu", torch.float16)


def test_host_tensors_are_refused(host_cache):
    g = _good()
    for call in (lambda: host_cache.append(g["qkv"], g["cu"], g["lens"], g["table"], g["cos"], g["sin"]),
                 lambda: host_cache.attend(g["q"], g["cu"], g["lens"], g["table"], 2, 64),
                 lambda: host_cache.read(g["table"], None, g["cu"], 5)):
        with pytest.raises(ValueError, match="not as documented"):
            call()
    for call in (lambda: host_cache.attend(g["q"], g["cu"], g["lens"], g["table"], 2, "64"),
                 lambda: host_cache.attend(g["q"], g["cu"], g["lens"], g["table"], 2, 64, scale="1")):
        with pytest.raises((TypeError, ValueError)):
            call()


def _specific(call, **over):
    """Refused with a reason of its own."""
    with pytest.raises(ValueError) as e:
        call(**over)
    assert "not as documented" not in str(e.value), over


def test_append_checks_its_arguments(host_cache):
    def call(**over):
        g = _good() | over
        host_cache.append(g["qkv"], g["cu"], g["lens"], g["table"], g["cos"], g["sin"], g.get("q_out"))

    z = torch.zeros
    for over in [{"table": z((2, 4))}, {"table": z(8, dtype=torch.int32)}, {"cu": z(2, dtype=torch.int32)},
                 {"cu": z(3, dtype=torch.int64)}, {"lens": z(3, dtype=torch.int32)},
                 {"table": z((4, 2), dtype=torch.int32).t()}, {"qkv": z((3, 512))},
                 {"qkv": z((512, 3), dtype=torch.bfloat16).t()}, {"qkv": z((3, 500), dtype=torch.bfloat16)},
                 {"qkv": z((3, 256), dtype=torch.bfloat16)}, {"qkv": z((3, 448), dtype=torch.bfloat16)},
                 {"cos": z((64, 32), dtype=torch.float64), "sin": z((64, 32), dtype=torch.float64)},
                 {"cos": z((64, 16))}, {"sin": z((64, 32), dtype=torch.bfloat16)},
                 {"q_out": z((3, 256))}, {"q_out": z((4, 256), dtype=torch.bfloat16)}]:
        _specific(call, **over)


def test_attend_and_read_check_their_arguments(host_cache):
    def attend(**over):
        g = _good() | over
        host_cache.attend(g["q"], g["cu"], g["lens"], g["table"], 2, 64, out=g.get("out"))

    def read(**over):
        g = _good() | over
        host_cache.read(g["table"], g.get("starts"), g["cu"], g.get("total", 5), g.get("k_out"), g.get("v_out"))

    z = torch.zeros
    for over in [{"q": z((3, 256))}, {"q": z((3, 192), dtype=torch.bfloat16)}, {"q": z((3, 100), dtype=torch.bfloat16)},
                 {"q": z(256, dtype=torch.bfloat16)}, {"cu": z(2, dtype=torch.int32)}, {"lens": z(2)},
                 {"out": z((3, 128), dtype=torch.bfloat16)}, {"out": z((3, 512), dtype=torch.bfloat16)[:, :256]}]:
        _specific(attend, **over)
    for over in [{"cu": z(4, dtype=torch.int32)}, {"starts": z(3, dtype=torch.int32)}, {"starts": z(2)}, {"total": -1},
                 {"k_out": z((5, 2, 128), dtype=torch.bfloat16)}, {"v_out": z((5, 2, 64))}]:
        _specific(read, **over)
