"""What a PagedKVCache and its module hold on the host."""

import pytest
import torch


def _pool(dtype=torch.bfloat16):
    return torch.zeros((8, 2, 16, 64), dtype=dtype)


@pytest.fixture
def host(monkeypatch):
    from bitnet_tt import _lib

    monkeypatch.setattr(_lib, "ptr", lambda t: None if t is None else t.data_ptr())


def test_pools_cannot_be_replaced_under_the_handle(host):
    """The handle keeps addresses: another tensor in an attribute would leave them on freed memory."""
    from bitnet_tt.layers import PagedKVCache

    k, v, s = _pool(torch.int8), _pool(torch.int8), torch.zeros((8, 2, 16))
    c = PagedKVCache.from_tensors(k, v, s, s.clone())
    assert c.key_pages is k and c.value_pages is v and c.key_scale is s
    for name in ("key_pages", "value_pages", "key_scale", "value_scale"):
        with pytest.raises(AttributeError):
            setattr(c, name, torch.ones(4))
    assert c.key_pages is k and c.key_scale is s


def test_nbytes_counts_pools_and_scales(host):
    from bitnet_tt.layers import PagedKVCache

    n = 8 * 2 * 16
    assert PagedKVCache.from_tensors(_pool(), _pool()).nbytes() == 2 * n * 64 * 2
    s = torch.zeros((8, 2, 16))
    assert PagedKVCache.from_tensors(_pool(torch.int8), _pool(torch.int8), s, s.clone()).nbytes() == 2 * n * (64 + 4)


def test_workspace_bounds_beyond_32_bits_are_refused(host):
    """As attend() refuses them; cut to 32 bits they would size another call's workspace."""
    from bitnet_tt.layers import PagedKVCache

    c = PagedKVCache.from_tensors(_pool(), _pool())
    good = dict(batch=1, total_tokens=1, max_seqlen=1, max_kv_len=40, num_heads=4)
    assert c.attention_workspace(**good) is None
    for name in good:
        for bad in ((1 << 32) + good[name], 1 << 31, -1):
            with pytest.raises(ValueError):
                c.attention_workspace(**(good | {name: bad}))


def test_the_module_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    import os
    import subprocess

    from bitnet_tt import _build

    ext = tmp_path / "_paged.so"
    monkeypatch.setattr(_build, "EXT_PATH", str(ext))
    built = []

    def compiler(cmd, **kw):
        built.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(_build.subprocess, "run", compiler)
    for _ in range(2):
        assert _build.build_binding() == str(ext)
    assert len(built) == 1
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    for _ in range(2):
        _build.build_binding()
    assert len(built) == 2
    os.utime(ext, (1, 1))  # older than its sources
    _build.build_binding()
    assert len(built) == 3


def test_a_module_of_another_torch_is_refused(monkeypatch):
    from bitnet_tt import _lib

    assert _lib.paged_module().torch_version == torch.__version__.split("+")[0]
    monkeypatch.setattr(_lib, "_paged", None)
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    with pytest.raises(RuntimeError, match="2.99.0"):
        _lib.paged_module()
