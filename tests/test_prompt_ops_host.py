"""What the many-row entry points refuse before any GPU work: arguments that are missing, tensors of the wrong type, layout or device."""
import ctypes

import pytest
import torch

from leviathan_b200 import _lib as L
from leviathan_b200 import api


@pytest.fixture(scope="module")
def lib():
    import os

    if not os.path.exists(L.LIB_PATH):
        from leviathan_b200.build import build_library

        build_library()
    return L.load()


@pytest.mark.parametrize("name", ["lev_attn_chunk", "lev_attn_prompt", "lev_logprobs", "lev_norm_residual"])
def test_null_arguments_are_an_error_code(lib, name):
    f = getattr(lib, name)
    args = [t() if t in (ctypes.c_int, ctypes.c_int32, ctypes.c_int64) else (t(0.0) if t is ctypes.c_float else None) for t in f.argtypes]
    assert lib.lev_status_name(f(*args)) == b"badArgument"


def test_head_rows():
    api._torch()
    fused = torch.zeros(5, 10, 128)
    assert api._head_rows(fused[:, :6], "q") == (torch.Size([5, 6, 128]), 1280)
    assert api._head_rows(fused[1:, 8:], "v") == (torch.Size([4, 2, 128]), 1280)
    for bad in (torch.zeros(5, 128), fused[:, ::2], fused[..., ::2], fused.transpose(0, 1), fused[..., :64]):
        with pytest.raises(ValueError, match="q: "):
            api._head_rows(bad, "q")


def test_element_types():
    api._torch()
    assert [api._elem(torch.zeros(1, dtype=t), "x", api._ANY) for t in (torch.float32, torch.float16, torch.bfloat16)] == [L.ELEM_F32, L.ELEM_F16, L.ELEM_BF16]
    for t, allowed in ((torch.bfloat16, api._F32_F16), (torch.float32, api._ANY16), (torch.float64, api._ANY), (torch.int32, api._ANY)):
        with pytest.raises(TypeError, match="x is "):
            api._elem(torch.zeros(1, dtype=t), "x", allowed)


def test_index_vectors():
    api._torch()
    api._i32(torch.zeros(3, dtype=torch.int32), 3, "start")
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="start: 3"):
            api._i32(bad, 3, "start")
    with pytest.raises(ValueError, match="cuda:0"):
        api._on(0, None, torch.zeros(1))


def test_cache_over_pools_of_the_caller():
    k = torch.zeros(4, 16, 2, 128, dtype=torch.float16)
    table = torch.zeros(2, 3, dtype=torch.int32)
    c = api.PagedKV.over(k, torch.zeros_like(k), table)
    l = c.layout
    assert (l.kv_type, l.page, l.kv_heads, l.head_dim, l.blocks, l.max_blocks, l.slots) == (L.KV_F16, 16, 2, 128, 4, 3, 2)
    assert c.k is k and c.table is table
    with pytest.raises(ValueError):
        api.PagedKV.over(k, torch.zeros(4, 16, 2, 64, dtype=torch.float16), table)
    with pytest.raises(ValueError):
        api.PagedKV.over(k, torch.zeros(4, 2, 16, 128, dtype=torch.float16).transpose(1, 2), table)
    with pytest.raises(ValueError):
        api.PagedKV.over(k, torch.zeros_like(k), table.long())
    with pytest.raises(TypeError):
        api.PagedKV.over(k.bfloat16(), k.bfloat16(), table)


# the arguments each native call over many rows takes, handles NULL
ROW_CALLS = {
    "attn_chunk": (None, None, None, None, None, 1, None, None, None, 1, 8, None, 0, 1024, 0, 1.0, None, 2, 1024),
    "attn_prompt": (None, 1, None, 1, 8, 2, 128, 2, None, 1024, None, 256, None, 256, 0, 1.0, None, 1024),
    "norm_residual": (None, None, None, 1, 32, 0, None, None, 0, 1.0, 1.0, None, 1e-6, None, None, 0),
    "logprobs": (None, None, 0, 1, 32, 32, 0.0, None, 0, None, None, None, None),
}


def test_row_calls_native_and_through_ctypes(lib, monkeypatch, tmp_path):
    native = L.host()._rows
    assert sorted(n for n in dir(native) if not n.startswith("_")) == sorted(ROW_CALLS)
    monkeypatch.setattr(L, "_host", None)
    monkeypatch.setattr(L, "HOST_PATH", str(tmp_path / "missing.so"))
    through_ctypes = L.host()._rows
    for name, args in ROW_CALLS.items():
        for form in (native, through_ctypes):
            assert L.STATUS[getattr(form, name)(*args)] == "badArgument", name
            with pytest.raises(TypeError):
                getattr(form, name)(*args[:-1])


def test_head_rows_of_one_row_or_one_head():
    """strides of dimensions of size one mean nothing"""
    api._torch()
    x = torch.zeros(4, 128)
    one_row = x[None].expand(1, 4, 128).as_strided((1, 4, 128), (0, 128, 1))
    assert api._head_rows(one_row, "q") == (torch.Size([1, 4, 128]), 512)
    assert api._head_rows(x[None].as_strided((1, 4, 128), (7, 128, 1)), "q")[1] == 512
    one_head = x.as_strided((4, 1, 128), (128, 1, 1))
    assert api._head_rows(one_head, "k") == (torch.Size([4, 1, 128]), 128)
    assert api._head_rows(x[:1].as_strided((1, 1, 128), (0, 0, 1)), "k")[1] == 128


@pytest.mark.parametrize("where", ["v", "table"])
def test_cache_over_pools_of_two_devices_is_refused(where):
    """a kernel would follow the other device's address"""
    t = dict(k=torch.zeros(4, 16, 2, 128, dtype=torch.float16), v=torch.zeros(4, 16, 2, 128, dtype=torch.float16), table=torch.zeros(2, 3, dtype=torch.int32))
    t[where] = t[where].to("meta")
    with pytest.raises(ValueError, match="one device"):
        api.PagedKV.over(t["k"], t["v"], t["table"])


def test_blocks_of_a_cache_over_pools_are_the_callers():
    c = api.PagedKV.over(torch.zeros(4, 16, 2, 128, dtype=torch.float16), torch.zeros(4, 16, 2, 128, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int32))
    for call in (lambda: c.ensure(0, 5), lambda: c.release(0)):
        with pytest.raises(ValueError, match="hands out"):
            call()
