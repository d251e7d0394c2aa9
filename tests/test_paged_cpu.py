"""Refusals of the paged cache entry points: checks that run before any device work, so they hold without a GPU."""
import ctypes

import pytest

from gptoss_b200 import capi


@pytest.fixture(scope="module")
def lib():
    if not capi.DEFAULT_LIB.exists():
        import importlib.util
        spec = importlib.util.spec_from_file_location("gptoss_build", capi.PKG / "build.py")
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.build()
    return capi.load()


A = 1 << 20          # an aligned address nothing reads
S4 = ctypes.c_longlong * 4


@pytest.mark.parametrize("change,message", [
    ({"type": 0}, b"cache type"), ({"type": 7}, b"cache type"), ({"head_dim": 96}, b"head_dim"),
    ({"layers": 0}, b"at least 1"), ({"num_pages": 0}, b"at least 1"), ({"page_size": 0}, b"at least 1"),
    ({"kv_heads": -1}, b"at least 1"), ({"k": None}, b"null"), ({"v": A + 2}, b"16-byte"),
    ({"strides": S4(0, 1024, 68, 64)}, b"multiples of 8"), ({"strides": S4(0, 1024, -64, 64)}, b"multiples of 8"),
    ({"strides": None}, b"null"), ({"kv_heads": 5000}, b"1024"),
])
def test_pool_create_refuses(lib, change, message):
    a = {"k": A, "v": A, "type": 1, "layers": 1, "num_pages": 4, "page_size": 16, "kv_heads": 1, "head_dim": 64,
         "strides": S4(0, 1024, 64, 64)} | change
    assert not lib.gptoss_kv_pool_create(*a.values())
    assert message in lib.gptoss_last_error(), lib.gptoss_last_error()


def test_null_pool_is_refused_everywhere(lib):
    b = capi.KvBatch(1, 1, 1, 1, A, A, A)
    calls = [
        lambda: lib.gptoss_kv_pool_status(None, ctypes.byref(ctypes.c_int())),
        lambda: lib.gptoss_kv_append(None, 0, ctypes.byref(b), A, A, A, 0, 64, 64, 1, A, A, 1, 64, 0, A, 0, None),
        lambda: lib.gptoss_paged_attention(None, 0, ctypes.byref(b), A, 1, 64, 1, None, 1.0, 0, A, 64, None),
        lambda: lib.gptoss_kv_fork(None, A, A, A, 1, A, None, 1, 1, A, A, A, None),
        lambda: lib.gptoss_kv_compact(None, A, A, A, 1, 1, A, A, A, A, None),
    ]
    for call in calls:
        assert call() == -1
        assert b"null pool" in lib.gptoss_last_error()
    lib.gptoss_kv_pool_destroy(None)


@pytest.mark.parametrize("change,message", [
    ({"type": 5}, b"unknown type"), ({"beams": 0}, b"1 .. 64"), ({"beams": 65}, b"1 .. 64"), ({"picks": 0}, b"1 .. 64"),
    ({"picks": 65}, b"1 .. 64"), ({"vocab": 0}, b"vocab"), ({"batch": -1}, b"batch"), ({"stride": 99}, b"row_stride"),
    ({"beams": 64, "vocab": 1 << 26, "stride": 1 << 26}, b"2^31"), ({"done": A, "token": 100}, b"done_token"),
    ({"done": A, "token": -1}, b"done_token"), ({"logits": None}, b"null"), ({"scores": None}, b"null"),
    ({"rows": None}, b"null"), ({"logits": A + 1}, b"aligned"),
])
def test_beam_select_refuses(lib, change, message):
    a = {"logits": A, "type": 0, "stride": 100, "scores": A, "done": None, "token": 0, "batch": 1, "beams": 4,
         "vocab": 100, "picks": 4, "out": A, "rows": A, "tokens": A, "stream": None} | change
    assert lib.gptoss_beam_select(*a.values()) == -1
    assert message in lib.gptoss_last_error(), lib.gptoss_last_error()


def test_beam_select_of_no_requests_is_done(lib):
    assert lib.gptoss_beam_select(A, 0, 100, A, None, 0, 0, 4, 100, 4, A, A, A, None) == 0
