"""The native checks in front of the attention calls, as far as they go without a GPU: whatever does not fit is
a Python exception before the library is reached."""

import ctypes

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import _abi, attn  # noqa: E402


@pytest.fixture(scope="module")
def native():
    return attn._native()


CACHE = _abi.KvCacheC(16, 16, None, None, 4096, 4096, 1, 16, 2, 128, 0)
AT = ctypes.addressof(CACHE)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_host_tensors_are_refused(native):
    i32, i64 = torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="q must be .*cuda:0.*on cpu"):
        native.decode(AT, 0, 4, 2, 1.0, 256, bf(2, 4, 128), i32[None], i32, None, 0)
    with pytest.raises(ValueError, match="q must be"):
        native.prefill(0, bf(2, 4, 128), bf(2, 2, 128), bf(2, 2, 128), i32, None, 1.0, None, 0)
    with pytest.raises(ValueError, match="q must be"):
        native.append(AT, 0, bf(2, 4, 128), bf(2, 2, 128), bf(2, 2, 128), None, i64, None, None, None, 1e-6, False, None,
                      None, None, 0)


def test_wrong_kinds_of_arguments(native):
    q = bf(2, 4, 128)
    for bad in (None, 3, "q", [q]):
        with pytest.raises(ValueError, match="q must be a tensor"):
            native.prefill(0, bad, q, q, q, None, 1.0, None, 0)
    with pytest.raises(ValueError, match="64 or 128"):
        native.prefill(0, bf(2, 4, 96), q, q, q, None, 1.0, None, 0)
    with pytest.raises(ValueError, match="64 or 128"):
        native.prefill(0, bf(2, 128), q, q, q, None, 1.0, None, 0)
    with pytest.raises(TypeError, match="wanted"):
        native.decode(AT, 0)
    with pytest.raises(TypeError):
        native.decode(AT, "0", 4, 2, 1.0, 256, q, q, q, None, 0)
    with pytest.raises(OverflowError):
        native.decode(AT, 1 << 70, 4, 2, 1.0, 256, q, q, q, None, 0)


def test_cache_of_host_tensors_is_refused():
    with pytest.raises(ValueError, match="CUDA"):
        attn.KvCache(bf(2, 2, 16, 128), bf(2, 2, 16, 128))
    with pytest.raises(ValueError, match="CUDA"):
        attn.prefill(bf(2, 4, 128), bf(2, 2, 128), bf(2, 2, 128), torch.zeros(2, dtype=torch.int32))
