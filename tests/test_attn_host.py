"""Host side of the attention calls, without a GPU: tensors that only claim to lie on one, and stand-ins for the
library's entry points."""

import ctypes
import shutil
import subprocess
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import _abi, attn  # noqa: E402


class OnPaper(torch.Tensor):
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(str(func))


def paper(*shape, dtype=torch.bfloat16, device="cuda:0"):
    """A tensor of that shape and device without memory (data pointer 0)."""
    return torch.Tensor._make_wrapper_subclass(OnPaper, shape, dtype=dtype, device=device)


CACHE = _abi.KvCacheC(16, 16, None, None, 4096, 4096, 1, 16, 2, 128, 0)


@pytest.fixture
def native():
    """The binding; the library's own entry points are put back at the end."""
    yield attn._native()
    attn._bound = None
    attn._native()


def calls(native):
    """The three native calls on tensors that fit."""
    q, kv, i32 = paper(2, 4, 128), paper(2, 2, 128), paper(2, dtype=torch.int32)
    return {
        "append": lambda: native.append(ctypes.addressof(CACHE), 0, q, kv, kv, None, paper(2, dtype=torch.int64), None,
                                        None, None, 1e-6, False, paper(2, 4, 128), None, None, 0),
        "decode": lambda: native.decode(ctypes.addressof(CACHE), 0, 4, 2, 1.0, 256, q, paper(2, 3, dtype=torch.int32), i32,
                                        paper(2, 4, 128), 0),
        "prefill": lambda: native.prefill(0, q, kv, kv, i32, None, 1.0, paper(2, 4, 128), 0),
    }


@pytest.mark.skipif(shutil.which("cc") is None, reason="no C compiler")
@pytest.mark.parametrize("which", ["append", "decode", "prefill"])
def test_other_threads_run_while_a_call_waits(native, tmp_path, which):
    """The library's calls may wait for its mutex (another thread's call holds it until its stream is done): a thread
    that waits there must not keep the interpreter from the others."""
    src, lib = tmp_path / "wait.c", tmp_path / "wait.so"
    src.write_text("#include <unistd.h>\n"
                   "volatile int entered, go;\n"
                   "int stand_in(void) { entered = 1; for (int i = 0; i < 3000 && !go; ++i) usleep(1000);\n"
                   "                     return go ? 41 : 42; }\n")
    subprocess.run(["cc", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    L = ctypes.CDLL(str(lib))
    at = ctypes.cast(L.stand_in, ctypes.c_void_p).value
    native.bind(at, at, at)
    got = []
    t = threading.Thread(target=lambda: got.append(calls(native)[which]()))
    t.start()
    entered = ctypes.c_int.in_dll(L, "entered")
    end = time.monotonic() + 10
    while not entered.value and time.monotonic() < end:
        time.sleep(0.001)
    ctypes.c_int.in_dll(L, "go").value = 1
    t.join(20)
    assert got == [41]  # 42: nobody could let it go
