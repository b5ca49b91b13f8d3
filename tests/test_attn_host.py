"""Host side of the attention calls, without a GPU: tensors that only claim to lie on one, and stand-ins for the
library's entry points."""

import contextlib
import ctypes
import shutil
import subprocess
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import _abi, attn, gpu  # noqa: E402


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


@pytest.fixture
def on_paper(native, monkeypatch):
    """The library as if it were up on device 0, with entry points that count their calls and launch nothing, and a cache
    and a plan of tensors without memory."""
    done = []
    at = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: done.append(1) or 0)
    native.bind(*[ctypes.cast(at, ctypes.c_void_p).value] * 3)
    monkeypatch.setattr(gpu, "_ready", True)
    monkeypatch.setattr(gpu, "_device", 0)
    monkeypatch.setattr(attn, "_current", lambda index: 0)
    cache = attn.KvCache(paper(2, 2, 16, 128), paper(2, 2, 16, 128))
    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", lambda *a, **k: paper(1024, dtype=torch.uint8))
        m.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        plan = attn.DecodePlan(cache, 4, 2)
    yield cache, plan, done
    del at


def python_calls(cache, plan):
    q, kv, i32 = paper(2, 4, 128), paper(2, 2, 128), paper(2, dtype=torch.int32)
    return [lambda: attn.append(cache, q, kv, kv, None, paper(2, dtype=torch.int64), q_out=paper(2, 4, 128)),
            lambda: plan.run(q, paper(2, 3, dtype=torch.int32), i32, out=paper(2, 4, 128)),
            lambda: attn.prefill(q, kv, kv, i32, out=paper(2, 4, 128))]


def test_calls_go_through_on_the_library_s_device(on_paper):
    cache, plan, done = on_paper
    for f in python_calls(cache, plan):
        f()
    assert len(done) == 3


def test_calls_are_refused_when_the_library_moved_to_another_device(on_paper, monkeypatch):
    """A cache and a plan made before a shutdown and an init on another device: the kernels would run there, on the first
    device's addresses."""
    cache, plan, done = on_paper
    monkeypatch.setattr(gpu, "_device", 1)
    for f in python_calls(cache, plan):
        with pytest.raises(ValueError, match="cuda:0, the library runs on cuda:1"):
            f()
    assert not done


def test_check_waits_for_a_stream_of_the_library_s_device(monkeypatch):
    """Not of torch's current device, whose stream the library's device cannot wait for."""
    seen = []

    class Library:
        @staticmethod
        def colizig_cuda_attn_check(handle):
            seen.append(handle)
            return 0

    monkeypatch.setattr(gpu, "_device", 3)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(attn, "_current", lambda index: 1000 + index)
    monkeypatch.setattr(_abi, "load", lambda: Library)
    attn.check()
    attn.check(stream=7)
    assert seen == [1003, 7]


@pytest.mark.parametrize("elsewhere", [False, True])
@pytest.mark.parametrize("q", [None, 3, [paper(2, 4, 128)], paper(), paper(2, 4, 0), paper(2, 4, 96)])
def test_queries_that_are_no_rows_of_heads_are_refused(on_paper, monkeypatch, q, elsewhere):
    """ValueError, on the current stream and on a given one."""
    cache, plan, done = on_paper
    kw = {}
    if elsewhere:
        monkeypatch.setattr(attn, "_elsewhere", lambda stream, index: (stream, contextlib.nullcontext()))
        monkeypatch.setattr(attn, "_mark", lambda *a: None)
        monkeypatch.setattr(torch.cuda, "stream", lambda s: s)
        monkeypatch.setattr(torch, "empty", lambda shape, **k: paper(*shape))
        kw = {"stream": 5}
    kv, i32 = paper(2, 2, 128), paper(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="q must be"):
        attn.prefill(q, kv, kv, i32, **kw)
    with pytest.raises(ValueError, match="q must be"):
        plan.run(q, paper(2, 3, dtype=torch.int32), i32, **kw)
    with pytest.raises(ValueError, match="q must be"):
        attn.append(cache, q, kv, kv, None, paper(2, dtype=torch.int64), **kw)
    assert not done
