"""Where a registered layer's memory begins must not decide which kernels run it."""

import ctypes

import pytest
import torch

import colizig_b200 as cz
from colizig_b200 import moe, synth

pytestmark = pytest.mark.gpu


def test_a_small_layer_on_512_bytes_keeps_the_grouped_path():
    """cudaMalloc gives small blocks on 512 bytes, not on 1,024: a layer registered when the next free place is such a
    one still runs 64 tokens as two grouped products, not as decode launches."""
    torch.cuda.init()
    cz.gpu.init()
    rt = ctypes.CDLL("libcudart.so.12")
    rt.cudaMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
    rt.cudaFree.argtypes = [ctypes.c_void_p]

    def block(n):
        p = ctypes.c_void_p()
        assert rt.cudaMalloc(ctypes.byref(p), n) == 0
        return p.value

    d = moe.Dims(hidden=256, experts=4, topk=2, inter=128)
    w = synth.make_layer(d, seed=5, device="cuda")
    x = synth.make_tokens(64, d.hidden, 2, device="cuda")
    room = 400 * 1024  # what the layer takes, and a little
    held, layers = [], []
    try:
        for _ in range(200):
            held.append(block(room + 512))  # the next block of this hole lies 512 bytes further on
            at = block(room)
            rt.cudaFree(at)
            if at % 1024:
                break
        assert at % 1024 == 512
        layers.append(moe.Layer.from_weights(820, d, w))
        moe.kernel_timer(64)
        moe.forward(layers[0], x)
        assert [k for k, _ in moe.kernel_timer_read()] == [moe.TIMER_PREFILL_GATE_UP, moe.TIMER_PREFILL_DOWN]
        moe.check()
    finally:
        moe.kernel_timer(0)
        for layer in layers:
            layer.unregister()
        for p in held:
            rt.cudaFree(p)
