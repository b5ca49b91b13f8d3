"""examples/decoder.py: append, prompt attention, decode attention, the FP8 projections and the MoE
layer as one decoder runs them."""

import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

from colizig_b200 import attn, moe  # noqa: E402

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder.py")
    spec = importlib.util.spec_from_file_location("decoder_example", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_tokens_after_a_prompt_match_the_whole_prompt(cache):
    """The attention sublayer of a token that comes after a prompt, over the cache, against the same token at the
    end of the whole prompt.  Both run the same f32 projections; q and k are rounded to bf16 alike, the two
    attentions to bf16 (2^-8 of the weighted values each, and the E4M3 cache 2^-4 of every key and value: scores of
    about 1 move a weight by up to as much), and the output projection sums such errors with random signs: 2^-7 of
    the sublayer's norm bounds them, 2^-3 on E4M3."""
    ex = _example()
    dims = moe.Dims(hidden=256, experts=16, topk=4, inter=128)
    dt = torch.bfloat16 if cache == "bf16" else attn.E4M3
    n = [70, 33, 1]
    g = torch.Generator().manual_seed(3)
    x = [torch.randn((k + 1, 256), generator=g) for k in n]
    whole = ex.Decoder(1, dims, 8, 2, 64, 16, 128, 3, dt)
    cut = ex.Decoder(1, dims, 8, 2, 64, 16, 128, 3, dt)
    for dec in (whole, cut):  # the state behind the attention sublayer
        layer = dec.layers[0]
        layer.forward = lambda h, *a, _l=layer, **k: _l.attention(h, *a, **k)
    h = whole.prompt(x)
    ends = torch.tensor([k + 1 for k in n]).cumsum(0) - 1
    want = h[ends.cuda()]
    cut.prompt([t[:-1] for t in x])
    got = cut.step(torch.stack([t[-1] for t in x]).cuda())
    attn.check()
    base = torch.stack([t[-1] for t in x]).cuda()  # the sublayer's own part
    rel = ((got - want).norm(dim=1) / (want - base).norm(dim=1)).max()
    assert float(rel) <= (2.0 ** -7 if cache == "bf16" else 2.0 ** -3), float(rel)


def test_a_few_layers_and_tokens_run():
    ex = _example()
    dims = moe.Dims(hidden=256, experts=16, topk=4, inter=128)
    dec = ex.Decoder(3, dims, 4, 4, 128, 32, 256, 4, torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    h = dec.prompt([torch.randn((k, 256), generator=g) for k in (40, 5, 100, 64)])
    last = h[torch.tensor([39, 44, 144, 208]).cuda()]
    for _ in range(40):  # over several page ends
        last = dec.step(ex.rms(last, torch.ones(256, device="cuda")))
    attn.check()
    moe.check()
    assert torch.isfinite(last).all() and dec.lens == [80, 45, 140, 104]
