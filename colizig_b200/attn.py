"""Attention over a paged key/value cache: what the decoder layer runs between its FP8
projections (src/qwen3moe/attn.zig:46-78 keys q/k/v/o; the projections themselves are
``fp8.matmul_fp8_keyed``).

  KvCache      the caller's cache tensors [pages, kv_heads, page_size, head_dim], bf16 or E4M3
  rope_table   cosines and sines of the position rotation, from 64-bit angles
  append       per-head norm + rotation of a step's q/k/v, keys and values into the cache
  DecodePlan   attention of one new token per sequence over the cache
  prefill      causal attention over whole prompts, packed, grouped heads
  check        raises if a call met a slot, position, page or length outside its buffer

Tensors are torch CUDA tensors on the library's device; every call is queued on `stream`
(default: torch's current stream), allocates outputs only when they are not given, and can
be captured into a CUDA graph.  Given another stream than the current one, a call allocates its
outputs there and marks the tensors it takes as used there, so that their memory is not handed
out while it runs.  Tensors that do not fit raise ValueError before anything is queued (the
checks are native code, csrc/attn_binding.cpp).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _abi, gpu

HEAD_DIMS = (64, 128)
E4M3 = torch.float8_e4m3fn


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_bound = None


def _native():
    """The native binding, given the library's entry points."""
    global _bound
    if _bound is None:
        try:
            from . import _attn_native as m
        except ImportError as e:
            raise RuntimeError("colizig_b200/_attn_native.so is missing: build it with __graft_entry__.build()") from e
        L = _abi.load()
        m.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in
                 (L.colizig_cuda_attn_append, L.colizig_cuda_attn_decode, L.colizig_cuda_attn_prefill)))
        _bound = m
    return _bound


def _ready(index: int) -> None:
    """The library is up on the tensors' device (brought up there if it was not)."""
    if not gpu.available():
        gpu.init(index)
    elif gpu.device() != index:
        raise ValueError(f"tensors on cuda:{index}, the library runs on cuda:{gpu.device()}")


def _current(index: int) -> int:
    """Handle of torch's current stream on device `index`."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _elsewhere(stream, index: int):
    """(handle, torch stream) of a given stream; the torch stream is None when it is the current one."""
    handle = getattr(stream, "cuda_stream", stream)
    if handle == _current(index):
        return handle, None
    return handle, stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(handle, device=index)


def _mark(s, *tensors) -> None:
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_cuda:
            t.record_stream(s)


def _room(s, t: Optional[torch.Tensor], like, device):
    """An output for work on stream s: given, or allocated there in `like`'s shape."""
    if t is not None or not isinstance(like, torch.Tensor):  # (what is no tensor is refused by the call itself)
        return t
    with torch.cuda.stream(s):
        return torch.empty(like.shape, dtype=torch.bfloat16, device=device)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class KvCache:
    """A paged cache held in the caller's tensors.  k and v are [pages, kv_heads, page_size,
    head_dim], bf16 or float8_e4m3fn; a page's heads are packed, pages may lie further
    apart (k and v as halves of one allocation).  k_scale / v_scale (E4M3 only, f32
    [kv_heads]): cached element = code * scale."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.device == v.device,
              "k and v must be CUDA tensors [pages, kv_heads, page_size, head_dim] of one shape")
        _ready(k.get_device())
        _need(k.dtype == v.dtype and k.dtype in (torch.bfloat16, E4M3), "the cache is bf16 or float8_e4m3fn")
        pages, hk, page, d = k.shape
        _need(d in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {d}")
        _need(page >= 16 and page % 16 == 0 and page <= 65536, f"page_size must be a multiple of 16, got {page}")
        _need(pages >= 1 and hk >= 1, "the cache is empty")
        strides = []
        for name, t in (("k", k), ("v", v)):
            st = t.stride()
            _need(st[3] == 1 and st[2] == d and (hk == 1 or st[1] == page * d), f"{name}: a page must be packed")
            stride = st[0] if pages > 1 else hk * page * d
            _need(stride >= hk * page * d and stride * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0,
                  f"{name}: pages must be 16-byte aligned and must not overlap")
            strides.append(stride)
        e4m3 = k.dtype == E4M3
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(t is None or e4m3, f"{name}: a bf16 cache takes no scales")
            _need(t is None or (t.dtype == torch.float32 and tuple(t.shape) == (hk,) and t.device == k.device and
                                t.is_contiguous()), f"{name} must be a contiguous f32 [{hk}] tensor on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, hk, page, d
        self.device, self._index = k.device, k.get_device()
        self._c = _abi.KvCacheC(k.data_ptr(), v.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
                                None if v_scale is None else v_scale.data_ptr(), strides[0], strides[1], pages, page,
                                hk, d, _abi.COLIZIG_KV_E4M3 if e4m3 else _abi.COLIZIG_KV_BF16)
        self._at = ctypes.addressof(self._c)
        self._lib = _native()

    @staticmethod
    def empty(pages: int, kv_heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16, device="cuda",
              k_scale=None, v_scale=None) -> "KvCache":
        """A cache of its own zeroed tensors."""
        shape = (pages, kv_heads, page_size, head_dim)
        z = [torch.zeros(shape, dtype=torch.uint8 if dtype == E4M3 else dtype, device=device) for _ in range(2)]
        k, v = (t.view(E4M3) for t in z) if dtype == E4M3 else z
        return KvCache(k, v, k_scale, v_scale)


def rope_table(positions: int, rot_dim: int, theta: float = 1e6, device="cuda") -> torch.Tensor:
    """f32 [positions, rot_dim]: rot_dim/2 cosines, then rot_dim/2 sines of position * theta^(-2i/rot_dim),
    the angles in 64 bits."""
    inv = float(theta) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def append(cache: KvCache, q, k, v, positions, slots, rope=None, q_norm=None, k_norm=None, eps: float = 1e-6,
           packed: bool = False, q_out=None, k_out=None, v_out=None, stream=None):
    """Norm (when q_norm / k_norm f32 [head_dim] are given) and rotation (rope: ``rope_table``) of
    a step's projections q [T, q_heads, head_dim], k and v [T, kv_heads, head_dim] (f32 or bf16,
    slices of a fused projection as they are; no output may overlap them); k and v go to cache row slots[t] (i64; page *
    page_size + row, negative: not cached, no slot twice), positions i32 [T].  Returns (q, k, v)
    packed in bf16; k and v (what ``prefill`` reads) are None unless packed or given."""
    dev = cache._index
    _ready(dev)
    if stream is None:
        handle = _current(dev)
    else:
        handle, s = _elsewhere(stream, dev)
        if s is not None:
            _mark(s, q, k, v, positions, slots, rope, q_norm, k_norm, cache.k, cache.v, cache.k_scale, cache.v_scale, q_out,
                  k_out, v_out)
            q_out = _room(s, q_out, q, cache.device)
            k_out = _room(s, k_out, k, cache.device) if packed else k_out
            v_out = _room(s, v_out, v, cache.device) if packed else v_out
    r = cache._lib.append(cache._at, dev, q, k, v, positions, slots, rope, q_norm, k_norm, eps, packed, q_out, k_out, v_out,
                          handle)
    if r.__class__ is int:
        _abi.check("colizig_cuda_attn_append", r)
    return r


class DecodePlan:
    """Attention of one new token per sequence over `cache`, for up to max_batch sequences of
    q_heads query heads; scale defaults to head_dim ** -0.5.  Holds the workspace of the split
    over the cache's length, so calls of one plan must not overlap in time (one plan per
    stream).  Making a plan waits for the current stream."""

    def __init__(self, cache: KvCache, q_heads: int, max_batch: int, scale: Optional[float] = None):
        _need(q_heads >= 1 and q_heads % cache.kv_heads == 0,
              f"{q_heads} query heads are not a multiple of {cache.kv_heads} key/value heads")
        _need(1 <= max_batch <= _abi.COLIZIG_ATTN_MAX_BATCH, f"max_batch must be 1..{_abi.COLIZIG_ATTN_MAX_BATCH}")
        self.cache, self.q_heads, self.max_batch = cache, q_heads, max_batch
        self.scale = cache.head_dim ** -0.5 if scale is None else float(scale)
        with torch.cuda.device(cache.device):
            self._ws = torch.zeros(_abi.load().colizig_cuda_attn_decode_workspace(), dtype=torch.uint8,
                                   device=cache.device)
            # the zeros have landed before a call on any stream starts counting in them
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        self._wsp, self._home = self._ws.data_ptr(), _current(cache._index)

    def run(self, q, table, lens, out=None, stream=None):
        """out [B, q_heads, head_dim] bf16 = attention of q (bf16, row stride free) over the lens[b]
        first tokens of the pages table[b] (i32 [B, width], row stride free; lens i32 [B])."""
        c = self.cache
        dev = c._index
        _ready(dev)
        handle, s = (_current(dev), None) if stream is None else _elsewhere(stream, dev)
        if s is not None:
            _mark(s, q, table, lens, out, c.k, c.v, c.k_scale, c.v_scale, self._ws)
            out = _room(s, out, q, c.device)
        elif handle != self._home:  # the plan may be dropped while the call runs
            self._ws.record_stream(torch.cuda.current_stream(dev))
        r = c._lib.decode(c._at, dev, self.q_heads, self.max_batch, self.scale, self._wsp, q, table, lens, out, handle)
        if r.__class__ is int:
            _abi.check("colizig_cuda_attn_decode", r)
        return r


def prefill(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, out=None, stream=None):
    """Causal attention over packed prompts: sequence b holds rows cu_q[b]..cu_q[b+1] of q
    [Tq, q_heads, head_dim] and cu_k[b]..cu_k[b+1] of k, v [Tk, kv_heads, head_dim] (bf16, row
    strides free; cu i32 [B + 1], cu_k defaults to cu_q).  Queries are the last tokens of
    their sequence; a query that sees no key gives zeros; rows past the last sequence's are not written.  scale
    defaults to head_dim ** -0.5."""
    if not isinstance(q, torch.Tensor):
        raise ValueError(f"q must be a tensor, got {type(q).__name__}")
    dev = q.get_device()
    if dev < 0:
        raise ValueError(f"q must be a CUDA tensor, got one on {q.device}")
    _ready(dev)
    if scale is None:
        scale = q.shape[2] ** -0.5 if q.dim() == 3 and q.shape[2] else 1.0  # (other shapes are refused below)
    if stream is None:
        handle = _current(dev)
    else:
        handle, s = _elsewhere(stream, dev)
        if s is not None:
            _mark(s, q, k, v, cu_q, cu_k, out)
            out = _room(s, out, q, q.device)
    r = _native().prefill(dev, q, k, v, cu_q, cu_k, scale, out, handle)
    if r.__class__ is int:
        _abi.check("colizig_cuda_attn_prefill", r)
    return r


def check(stream=None) -> None:
    """Raise if an attention call since the last check met an index outside its buffer (slot,
    position, page, length or sequence bound).  Waits for `stream` (default: the current one of the library's
    device)."""
    handle = _current(gpu.device()) if stream is None else getattr(stream, "cuda_stream", stream)
    _abi.check("colizig_cuda_attn_check", _abi.load().colizig_cuda_attn_check(handle))
