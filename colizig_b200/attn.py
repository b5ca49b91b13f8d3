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
be captured into a CUDA graph.  Given another stream than the current one, a call marks the
tensors it takes as used there, so that their memory is not handed out while it runs.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _abi, gpu

HEAD_DIMS = (64, 128)
E4M3 = torch.float8_e4m3fn


# A decode step is a few microseconds on the device: the checks below read each attribute
# once and build messages only when something is wrong.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_F32, _BF16, _I32, _I64 = torch.float32, torch.bfloat16, torch.int32, torch.int64


def _ready(index: int) -> None:
    """The library is up on the tensors' device (brought up there if it was not)."""
    if not gpu.available():
        gpu.init(index)
    elif gpu.device() != index:
        raise ValueError(f"tensors on cuda:{index}, the library runs on cuda:{gpu.device()}")


def _current(index: int) -> int:
    """Handle of torch's current stream on device `index`."""
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _stream(stream, index: int, tensors) -> int:
    """The stream's handle; tensors used on another stream than the current one are marked."""
    handle = getattr(stream, "cuda_stream", stream)
    if handle != _current(index):
        s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(handle, device=index)
        for t in tensors:
            if t is not None:
                t.record_stream(s)
    return handle


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(name: str, t: torch.Tensor, heads: Optional[int], dim: int, dtype, index: int):
    """Checks [rows, heads, dim] with packed heads and any 16-byte aligned row stride; returns
    (rows, heads, row stride in elements, address)."""
    shape = t.shape
    if len(shape) == 3 and t.dtype is dtype and t.get_device() == index:
        n, h, d = shape
        s0, s1, s2 = t.stride()
        if d == dim and (h == heads or heads is None) and s2 == 1 and (s1 == dim or h <= 1):
            at = t.data_ptr()
            if n <= 1:
                s0 = h * dim  # one row (or none): its stride is never used
            if s0 >= h * dim and not (s0 * (4 if dtype is _F32 else 2) | at) & 15:
                return n, h, s0, at
            raise ValueError(f"{name}: rows must be 16-byte aligned and must not overlap")
    raise ValueError(f"{name} must be {dtype} [rows, {heads if heads is not None else 'heads'}, {dim}] with packed heads "
                     f"on cuda:{index}, got {t.dtype} {tuple(shape)} (strides {t.stride()}) on {t.device}")


def _ints(name: str, t: torch.Tensor, n: int, dtype, index: int) -> int:
    shape = t.shape
    if len(shape) == 1 and shape[0] == n and t.dtype is dtype and t.get_device() == index and \
            (n <= 1 or t.stride(0) == 1):
        return t.data_ptr()
    raise ValueError(f"{name} must be a packed {dtype} tensor [{n}] on cuda:{index}, got {t.dtype} {tuple(shape)} on "
                     f"{t.device}")


def _vector(name: str, t: Optional[torch.Tensor], n: int, index: int) -> Optional[int]:
    if t is None:
        return None
    shape = t.shape
    if len(shape) == 1 and shape[0] == n and t.dtype is _F32 and t.get_device() == index and t.stride(0) == 1:
        at = t.data_ptr()
        if not at & 15:
            return at
    raise ValueError(f"{name} must be a packed, 16-byte aligned f32 [{n}] tensor on cuda:{index}, got {t.dtype} "
                     f"{tuple(shape)} on {t.device}")


def _output(name: str, t: Optional[torch.Tensor], n: int, heads: int, dim: int, bf16: torch.Tensor, index: int):
    """(t, its address), or a new tensor when t is None (bf16: any bf16 tensor of the device)."""
    if t is None:
        t = bf16.new_empty((n, heads, dim))
        return t, t.data_ptr()
    if t.dtype is not _BF16 or t.shape != (n, heads, dim) or t.get_device() != index or not t.is_contiguous() or \
            t.data_ptr() & 15:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned bf16 tensor {(n, heads, dim)} on cuda:{index}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t, t.data_ptr()


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
        self._bf16 = k if k.dtype is _BF16 else torch.empty(0, dtype=_BF16, device=k.device)
        self._c = _abi.KvCacheC(k.data_ptr(), v.data_ptr(), None if k_scale is None else k_scale.data_ptr(),
                                None if v_scale is None else v_scale.data_ptr(), strides[0], strides[1], pages, page,
                                hk, d, _abi.COLIZIG_KV_E4M3 if e4m3 else _abi.COLIZIG_KV_BF16)
        self._ref = ctypes.byref(self._c)

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
    dev, d, hk = cache._index, cache.head_dim, cache.kv_heads
    dt = _F32 if q.dtype is _F32 else _BF16
    T, hq, qs, qp = _rows("q", q, None, d, dt, dev)
    if hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads are not a multiple of {hk} key/value heads")
    tk, _, ks, kp = _rows("k", k, hk, d, dt, dev)
    tv, _, vs, vp = _rows("v", v, hk, d, dt, dev)
    if tk != T or tv != T:
        raise ValueError("q, k and v must hold the same tokens")
    sp = _ints("slots", slots, T, _I64, dev)
    rp, rlen, rot, pp = None, 0, 0, None
    if rope is not None:
        shape = rope.shape
        if len(shape) != 2 or rope.dtype is not _F32 or rope.get_device() != dev or not rope.is_contiguous() or \
                rope.data_ptr() & 15 or shape[1] % 16 or not 0 < shape[1] <= d or shape[0] < 1:
            raise ValueError(f"rope must be a contiguous f32 [positions, rot_dim] table on cuda:{dev}, rot_dim a "
                             f"multiple of 16 up to {d}")
        rlen, rot = shape
        rp = rope.data_ptr()
        pp = _ints("positions", positions, T, _I32, dev)
    qn, kn = _vector("q_norm", q_norm, d, dev), _vector("k_norm", k_norm, d, dev)
    kop = vop = None
    q_out, qop = _output("q_out", q_out, T, hq, d, cache._bf16, dev)
    if packed or k_out is not None:
        k_out, kop = _output("k_out", k_out, T, hk, d, cache._bf16, dev)
    if packed or v_out is not None:
        v_out, vop = _output("v_out", v_out, T, hk, d, cache._bf16, dev)
    handle = _current(dev) if stream is None else _stream(stream, dev, (
        q, k, v, positions, slots, rope, q_norm, k_norm, cache.k, cache.v, cache.k_scale, cache.v_scale, q_out, k_out,
        v_out))
    rc = _abi.load().colizig_cuda_attn_append(cache._ref, qp, kp, vp, 0 if dt is _F32 else 1, T, hq, qs, ks, vs, pp, sp,
                                              rp, rlen, rot, qn, kn, eps, qop, kop, vop, handle)
    if rc:
        _abi.check("colizig_cuda_attn_append", rc)
    return q_out, k_out, v_out


class DecodePlan:
    """Attention of one new token per sequence over `cache`, for up to max_batch sequences of
    q_heads query heads; scale defaults to head_dim ** -0.5.  Holds the workspace of the split
    over the cache's length, so calls of one plan must not overlap in time (one plan per
    stream)."""

    def __init__(self, cache: KvCache, q_heads: int, max_batch: int, scale: Optional[float] = None):
        _need(q_heads >= 1 and q_heads % cache.kv_heads == 0,
              f"{q_heads} query heads are not a multiple of {cache.kv_heads} key/value heads")
        _need(1 <= max_batch <= _abi.COLIZIG_ATTN_MAX_BATCH, f"max_batch must be 1..{_abi.COLIZIG_ATTN_MAX_BATCH}")
        self.cache, self.q_heads, self.max_batch = cache, q_heads, max_batch
        self.scale = cache.head_dim ** -0.5 if scale is None else float(scale)
        L = _abi.load()
        self._fn = L.colizig_cuda_attn_decode
        with torch.cuda.device(cache.device):
            self._ws = torch.zeros(L.colizig_cuda_attn_decode_workspace(), dtype=torch.uint8, device=cache.device)
        self._wsp = self._ws.data_ptr()

    def run(self, q, table, lens, out=None, stream=None):
        """out [B, q_heads, head_dim] bf16 = attention of q (bf16, row stride free) over the lens[b]
        first tokens of the pages table[b] (i32 [B, width], row stride free; lens i32 [B])."""
        c = self.cache
        dev, d, hq = c._index, c.head_dim, self.q_heads
        B, _, qs, qp = _rows("q", q, hq, d, _BF16, dev)
        if B > self.max_batch:
            raise ValueError(f"{B} sequences, the plan holds {self.max_batch}")
        shape = table.shape
        if len(shape) != 2 or shape[0] != B or shape[1] < 1 or table.dtype is not _I32 or table.get_device() != dev:
            raise ValueError(f"table must be an i32 tensor [{B}, width] on cuda:{dev}, got {table.dtype} {tuple(shape)} "
                             f"on {table.device}")
        width = shape[1]
        t0, t1 = table.stride()
        if B <= 1:
            t0 = width
        if (t1 != 1 and width > 1) or t0 < width:
            raise ValueError(f"table: rows must be packed and must not overlap, strides {table.stride()}")
        lp = _ints("lens", lens, B, _I32, dev)
        out, op = _output("out", out, B, hq, d, q, dev)
        handle = _current(dev) if stream is None else _stream(stream, dev, (
            q, table, lens, out, c.k, c.v, c.k_scale, c.v_scale, self._ws))
        rc = self._fn(c._ref, qp, qs, B, hq, table.data_ptr(), width, t0, lp, self.scale, op, self._wsp, handle)
        if rc:
            _abi.check("colizig_cuda_attn_decode", rc)
        return out


def prefill(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, out=None, stream=None):
    """Causal attention over packed prompts: sequence b holds rows cu_q[b]..cu_q[b+1] of q
    [Tq, q_heads, head_dim] and cu_k[b]..cu_k[b+1] of k, v [Tk, kv_heads, head_dim] (bf16, row
    strides free; cu i32 [B + 1], cu_k defaults to cu_q).  Queries are the last tokens of
    their sequence; a query that sees no key gives zeros; rows past the last sequence's are not written.  scale
    defaults to head_dim ** -0.5."""
    dev, d = q.get_device(), q.shape[-1]
    if dev < 0 or d not in HEAD_DIMS:
        raise ValueError(f"q must be a CUDA tensor of head_dim {HEAD_DIMS}, got {tuple(q.shape)} on {q.device}")
    _ready(dev)
    Tq, hq, qs, qp = _rows("q", q, None, d, _BF16, dev)
    Tk, hk, ks, kp = _rows("k", k, None, d, _BF16, dev)
    tv, _, vs, vp = _rows("v", v, hk, d, _BF16, dev)
    if hk < 1 or hq < 1 or hq % hk or tv != Tk:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if cu_k is None:
        cu_k = cu_q
        if Tk != Tq:
            raise ValueError("without cu_k, q and k must hold the same tokens")
    n = cu_q.shape[0]
    if n < 1:
        raise ValueError("cu_q must hold at least the leading 0")
    cq, ck = _ints("cu_q", cu_q, n, _I32, dev), _ints("cu_k", cu_k, n, _I32, dev)
    out, op = _output("out", out, Tq, hq, d, q, dev)
    handle = _current(dev) if stream is None else _stream(stream, dev, (q, k, v, cu_q, cu_k, out))
    rc = _abi.load().colizig_cuda_attn_prefill(qp, kp, vp, qs, ks, vs, Tq, Tk, n - 1, hq, hk, d, cq, ck,
                                               d ** -0.5 if scale is None else scale, op, handle)
    if rc:
        _abi.check("colizig_cuda_attn_prefill", rc)
    return out


def check(stream=None) -> None:
    """Raise if an attention call since the last check met an index outside its buffer (slot,
    position, page, length or sequence bound).  Waits for `stream` (default: the current one)."""
    handle = _current(torch.cuda.current_device()) if stream is None else getattr(stream, "cuda_stream", stream)
    _abi.check("colizig_cuda_attn_check", _abi.load().colizig_cuda_attn_check(handle))
