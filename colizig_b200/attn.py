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


def _ready() -> None:
    if not gpu.available():
        gpu.init()


def _stream(stream, tensors) -> int:
    """The stream's handle; tensors used on another stream than the current one are marked."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    handle = getattr(stream, "cuda_stream", stream)
    if handle != torch.cuda.current_stream().cuda_stream:
        s = stream if isinstance(stream, torch.cuda.Stream) else torch.cuda.ExternalStream(handle)
        for t in tensors:
            if t is not None:
                t.record_stream(s)
    return handle


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _rows(name: str, t: torch.Tensor, heads: Optional[int], dim: int, dtypes, device) -> int:
    """Checks [rows, heads, dim] with packed heads and any 16-byte aligned row stride;
    returns the row stride in elements."""
    shape, st = t.shape, t.stride()
    if not (len(shape) == 3 and shape[2] == dim and (heads is None or shape[1] == heads)):
        raise ValueError(f"{name} must be [rows, {heads if heads is not None else 'heads'}, {dim}], got {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {dtypes}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    row = shape[1] * dim
    if st[2] != 1 or (shape[1] > 1 and st[1] != dim):
        raise ValueError(f"{name}: heads of a row must be packed")
    stride = st[0] if shape[0] > 1 else row  # one row (or none): its stride is never used
    if stride < row or (stride * t.element_size()) & 15 or t.data_ptr() & 15:
        raise ValueError(f"{name}: rows must be 16-byte aligned and must not overlap")
    return stride


def _ints(name: str, t: torch.Tensor, shape, dtype, device) -> int:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _vector(name: str, t: Optional[torch.Tensor], n: int, device) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != (n,) or t.device != device or t.stride(0) != 1 or \
            t.data_ptr() & 15:
        raise ValueError(f"{name} must be a packed, 16-byte aligned f32 [{n}] tensor on {device}")
    return t.data_ptr()


def _output(name: str, t: Optional[torch.Tensor], shape, like: torch.Tensor) -> torch.Tensor:
    if t is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=like.device)
    if t.dtype != torch.bfloat16 or tuple(t.shape) != tuple(shape) or t.device != like.device or \
            not t.is_contiguous() or t.data_ptr() & 15:
        raise ValueError(f"{name} must be a contiguous, 16-byte aligned bf16 tensor {tuple(shape)} on {like.device}")
    return t


class KvCache:
    """A paged cache held in the caller's tensors.  k and v are [pages, kv_heads, page_size,
    head_dim], bf16 or float8_e4m3fn; a page's heads are packed, pages may lie further
    apart (k and v as halves of one allocation).  k_scale / v_scale (E4M3 only, f32
    [kv_heads]): cached element = code * scale."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        _ready()
        _need(k.is_cuda and k.dim() == 4 and k.shape == v.shape and k.device == v.device,
              "k and v must be CUDA tensors [pages, kv_heads, page_size, head_dim] of one shape")
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
        self.device = k.device
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
    slices of a fused projection as they are); k and v go to cache row slots[t] (i64; page *
    page_size + row, negative: not cached, no slot twice), positions i32 [T].  Returns (q, k, v)
    packed in bf16; k and v (what ``prefill`` reads) are None unless packed or given."""
    dev, d, hk = cache.device, cache.head_dim, cache.kv_heads
    dts = (q.dtype,) if q.dtype in (torch.float32, torch.bfloat16) else (torch.float32, torch.bfloat16)
    qs = _rows("q", q, None, d, dts, dev)
    T, hq = q.shape[0], q.shape[1]
    if hq < 1 or hq % hk:
        raise ValueError(f"{hq} query heads are not a multiple of {hk} key/value heads")
    ks = _rows("k", k, hk, d, dts, dev)
    vs = _rows("v", v, hk, d, dts, dev)
    if k.shape[0] != T or v.shape[0] != T:
        raise ValueError("q, k and v must hold the same tokens")
    sp = _ints("slots", slots, (T,), torch.int64, dev)
    rp, rlen, rot, pp = None, 0, 0, None
    if rope is not None:
        rlen, rot = rope.shape
        if rope.dtype != torch.float32 or rope.device != dev or not rope.is_contiguous() or rope.data_ptr() & 15 or \
                rot % 16 or not 0 < rot <= d or rlen < 1:
            raise ValueError(f"rope must be a contiguous f32 [positions, rot_dim] table on {dev}, rot_dim a multiple "
                             f"of 16 up to {d}")
        pp = _ints("positions", positions, (T,), torch.int32, dev)
        rp = rope.data_ptr()
    qn, kn = _vector("q_norm", q_norm, d, dev), _vector("k_norm", k_norm, d, dev)
    handle = _stream(stream, (q, k, v, positions, slots, rope, q_norm, k_norm, cache.k, cache.v, cache.k_scale,
                              cache.v_scale, q_out, k_out, v_out)) if stream is not None else \
        torch.cuda.current_stream().cuda_stream
    q_out = _output("q_out", q_out, (T, hq, d), q)
    if packed or k_out is not None:
        k_out = _output("k_out", k_out, (T, hk, d), q)
    if packed or v_out is not None:
        v_out = _output("v_out", v_out, (T, hk, d), q)
    if stream is not None:
        _stream(stream, (q_out, k_out, v_out))
    rc = _abi.load().colizig_cuda_attn_append(
        cache._ref, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        _abi.COLIZIG_X_BF16 if q.dtype == torch.bfloat16 else _abi.COLIZIG_X_F32, T, hq, qs, ks, vs, pp, sp, rp, rlen,
        rot, qn, kn, eps, q_out.data_ptr(), None if k_out is None else k_out.data_ptr(),
        None if v_out is None else v_out.data_ptr(), handle)
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

    def run(self, q, table, lens, out=None, stream=None):
        """out [B, q_heads, head_dim] bf16 = attention of q (bf16, row stride free) over the lens[b]
        first tokens of the pages table[b] (i32 [B, width], row stride free; lens i32 [B])."""
        c = self.cache
        qs = _rows("q", q, self.q_heads, c.head_dim, (torch.bfloat16,), c.device)
        B = q.shape[0]
        if B > self.max_batch:
            raise ValueError(f"{B} sequences, the plan holds {self.max_batch}")
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or table.device != c.device or \
                table.shape[1] < 1 or table.stride(1) != 1 or (B > 1 and table.stride(0) < table.shape[1]):
            raise ValueError(f"table must be an i32 tensor [{B}, width] on {c.device}, got {table.dtype} "
                             f"{tuple(table.shape)}")
        lp = _ints("lens", lens, (B,), torch.int32, c.device)
        if stream is None:
            handle = torch.cuda.current_stream().cuda_stream
        else:
            handle = _stream(stream, (q, table, lens, out, c.k, c.v, c.k_scale, c.v_scale, self._ws))
        out = _output("out", out, (B, self.q_heads, c.head_dim), q)
        if stream is not None:
            _stream(stream, (out,))
        rc = self._fn(c._ref, q.data_ptr(), qs, B, self.q_heads, table.data_ptr(), table.shape[1],
                      table.stride(0) if B > 1 else table.shape[1], lp, self.scale, out.data_ptr(),
                      self._ws.data_ptr(), handle)
        if rc:
            _abi.check("colizig_cuda_attn_decode", rc)
        return out


def prefill(q, k, v, cu_q, cu_k=None, scale: Optional[float] = None, out=None, stream=None):
    """Causal attention over packed prompts: sequence b holds rows cu_q[b]..cu_q[b+1] of q
    [Tq, q_heads, head_dim] and cu_k[b]..cu_k[b+1] of k, v [Tk, kv_heads, head_dim] (bf16, row
    strides free; cu i32 [B + 1], cu_k defaults to cu_q).  Queries are the last tokens of
    their sequence; a query that sees no key gives zeros.  scale defaults to head_dim ** -0.5."""
    _ready()
    dev = q.device
    d = q.shape[-1]
    if not q.is_cuda or d not in HEAD_DIMS:
        raise ValueError(f"q must be a CUDA tensor of head_dim {HEAD_DIMS}, got {tuple(q.shape)} on {dev}")
    bf = (torch.bfloat16,)
    qs = _rows("q", q, None, d, bf, dev)
    ks = _rows("k", k, None, d, bf, dev)
    hq, hk = q.shape[1], k.shape[1]
    vs = _rows("v", v, hk, d, bf, dev)
    if hk < 1 or hq < 1 or hq % hk or v.shape[0] != k.shape[0]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if cu_k is None:
        cu_k = cu_q
        if k.shape[0] != q.shape[0]:
            raise ValueError("without cu_k, q and k must hold the same tokens")
    n = cu_q.shape[0]
    if n < 1:
        raise ValueError("cu_q must hold at least the leading 0")
    cq, ck = _ints("cu_q", cu_q, (n,), torch.int32, dev), _ints("cu_k", cu_k, (n,), torch.int32, dev)
    handle = torch.cuda.current_stream().cuda_stream if stream is None else _stream(stream, (q, k, v, cu_q, cu_k, out))
    out = _output("out", out, (q.shape[0], hq, d), q)
    if stream is not None:
        _stream(stream, (out,))
    rc = _abi.load().colizig_cuda_attn_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks, vs, q.shape[0],
                                               k.shape[0], n - 1, hq, hk, d, cq, ck,
                                               d ** -0.5 if scale is None else scale, out.data_ptr(), handle)
    if rc:
        _abi.check("colizig_cuda_attn_prefill", rc)
    return out


def check(stream=None) -> None:
    """Raise if an attention call since the last check met an index outside its buffer (slot,
    position, page, length or sequence bound).  Waits for `stream` (default: the current one)."""
    handle = torch.cuda.current_stream().cuda_stream if stream is None else getattr(stream, "cuda_stream", stream)
    _abi.check("colizig_cuda_attn_check", _abi.load().colizig_cuda_attn_check(handle))
