"""The 8-bit KV cache and the attention over a cache (csrc/kv8.hip, csrc/attn_cached.hip).

``Kv8Cache`` holds one layer's K and V as e4m3 codes [rows, heads, max_kv, head_dim] with one power-of-two scale byte
per (row, head, position) for each of K and V: (head_dim + 1) / (2 head_dim) of the bf16 cache's bytes.  ``write``
quantises new tokens into their slots, ``read`` gives slots back, ``decode`` is the single-token attention (left
padding, the beams' lineage table, shared K/V heads) and ``tree`` the attention of up to 64 drafted tokens per row.
``Kv16Cache`` is the bf16 decode cache (``[rows, heads, max_kv, head_dim]``, one layer of ``HipGPT``'s) with ``tree``.

Every call runs on the current stream of the cache's device, which must be the current device; nothing synchronises,
and every argument that changes from step to step lives on the device, so calls may be captured in a graph.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .. import _hip

_CODE = {torch.float32: _hip.F32, torch.bfloat16: _hip.BF16}


# Where tensors with unit last stride lie in memory.  A layout is (shape, strides, bytes of an element); its pieces are the runs of the
# last dim.  Layouts repeat from call to call, so what is worked out for them is kept.

@lru_cache(4096)
def _extent(shape, strides, size) -> int:
    """bytes from the first element to behind the last"""
    return size * (1 + sum((n - 1) * s for n, s in zip(shape, strides))) if 0 not in shape else 0


def _pieces(shape, strides, size) -> torch.Tensor:
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(shape[:-1], strides[:-1]):
        at = (at[:, None] + torch.arange(n) * (s * size)).reshape(-1)
    return at.sort().values


@lru_cache(4096)
def _distinct(shape, strides, size) -> bool:
    """whether no two elements share memory"""
    dims = sorted((s, n) for n, s in zip(shape[:-1], strides[:-1]) if n > 1)
    span = shape[-1]
    for s, n in dims:  # each dim steps over the ones within it: the usual case
        if s < span:
            at = _pieces(shape, strides, size)
            return bool((at[1:] - at[:-1] >= shape[-1] * size).all())
        span += (n - 1) * s
    return True


@lru_cache(4096)
def _out_extent(shape, strides, size) -> int:
    """_extent (1 for an empty tensor), 0 where elements share memory"""
    return max(_extent(shape, strides, size), 1) if _distinct(shape, strides, size) else 0


@lru_cache(4096)
def _meet(a, b, offset) -> bool:
    """whether layouts a and b share memory, b's first element ``offset`` bytes behind a's"""
    pa, pb = _pieces(*a), _pieces(*b) + offset
    la, lb = a[0][-1] * a[2], b[0][-1] * b[2]
    return bool((torch.searchsorted(pb, pa + la) > torch.searchsorted(pb, pa - lb, right=True)).any())


class _Cache:
    """What both caches share: the C view of the tensors, argument checks, the tree attention."""

    def _bind(self, k, v, k_scale, v_scale, dtype):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride():
            raise ValueError(f"k and v must be [rows, heads, max_kv, head_dim] alike, got {tuple(k.shape)} and {tuple(v.shape)}")
        rows, heads, max_kv, hd = k.shape
        if hd not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {hd}")
        if min(rows, heads, max_kv) < 1:
            raise ValueError("an empty cache")
        want = torch.uint8 if dtype == _hip.E4M3 else torch.bfloat16
        if k.dtype != want or v.dtype != want or not k.is_cuda or v.device != k.device:
            raise ValueError(f"k and v must be {want} on one GPU")
        if k.stride(3) != 1 or k.stride(2) != hd:
            raise ValueError("positions must lie one behind another (strides head_dim and 1)")
        if k_scale is not None:
            for s in (k_scale, v_scale):
                if tuple(s.shape) != (rows, heads, max_kv) or s.dtype != torch.uint8 or s.device != k.device or \
                        s.stride(2) != 1 or s.stride() != k_scale.stride():
                    raise ValueError(f"scales must be uint8 [{rows}, {heads}, {max_kv}] with unit position stride")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.rows, self.heads, self.max_kv, self.head_dim = rows, heads, max_kv, hd
        self.dev, self.index = k.device, k.get_device()
        self._c = _hip.KvCache(k.data_ptr(), v.data_ptr(), _hip.ptr(k_scale), _hip.ptr(v_scale), k.stride(0), k.stride(1),
                               0 if k_scale is None else k_scale.stride(0), 0 if k_scale is None else k_scale.stride(1),
                               rows, heads, max_kv, hd, dtype)
        self._ref = ctypes.byref(self._c)
        self.scale = hd ** -0.5
        self.lib = _hip.load()
        self._need = {}  # workspace bytes by the sizes of a call
        self._held = []  # (first byte, last + 1, layout) of the cache's tensors; a head's positions are one piece
        for t in (k, v) if k_scale is None else (k, v, k_scale, v_scale):
            layout = ((rows, heads, t[0, 0].numel()), (t.stride(0), t.stride(1), 1), t.element_size())
            self._held.append((t.data_ptr(), t.data_ptr() + _extent(*layout), layout))
        self._first, self._end = min(t[0] for t in self._held), max(t[1] for t in self._held)

    def _index(self, t: Optional[torch.Tensor], n: int, name: str) -> Optional[int]:
        if t is None:
            return None
        if t.dtype != torch.int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous() or t.get_device() != self.index:
            raise ValueError(f"{name} must be a contiguous int32 tensor of {n} on {self.dev}")
        return t.data_ptr()

    def _lineage(self, t: Optional[torch.Tensor], B: int) -> Tuple[Optional[int], int]:
        if t is None:
            if B > self.rows:
                raise ValueError(f"{B} rows over a cache of {self.rows}")
            return None, 0
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != B or t.shape[1] < self.max_kv or t.stride(1) != 1 or \
                t.get_device() != self.index:
            raise ValueError(f"kv_rows must be int32 [{B}, >= {self.max_kv}] with unit column stride on {self.dev}")
        ld = t.stride(0) if B > 1 else self.max_kv
        if 0 < ld < self.max_kv:
            raise ValueError("rows of kv_rows must not overlap (one table expanded over all rows is taken)")
        return t.data_ptr(), ld

    def _heads(self, t: torch.Tensor, shape, name: str) -> int:
        """query heads per K/V head of t [..., heads * group, head_dim]"""
        group = shape[-2] // self.heads
        if t.dtype not in _CODE or shape[-1] != self.head_dim or not group or shape[-2] != group * self.heads or \
                t.stride(-1) != 1 or t.get_device() != self.index:
            raise ValueError(f"{name} must be f32 or bf16 [..., a multiple of {self.heads} heads, {self.head_dim}] with unit "
                             f"last stride on {self.dev}, got {tuple(shape)} {t.dtype}")
        return group

    def _check_out(self, out: torch.Tensor, q: torch.Tensor, os, qs) -> None:
        """out over itself, over q (unless it is q: a column's q is read before its result is written) or over the cache"""
        shape, lo, at, size = out.shape, out.data_ptr(), q.data_ptr(), out.element_size()
        extent = _out_extent(shape, os, size)
        if not extent:
            raise ValueError("out holds the same memory twice")
        hi = lo + extent
        if at < hi and (at != lo or os != qs or q.dtype != out.dtype):
            layout = (shape, qs, q.element_size())
            same = at == lo and q.dtype == out.dtype and all(n == 1 or s == t for n, s, t in zip(shape, os, qs))
            if not same and lo < at + _extent(*layout) and _meet((shape, os, size), layout, at - lo):
                raise ValueError("out must be q itself or not overlap it")
        if lo < self._end and self._first < hi:
            for first, end, held in self._held:
                if first < hi and lo < end and _meet((shape, os, size), held, first - lo):
                    raise ValueError("out must not overlap the cache")

    def _workspace(self, B, T, group, max_len, q_dtype):
        n = self._need.get((B, T, group, max_len, q_dtype))
        if n is None:
            n = self.lib.itts_attn_cached_workspace_bytes(self._ref, B, T, group, max_len, q_dtype)
            if n < 0:
                raise ValueError("sizes the attention does not take (T <= 64, group <= 4096)")
            if len(self._need) >= 4096:
                self._need.clear()
            self._need[B, T, group, max_len, q_dtype] = n
        return torch.empty(n, dtype=torch.uint8, device=self.dev) if n else None

    def tree(self, q: torch.Tensor, kv_len: torch.Tensor, mask: torch.Tensor, n_tokens: Optional[torch.Tensor] = None,
             pad: Optional[torch.Tensor] = None, kv_rows: Optional[torch.Tensor] = None, max_len: Optional[int] = None,
             scale: Optional[float] = None, out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16):
        """Attention of drafted tokens: q [B, T, heads * group, head_dim], T <= 64, their K/V already in the cache behind
        each row's kv_len [B] accepted positions (drafted token j at position kv_len[b] + j).  mask [B, T] int64 (or [T]:
        one tree for all rows): bit j of mask[b, t] lets token t see drafted token j; every token also sees the row's
        positions pad[b] .. kv_len[b] - 1.  n_tokens [B]: drafted tokens of each row (all T if None); the outputs of the
        others stay as they are in ``out`` (zero without one).  ``out`` may be q itself; it must not overlap q otherwise, nor
        the cache.  ``tree_mask`` makes masks from parents."""
        shape = q.shape
        if len(shape) != 4:
            raise ValueError(f"q must be [B, T, heads, head_dim], got {tuple(shape)}")
        group = self._heads(q, shape, "q")
        B, T = shape[0], shape[1]
        one = mask.dim() == 1
        if mask.dtype != torch.int64 or mask.shape != ((T,) if one else (B, T)) or mask.stride(-1) != 1 and T > 1 or \
                mask.get_device() != self.index:
            raise ValueError(f"mask must be int64 [{B}, {T}] or [{T}] with unit last stride on {self.dev}")
        qs = q.stride()
        if out is None:
            out = torch.zeros(shape, dtype=dtype, device=self.dev)
            os = out.stride()
        else:
            os = out.stride()
            if out.shape != shape or os[3] != 1 or out.get_device() != self.index:
                raise ValueError(f"out must be {tuple(shape)} with unit last stride on {self.dev}")
            self._check_out(out, q, os, qs)
        qd, od = _CODE[q.dtype], _CODE.get(out.dtype)
        if od is None or od == _hip.F32 and self._c.dtype == _hip.BF16:
            raise ValueError("out must be bf16, or f32 over an 8-bit cache")
        rows, ld = self._lineage(kv_rows, B)
        longest = self.max_kv if max_len is None else int(max_len)
        ws = self._workspace(B, T, group, longest, qd)
        rc = self.lib.itts_attn_tree(
            self._ref, q.data_ptr(), qs[0], qs[1], qs[2], qd, B, T, group, self._index(kv_len, B, "kv_len"),
            self._index(pad, B, "pad"), self._index(n_tokens, B, "n_tokens"), mask.data_ptr(), 0 if one else mask.stride(0),
            rows, ld, self.scale if scale is None else float(scale), longest, out.data_ptr(), os[0], os[1], os[2], od,
            None if ws is None else ws.data_ptr(), _hip.current_stream_of(self.index))
        if rc:
            _hip.check(rc, "itts_attn_tree")
        return out


class Kv16Cache(_Cache):
    """A bf16 cache [rows, heads, max_kv, head_dim] (one layer of ``HipGPT``'s K and V); the tensors are held, not copied."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        self._bind(k, v, None, None, _hip.BF16)


class Kv8Cache(_Cache):
    """An e4m3 cache; the tensors are held, not copied (``empty`` makes them)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        self._bind(k, v, k_scale, v_scale, _hip.E4M3)

    @classmethod
    def empty(cls, rows: int, heads: int, max_kv: int, head_dim: int = 64, device="cuda:0") -> "Kv8Cache":
        codes = [torch.zeros(rows, heads, max_kv, head_dim, dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.zeros(rows, heads, max_kv, dtype=torch.uint8, device=device) for _ in range(2)]
        return cls(*codes, *scales)

    def write(self, k: torch.Tensor, v: torch.Tensor, row: torch.Tensor, pos: torch.Tensor) -> None:
        """Quantise k / v [M, heads, head_dim] (f32 or bf16, views of the c_attn output as they are) into the slots
        (row[i], pos[i]), int32 [M].  A slot outside the cache is skipped (-1 for a padding token); the slots of one
        call must differ from each other."""
        shape = k.shape
        if len(shape) != 3 or self._heads(k, shape, "k") != 1 or v.shape != shape or v.dtype != k.dtype or \
                v.stride(2) != 1 or v.get_device() != self.index:
            raise ValueError(f"k and v must be [M, {self.heads}, {self.head_dim}], alike, on {self.dev}")
        M, ks, vs = shape[0], k.stride(), v.stride()
        rc = self.lib.itts_kv8_write(self._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _CODE[k.dtype],
                                     self._index(row, M, "row"), self._index(pos, M, "pos"), M,
                                     _hip.current_stream_of(self.index))
        if rc:
            _hip.check(rc, "itts_kv8_write")

    def read(self, row: torch.Tensor, pos: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
        """(k, v) [M, heads, head_dim] of the slots (row[i], pos[i]); zeros for a slot outside the cache.  Writing what
        was read gives the same codes' values again, so an accepted path of drafted tokens moves without loss."""
        code = _CODE.get(dtype)
        if code is None or row.dim() != 1:
            raise ValueError("dtype must be f32 or bf16, row [M]")
        M, H, hd = row.numel(), self.heads, self.head_dim
        shape = (M, H, hd)
        k, v = self.k.new_empty(shape, dtype=dtype), self.k.new_empty(shape, dtype=dtype)
        rc = self.lib.itts_kv8_read(self._ref, self._index(row, M, "row"), self._index(pos, M, "pos"), M, k.data_ptr(), H * hd,
                                    hd, v.data_ptr(), H * hd, hd, code, _hip.current_stream_of(self.index))
        if rc:
            _hip.check(rc, "itts_kv8_read")
        return k, v

    def decode(self, q: torch.Tensor, kv_len: torch.Tensor, pad: Optional[torch.Tensor] = None,
               kv_rows: Optional[torch.Tensor] = None, max_len: Optional[int] = None, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """Single-token attention: q [B, heads * group, head_dim] over positions pad[b] .. kv_len[b] - 1 of each row
        (this step's K/V written before); scale defaults to head_dim ** -0.5; out bf16 or f32, q itself or apart
        from q and the cache.  kv_rows [B, >= max_kv] int32: the cache row that holds each position (beams; one table
        may be expanded over the rows).  max_len: the largest kv_len expected (the split over keys is sized by it;
        default max_kv)."""
        shape = q.shape
        if len(shape) != 3:
            raise ValueError(f"q must be [B, heads, head_dim], got {tuple(shape)}")
        group = self._heads(q, shape, "q")
        B, qs = shape[0], q.stride()
        if out is None:
            out = q.new_empty(shape, dtype=dtype)
            os = out.stride()
        else:
            os = out.stride()
            if out.shape != shape or os[2] != 1 or out.get_device() != self.index:
                raise ValueError(f"out must be {tuple(shape)} with unit last stride on {self.dev}")
            self._check_out(out, q, os, qs)
        qd, od = _CODE[q.dtype], _CODE.get(out.dtype)
        if od is None:
            raise ValueError("out must be f32 or bf16")
        rows, ld = self._lineage(kv_rows, B)
        longest = self.max_kv if max_len is None else int(max_len)
        ws = self._workspace(B, 1, group, longest, qd)
        rc = self.lib.itts_attn_decode_kv8(
            self._ref, q.data_ptr(), qs[0], qs[1], qd, B, group, self._index(kv_len, B, "kv_len"), self._index(pad, B, "pad"),
            rows, ld, self.scale if scale is None else float(scale), longest, out.data_ptr(), os[0], os[1], od,
            None if ws is None else ws.data_ptr(), _hip.current_stream_of(self.index))
        if rc:
            _hip.check(rc, "itts_attn_decode_kv8")
        return out


def tree_mask(parents: torch.Tensor) -> torch.Tensor:
    """Masks int64 [..., T] of trees given by each token's parent [..., T] (an earlier token, or -1 for the last
    accepted one): bit j of token t is set where j is t or an ancestor of t."""
    T = parents.shape[-1]
    if T > 64 or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError("at most 64 drafted tokens, parents int32 or int64")
    own = [(1 << t) - (1 << 64 if t == 63 else 0) for t in range(T)]
    mask = torch.zeros(*parents.shape[:-1], T + 1, dtype=torch.int64, device=parents.device)  # the last: no parent
    for t in range(T):
        up = torch.where((parents[..., t] >= 0) & (parents[..., t] < t), parents[..., t], T).long()
        mask[..., t] = mask.gather(-1, up[..., None])[..., 0] | own[t]
    return mask[..., :T].contiguous()
