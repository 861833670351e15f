"""The paged key-value cache of a full-attention layer in serving: `append` rotates new tokens' queries and keys and
writes keys and values into the cache, `attend` is the attention of one new token per sequence over it.

  cache    two tensors [pages, page, kv heads, dim] (cache() makes a pair), bf16 or float8_e4m3fn, unit stride in dim, any
           other strides that are whole 16-byte units: rows of all heads together or a page's rows of one head together.
           page: a power of two from 16; dim: 64, 128 or 256.  An e4m3 cache may have one fp32 scale per head
           (k_scale, v_scale [kv heads]): it holds x / scale, clamped to +-448, and stands for value * scale.
  table    int32 [sequences, columns]: token t of sequence s lies in row t % page of page table[s, t // page].  Entries
           past a sequence's tokens are not read.
  n        int32 [1] on the device (or None): the live rows of T, read by the kernels; other rows stay untouched.

As the other producers: outputs are the caller's buffers, calls go to torch's current stream and can be captured.  Built
for one GPU; sharded over several, each has its own heads' cache.
"""
import functools
import struct

import torch

from . import _lib as L
from . import scratch
from .quant import _live

_DIMS = (64, 128, 256)
_BF16, _F32, _I32, _E4M3 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn

# the C entries' structs (prism_kv_append_args, prism_kv_attend_args): 19 fields of the cache, then the call's
_APPEND = struct.Struct("19q 12q 5q 5q")
_ATTEND = struct.Struct("19q 6q 4q d 2q")

_WS_BYTES = 16 << 20
_WS = scratch.Scratch(_WS_BYTES)


def cache(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda"):
    """A key and a value cache [pages, page, heads, dim], zeroed, each page's rows of one head together (the order that
    attend reads in the longest runs)."""
    return tuple(torch.zeros(pages, heads, page, dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))


def rope_table(positions, rot, base=1e4, device="cuda"):
    """fp32 [positions, rot]: row p the rot / 2 cosines of p base^(-2 j / rot), then the sines (angles in 64 bits)."""
    j = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * j / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


# The checks below return what the C entries take.  Each is one condition in the usual case (a decode-size call is bound by
# this path); what was wrong is found out after it failed.  idx: the tensors' device index (-1: host memory).
def _refuse(name, x, dtype, want, idx):
    if x.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.get_device() != idx:
        raise ValueError(f"{name} must be on the other tensors' device")
    raise ValueError(f"{name} must be {want}, unit stride in its last dim; got {list(x.shape)}, strides {x.stride()}")


def _heads(name, x, T, heads, dim, idx, dtype=_BF16):
    """(pointer, row stride, head stride) of [>= T, heads, dim]."""
    s, st = x.shape, x.stride()
    if x.dtype is not dtype or len(s) != 3 or s[0] < T or s[1] != heads or s[2] != dim or st[2] != 1 \
            or x.get_device() != idx:
        _refuse(name, x, dtype, f"[>= {T}, {heads}, {dim}]", idx)
    return x.data_ptr(), st[0] if s[0] > 1 else 0, st[1] if heads > 1 else 0


def _i32(name, x, least, idx):
    """Pointer of an int32 vector of at least `least`."""
    if x.dtype is not _I32 or x.dim() != 1 or x.numel() < least or x.get_device() != idx or (least > 1 and x.stride(0) != 1):
        _refuse(name, x, _I32, f"[>= {least}]", idx)
    return x.data_ptr()


def _table(x, rows, idx):
    """(pointer, row stride, rows, columns) of the page table."""
    s, st = x.shape, x.stride()
    if x.dtype is not _I32 or len(s) != 2 or s[0] < rows or s[1] < 1 or (s[1] > 1 and st[1] != 1) or x.get_device() != idx:
        _refuse("table", x, _I32, f"[>= {rows}, >= 1]", idx)
    return x.data_ptr(), st[0] if s[0] > 1 else s[1], s[0], s[1]


def _rows(n, T, like, idx):
    """Pointer of the live row count (with the tensor that holds it)."""
    if n is None or n.dtype is not _I32 or n.get_device() != idx:
        n = _live(n, T, like.device)
    return n, n.data_ptr()


def _scale(name, s, heads, e4m3, idx):
    if s is None:
        return 0
    if not e4m3:
        raise ValueError(f"{name}: a bf16 cache has no scales")
    if s.dtype is not _F32 or s.numel() != heads or not s.is_contiguous() or s.get_device() != idx:
        raise ValueError(f"{name} must be contiguous fp32 [{heads}] on the cache's device")
    return s.data_ptr()


def _cache_args(k, v, k_scale, v_scale, idx):
    """(the fields of prism_kv_cache before the table, kv heads, dim, pages, page)"""
    s, dt = k.shape, k.dtype
    if (dt is not _BF16 and dt is not _E4M3) or v.dtype is not dt:
        raise TypeError("the caches must both be bf16 or both float8_e4m3fn")
    ks, vs = k.stride(), v.stride()
    if len(s) != 4 or s != v.shape or ks[3] != 1 or vs[3] != 1 or k.get_device() != idx or v.get_device() != idx:
        raise ValueError("the caches must be [pages, page, heads, dim] on the tensors' device, unit stride in dim")
    pages, page, heads, dim = s
    if dim not in _DIMS:
        raise ValueError(f"the heads' dim must be one of {_DIMS}")
    if page < 16 or page & (page - 1):
        raise ValueError("a page must hold a power of two of tokens, at least 16")
    if pages < 1 or heads < 1:
        raise ValueError("the caches must not be empty")
    e4m3 = dt is _E4M3
    a, b = (1, 0) if heads > 1 else (0, 0)                       # (the stride of a single head is not used)
    c = 1 if pages > 1 else 0
    return (k.data_ptr(), ks[0] * c, ks[1], ks[2] * a, v.data_ptr(), vs[0] * c, vs[1], vs[2] * a, e4m3,
            _scale("k_scale", k_scale, heads, e4m3, idx), _scale("v_scale", v_scale, heads, e4m3, idx)), \
        heads, dim, pages, page


def append(q, k, v, rope, pos, table, k_cache, v_cache, q_out, n, T, seq=None, pairs="half", k_scale=None, v_scale=None):
    """Token i (i < n[0] <= T) stands at position pos[i] of sequence seq[i] (None: sequence i): its key, rotated, and its
    value go into the cache there, its queries, rotated, into q_out[i].

    q, q_out bf16 [>= T, heads, dim] (or both None: no queries), k, v bf16 [>= T, kv heads, dim], each with unit stride in
    dim (column ranges of a projection's output will do); rope fp32 [positions, R] (rope_table; None: no rotation), R a
    multiple of 16 up to dim: the first R dims turn, in pairs (j, j + R / 2) with pairs="half" or (2 j, 2 j + 1) with
    pairs="adjacent": (a, b) -> (a cos - b sin, b cos + a sin) in fp32, rounded once to the type that is stored.  q_out may
    be q.  A token whose place is none is skipped, its q_out row untouched: a position that is negative or past the table
    or the rotations, a sequence or a page out of range.  Two tokens with one place: either's value."""
    idx = k.get_device()
    ca, hkv, dim, pages, page = _cache_args(k_cache, v_cache, k_scale, v_scale, idx)
    ka, va = _heads("k", k, T, hkv, dim, idx), _heads("v", v, T, hkv, dim, idx)
    if q is None or q_out is None:
        if q is not q_out:
            raise ValueError("append: q and q_out go together")
        qa = oa = (0, 0, 0)
        hq = 0
    else:
        hq = q.shape[1] if q.dim() == 3 else -1
        qa, oa = _heads("q", q, T, hq, dim, idx), _heads("q_out", q_out, T, hq, dim, idx)
    if rope is None:
        ra = (0, 0, 0, 0)
    else:
        s, st = rope.shape, rope.stride()
        if rope.dtype is not _F32 or len(s) != 2 or s[1] % 16 or not 0 < s[1] <= dim or st[1] != 1 \
                or rope.get_device() != idx:
            _refuse("rope", rope, _F32, f"[positions, R], R a multiple of 16 up to {dim}", idx)
        ra = (rope.data_ptr(), st[0] if s[0] > 1 else s[1], s[0], s[1])
    if pairs != "half" and pairs != "adjacent":
        raise ValueError('append: pairs must be "half" or "adjacent"')
    ta = _table(table, 1, idx)
    n, na = _rows(n, T, k, idx)
    L.call("prism_kv_append",
           _APPEND.pack(*ca, *ta, pages, page, hkv, dim, *qa, *ka, *va, *oa, *ra, pairs == "adjacent",
                        _i32("pos", pos, T, idx), 0 if seq is None else _i32("seq", seq, T, idx), na, T, hq),
           L.stream_of(k))


_workspace_bytes = functools.lru_cache(256)(lambda *sizes: L.lib().prism_kv_attend_workspace_bytes(*sizes))


def attend(q, k_cache, v_cache, table, lens, out, n, T, scale=None, window=0, k_scale=None, v_scale=None):
    """out[i] = softmax(scale q[i] K^T) V over the cached tokens of sequence i (i < n[0] <= T), query head h on the cache's
    head h // (heads / kv heads).  lens int32 [>= T]: tokens in the cache, the new one among them (more than the table
    holds counts as what it holds); window > 0: only the last `window` of them.  A sequence without tokens gets zeros.
    scale None: dim ** -0.5.

    q, out bf16 [>= T, heads, dim], unit stride in dim.  Softmax and sums in fp32, the weights in two bf16 parts (16 bits),
    the output rounded once.  Results do not depend on timing; how a sequence's length is split, and so the order of its
    sums, depends on the batch.  Table entries of visible tokens must name pages (others read some page, never memory
    outside the cache)."""
    idx = q.get_device()
    ca, hkv, dim, pages, page = _cache_args(k_cache, v_cache, k_scale, v_scale, idx)
    hq = q.shape[1] if q.dim() == 3 else -1
    qa, oa = _heads("q", q, T, hq, dim, idx), _heads("out", out, T, hq, dim, idx)
    if hq < hkv or hq % hkv:
        raise ValueError("attend: the query heads must be a multiple of the cache's heads")
    if window < 0:
        raise ValueError("attend: window must not be negative")
    ta = _table(table, T, idx)
    la = _i32("lens", lens, T, idx)
    n, na = _rows(n, T, q, idx)
    stream = L.stream_of(q)
    need = _workspace_bytes(T, hq, hkv, dim, ta[3], page)
    ws = None
    if need:
        # two launches hand the workspace on: the stream's own scratch, or the caching allocator's memory (this stream's too)
        ws = _WS.get(q.device, False, need, stream) if need <= _WS_BYTES else None
        if ws is None:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
    (scratch.locked_call if need else L.call)(
        "prism_kv_attend",
        _ATTEND.pack(*ca, ta[0], ta[1], T, ta[3], pages, page, hkv, dim, *qa, *oa, la, na, hq, window,
                     dim ** -0.5 if scale is None else scale, 0 if ws is None else ws.data_ptr(), need), stream)
