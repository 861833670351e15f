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
import torch

from . import _lib as L
from .quant import _live

_DIMS = (64, 128, 256)


def cache(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda"):
    """A key and a value cache [pages, page, heads, dim], zeroed, each page's rows of one head together (the order that
    attend reads in the longest runs)."""
    return tuple(torch.zeros(pages, heads, page, dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))


def rope_table(positions, rot, base=1e4, device="cuda"):
    """fp32 [positions, rot]: row p the rot / 2 cosines of p base^(-2 j / rot), then the sines (angles in 64 bits)."""
    j = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * j / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _i32(name, x, shape, dev):
    if x.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if x.dim() != len(shape) or any(a < b for a, b in zip(x.shape, shape)) or x.stride(-1) != 1 or x.device != dev:
        raise ValueError(f"{name} must be at least {list(shape)} on the tensors' device, unit stride in its last dim")


def _heads(name, x, T, heads, dim, dev):
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bf16")
    if x.dim() != 3 or x.shape[0] < T or x.shape[1] != heads or x.shape[2] != dim or x.stride(2) != 1 or x.device != dev:
        raise ValueError(f"{name} must be [>= {T}, {heads}, {dim}] on the tensors' device, unit stride in its last dim")


def _cache_args(k_cache, v_cache, k_scale, v_scale):
    """(arguments of the C entries up to v_scale, e4m3, heads, dim, pages, page)"""
    dt = k_cache.dtype
    if dt not in (torch.bfloat16, torch.float8_e4m3fn) or v_cache.dtype != dt:
        raise TypeError("the caches must both be bf16 or both float8_e4m3fn")
    dev = k_cache.device
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.stride(3) != 1 or v_cache.stride(3) != 1 \
            or v_cache.device != dev:
        raise ValueError("the caches must be [pages, page, heads, dim] on one device, unit stride in dim")
    pages, page, heads, dim = k_cache.shape
    if dim not in _DIMS:
        raise ValueError(f"the heads' dim must be one of {_DIMS}")
    if page < 16 or page & (page - 1):
        raise ValueError("a page must hold a power of two of tokens, at least 16")
    e4m3 = dt != torch.bfloat16
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is None:
            continue
        if not e4m3:
            raise ValueError(f"{name}: a bf16 cache has no scales")
        if s.dtype != torch.float32 or s.numel() != heads or not s.is_contiguous() or s.device != dev:
            raise ValueError(f"{name} must be contiguous fp32 [{heads}] on the cache's device")
    ks, vs = k_cache.stride(), v_cache.stride()
    return (k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2], int(e4m3), L.ptr(k_scale),
            L.ptr(v_scale)), heads, dim, pages, page


def append(q, k, v, rope, pos, table, k_cache, v_cache, q_out, n, T, seq=None, pairs="half", k_scale=None, v_scale=None):
    """Token i (i < n[0] <= T) stands at position pos[i] of sequence seq[i] (None: sequence i): its key, rotated, and its
    value go into the cache there, its queries, rotated, into q_out[i].

    q, q_out bf16 [>= T, heads, dim] (or both None: no queries), k, v bf16 [>= T, kv heads, dim], each with unit stride in
    dim (column ranges of a projection's output will do); rope fp32 [positions, R] (rope_table; None: no rotation), R a
    multiple of 16 up to dim: the first R dims turn, in pairs (j, j + R / 2) with pairs="half" or (2 j, 2 j + 1) with
    pairs="adjacent": (a, b) -> (a cos - b sin, b cos + a sin) in fp32, rounded once to the type that is stored.  q_out may
    be q.  A token whose place is none is skipped, its q_out row untouched: a position that is negative or past the table
    or the rotations, a sequence or a page out of range.  Two tokens with one place: either's value."""
    ca, hkv, dim, pages, page = _cache_args(k_cache, v_cache, k_scale, v_scale)
    dev = k.device
    _heads("k", k, T, hkv, dim, dev)
    _heads("v", v, T, hkv, dim, dev)
    if k_cache.device != dev:
        raise ValueError("append: the cache must be on the tensors' device")
    qa, oa, hq = (None, 0, 0), (None, 0, 0), 0
    if (q is None) != (q_out is None):
        raise ValueError("append: q and q_out go together")
    if q is not None:
        hq = q.shape[1]
        _heads("q", q, T, hq, dim, dev)
        _heads("q_out", q_out, T, hq, dim, dev)
        qa, oa = (q.data_ptr(), q.stride(0), q.stride(1)), (q_out.data_ptr(), q_out.stride(0), q_out.stride(1))
    ra = (None, 0, 0, 0)
    if rope is not None:
        if rope.dtype != torch.float32:
            raise TypeError("append: rope must be fp32")
        if rope.dim() != 2 or rope.shape[1] % 16 or not 0 < rope.shape[1] <= dim or rope.stride(1) != 1 \
                or rope.device != dev:
            raise ValueError("append: rope must be [positions, R], R a multiple of 16 up to dim, unit column stride")
        ra = (rope.data_ptr(), rope.stride(0), rope.shape[0], rope.shape[1])
    if pairs not in ("half", "adjacent"):
        raise ValueError('append: pairs must be "half" or "adjacent"')
    _i32("pos", pos, (T,), dev)
    _i32("table", table, (1, 1), dev)
    if seq is not None:
        _i32("seq", seq, (T,), dev)
    n = _live(n, T, dev)
    L.call("prism_kv_append", *qa, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), *oa,
           *ra, int(pairs == "adjacent"), pos.data_ptr(), L.ptr(seq), *ca, table.data_ptr(), table.stride(0),
           table.shape[0], table.shape[1], pages, page, n.data_ptr(), T, hq, hkv, dim, L.stream_of(k))


def attend(q, k_cache, v_cache, table, lens, out, n, T, scale=None, window=0, k_scale=None, v_scale=None):
    """out[i] = softmax(scale q[i] K^T) V over the cached tokens of sequence i (i < n[0] <= T), query head h on the cache's
    head h // (heads / kv heads).  lens int32 [>= T]: tokens in the cache, the new one among them (more than the table
    holds counts as what it holds); window > 0: only the last `window` of them.  A sequence without tokens gets zeros.
    scale None: dim ** -0.5.

    q, out bf16 [>= T, heads, dim], unit stride in dim.  Softmax and sums in fp32, the weights in two bf16 parts (16 bits),
    the output rounded once.  Results do not depend on timing; how a sequence's length is split, and so the order of its
    sums, depends on the batch.  Table entries of visible tokens must name pages (others read some page, never memory
    outside the cache)."""
    ca, hkv, dim, pages, page = _cache_args(k_cache, v_cache, k_scale, v_scale)
    dev = q.device
    hq = q.shape[1] if q.dim() == 3 else 0
    _heads("q", q, T, hq, dim, dev)
    _heads("out", out, T, hq, dim, dev)
    if k_cache.device != dev:
        raise ValueError("attend: the cache must be on the tensors' device")
    if hq < hkv or hq % hkv:
        raise ValueError("attend: the query heads must be a multiple of the cache's heads")
    if window < 0:
        raise ValueError("attend: window must not be negative")
    _i32("table", table, (T, 1), dev)
    _i32("lens", lens, (T,), dev)
    n = _live(n, T, dev)
    cols = table.shape[1]
    need = L.lib().prism_kv_attend_workspace_bytes(T, hq, hkv, dim, cols, page)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None      # the caching allocator's: this stream's
    L.call("prism_kv_attend", q.data_ptr(), q.stride(0), q.stride(1), *ca, table.data_ptr(), table.stride(0), cols, pages,
           page, lens.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1), n.data_ptr(), T, hq, hkv, dim,
           dim ** -0.5 if scale is None else float(scale), int(window), L.ptr(ws), need, L.stream_of(q))
