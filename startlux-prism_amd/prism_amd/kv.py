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


def cache(pages, page, heads, dim, dtype=torch.bfloat16, device="cuda"):
    """A key and a value cache [pages, page, heads, dim], zeroed, each page's rows of one head together (the order that
    attend reads in the longest runs)."""
    return tuple(torch.zeros(pages, heads, page, dim, dtype=dtype, device=device).transpose(1, 2) for _ in range(2))


def rope_table(positions, rot, base=1e4, device="cuda"):
    """fp32 [positions, rot]: row p the rot / 2 cosines of p base^(-2 j / rot), then the sines (angles in 64 bits)."""
    j = torch.arange(rot // 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-2 * j / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def append(q, k, v, rope, pos, table, k_cache, v_cache, q_out, n, T, seq=None, pairs="half", k_scale=None, v_scale=None):
    """Token i (i < n[0] <= T) stands at position pos[i] of sequence seq[i] (None: sequence i): its key, rotated, and its
    value go into the cache there, its queries, rotated, into q_out[i].

    q, q_out bf16 [>= T, heads, dim] (or both None: no queries), k, v bf16 [>= T, kv heads, dim], each with unit stride in
    dim (column ranges of a projection's output will do); rope fp32 [positions, R] (rope_table; None: no rotation), R a
    multiple of 16 up to dim: the first R dims turn, in pairs (j, j + R / 2) with pairs="half" or (2 j, 2 j + 1) with
    pairs="adjacent": (a, b) -> (a cos - b sin, b cos + a sin) in fp32, rounded once to the type that is stored.  q_out may
    be q.  A token whose place is none is skipped, its q_out row untouched: a position that is negative or past the table
    or the rotations, a sequence or a page out of range.  Two tokens with one place leave a mixture of both there (each
    piece of 8 dims is one's or the other's)."""
    if n is None:
        n = _live(n, T, k.device)
    rc = (L._host or L.host()).kv_append(q, k, v, rope, pos, table, k_cache, v_cache, q_out, n, T, seq, pairs, k_scale,
                                         v_scale)
    if rc:
        L.fail("prism_kv_append", rc)


def attend(q, k_cache, v_cache, table, lens, out, n, T, scale=None, window=0, k_scale=None, v_scale=None):
    """out[i] = softmax(scale q[i] K^T) V over the cached tokens of sequence i (i < n[0] <= T), query head h on the cache's
    head h // (heads / kv heads).  lens int32 [>= T]: tokens in the cache, the new one among them (more than the table
    holds counts as what it holds); window > 0: only the last `window` of them.  A sequence without tokens gets zeros; one
    whose scores are all -inf (q . k is fp32: it overflows) NaN, as softmax gives.  scale None: dim ** -0.5.

    q, out bf16 [>= T, heads, dim], unit stride in dim.  Softmax, weights and sums in fp32 (the products take the weights
    as three bf16 parts), the output rounded once.  Results do not depend on timing; how a sequence's length is split, and
    so the order of its sums, depends on the batch.  Table entries of visible tokens must name pages (others read some
    page, never memory outside the cache)."""
    if n is None:
        n = _live(n, T, q.device)
    rc = (L._host or L.host()).kv_attend(q, k_cache, v_cache, table, lens, out, n, T, scale, window, k_scale, v_scale)
    if rc:
        L.fail("prism_kv_attend", rc)
