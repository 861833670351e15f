"""The gated delta rule of a linear-attention layer in serving: `step` for one new token per sequence (the recurrent
form), `prefill` for whole prompts packed one after the other (chunks on the matrix cores).

Per value head, with its state S fp32 [dk, dv], a = exp(g), key k and query q of key head h // (value heads / key heads):

    S <- a S;   u = beta (v - S^T k);   S <- S + k u^T;   o = S^T q

  norm=True   k <- k / sqrt(|k|^2 + eps), q <- q / sqrt(|q|^2 + eps) first; q is then multiplied by scale (None:
              dk ** -0.5) either way
  q, k        bf16 [>= T, key heads, dk]; v bf16 [>= T, value heads, dv]: unit stride in the last dim, so column ranges of a
              projection's output will do; dk, dv 64 or 128
  g, beta     fp32 [>= T, value heads]: the decay's logarithm (<= 0; -inf clears the state) and the update's strength
  state       fp32 [slots, value heads, dk, dv], updated in place; slots int32: the state of each sequence (None: its own
              number).  A sequence with a slot out of range is skipped, its rows of out untouched; two sequences
              must not share a slot in one call.
  out         fp32 [>= T, value heads, dv], what quant.gated_norm_q8 / gated_norm_g read

Sums, states and norms are fp32 throughout.  As the other producers: outputs are the caller's buffers, calls go to torch's
current stream and can be captured.
"""
import functools
import struct

import torch

from . import _lib as L
from .kv import _F32, _heads, _i32, _refuse, _rows

_ARGS = struct.Struct("9q 4q 4q 3q q 7q 2d 2q")                   # prism_delta_args


def _gate(name, x, T, hv, idx):
    """(pointer, row stride) of fp32 [>= T, hv]."""
    s, st = x.shape, x.stride()
    if x.dtype is not _F32 or len(s) != 2 or s[0] < T or s[1] != hv or (st[1] != 1 and hv > 1) or x.get_device() != idx:
        _refuse(name, x, _F32, f"[>= {T}, {hv}]", idx)
    return x.data_ptr(), st[0]


def _args(q, k, v, g, beta, state, out, seqs, T, slots):
    """(the fields of prism_delta_args up to out, its sizes)"""
    idx = q.get_device()
    if q.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [rows, heads, dim]")
    _, hk, dk = q.shape
    _, hv, dv = v.shape
    qa, ka, va = _heads("q", q, T, hk, dk, idx), _heads("k", k, T, hk, dk, idx), _heads("v", v, T, hv, dv, idx)
    if (dk != 64 and dk != 128) or (dv != 64 and dv != 128):
        raise ValueError("the heads' dims must be 64 or 128")
    if hk < 1 or hv < hk or hv % hk:
        raise ValueError("the value heads must be a multiple of the key heads")
    ga, ba = _gate("g", g, T, hv, idx), _gate("beta", beta, T, hv, idx)
    s, st = state.shape, state.stride()
    if state.dtype is not _F32 or len(s) != 4 or s[1] != hv or s[2] != dk or s[3] != dv or st[3] != 1 or st[2] != dv \
            or (st[1] != dk * dv and hv > 1) or state.get_device() != idx:
        _refuse("state", state, _F32, f"[slots, {hv}, {dk}, {dv}], contiguous per slot", idx)
    oa = _heads("out", out, T, hv, dv, idx, _F32)
    return (*qa, *ka, *va, *ga, *ba, state.data_ptr(), st[0] if s[0] > 1 else hv * dk * dv, s[0],
            0 if slots is None else _i32("slots", slots, seqs, idx), *oa), (hk, hv, dk, dv), idx


def step(q, k, v, g, beta, state, out, n, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Row i (i < n[0] <= T) is one new token of sequence i: out[i] and the state of slots[i] (module comment)."""
    args, sizes, idx = _args(q, k, v, g, beta, state, out, T, T, slots)
    n, na = _rows(n, T, q, idx)
    L.call("prism_delta_step",
           _ARGS.pack(*args, na, 0, T, *sizes, bool(norm), sizes[2] ** -0.5 if scale is None else scale, eps, 0, 0),
           L.stream_of(q))


_workspace_bytes = functools.lru_cache(256)(lambda *sizes: L.lib().prism_delta_prefill_workspace_bytes(*sizes))


def prefill(q, k, v, g, beta, state, out, cu, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Sequence s is rows cu[s] .. cu[s + 1] - 1 (cu int32 [sequences + 1] on the device, non-decreasing, within 0 .. T),
    continued from its state, which is left as after its last row (module comment).  A sequence may be empty; rows outside
    every sequence are untouched.  A value that is not finite may show in the outputs of up to 63 earlier tokens of its
    sequence as well (they are computed together)."""
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError("cu must be int32 [sequences + 1]")
    seqs = cu.numel() - 1
    args, sizes, idx = _args(q, k, v, g, beta, state, out, seqs, T, slots)
    need = _workspace_bytes(T, seqs, *sizes)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None     # the caching allocator's: this stream's
    L.call("prism_delta_prefill",
           _ARGS.pack(*args, _i32("cu", cu, seqs + 1, idx), seqs, T, *sizes, bool(norm),
                      sizes[2] ** -0.5 if scale is None else scale, eps, 0 if ws is None else ws.data_ptr(), need),
           L.stream_of(q))
