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
import torch

from . import _lib as L
from .kv import _heads, _i32
from .quant import _live


def _args(q, k, v, g, beta, state, out, seqs, T, slots):
    dev = q.device
    if q.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [rows, heads, dim]")
    hk, dk, hv, dv = q.shape[1], q.shape[2], v.shape[1], v.shape[2]
    _heads("q", q, T, hk, dk, dev)
    _heads("k", k, T, hk, dk, dev)
    _heads("v", v, T, hv, dv, dev)
    if dk not in (64, 128) or dv not in (64, 128):
        raise ValueError("the heads' dims must be 64 or 128")
    if hk < 1 or hv < hk or hv % hk:
        raise ValueError("the value heads must be a multiple of the key heads")
    for name, x in (("g", g), ("beta", beta)):
        if x.dtype != torch.float32:
            raise TypeError(f"{name} must be fp32")
        if x.dim() != 2 or x.shape[0] < T or x.shape[1] != hv or x.stride(1) != 1 or x.device != dev:
            raise ValueError(f"{name} must be [>= {T}, {hv}] on the tensors' device, unit column stride")
    if state.dtype != torch.float32 or out.dtype != torch.float32:
        raise TypeError("state and out must be fp32")
    if state.dim() != 4 or tuple(state.shape[1:]) != (hv, dk, dv) or state.device != dev \
            or state.stride()[1:] != (dk * dv, dv, 1):
        raise ValueError(f"state must be [slots, {hv}, {dk}, {dv}] on the tensors' device, contiguous per slot")
    if out.dim() != 3 or out.shape[0] < T or tuple(out.shape[1:]) != (hv, dv) or out.stride(2) != 1 or out.device != dev:
        raise ValueError(f"out must be [>= {T}, {hv}, {dv}] on the tensors' device, unit stride in its last dim")
    if slots is not None:
        _i32("slots", slots, (seqs,), dev)
    return (q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), g.data_ptr(), g.stride(0), beta.data_ptr(), beta.stride(0), state.data_ptr(), state.stride(0),
            state.shape[0], L.ptr(slots), out.data_ptr(), out.stride(0), out.stride(1)), (hk, hv, dk, dv)


def step(q, k, v, g, beta, state, out, n, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Row i (i < n[0] <= T) is one new token of sequence i: out[i] and the state of slots[i] (module comment)."""
    args, (hk, hv, dk, dv) = _args(q, k, v, g, beta, state, out, T, T, slots)
    n = _live(n, T, q.device)
    L.call("prism_delta_step", *args, n.data_ptr(), T, hk, hv, dk, dv, int(bool(norm)),
           dk ** -0.5 if scale is None else float(scale), float(eps), L.stream_of(q))


def prefill(q, k, v, g, beta, state, out, cu, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Sequence s is rows cu[s] .. cu[s + 1] - 1 (cu int32 [sequences + 1] on the device, non-decreasing, within 0 .. T),
    continued from its state, which is left as after its last row (module comment).  A sequence may be empty; rows outside
    every sequence are untouched."""
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError("cu must be int32 [sequences + 1]")
    seqs = cu.numel() - 1
    args, (hk, hv, dk, dv) = _args(q, k, v, g, beta, state, out, seqs, T, slots)
    _i32("cu", cu, (1,), q.device)
    need = L.lib().prism_delta_prefill_workspace_bytes(T, seqs, hk, hv, dk, dv)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None     # the caching allocator's: this stream's
    L.call("prism_delta_prefill", *args, cu.data_ptr(), seqs, T, hk, hv, dk, dv, int(bool(norm)),
           dk ** -0.5 if scale is None else float(scale), float(eps), L.ptr(ws), need, L.stream_of(q))
