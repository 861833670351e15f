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

Sums, states and norms are fp32, and so are the operands of `prefill`'s products (as three bf16 parts each).  As the other
producers: outputs are the caller's buffers, calls go to torch's current stream and can be captured.
"""
from . import _lib as L
from .quant import _live


def step(q, k, v, g, beta, state, out, n, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Row i (i < n[0] <= T) is one new token of sequence i: out[i] and the state of slots[i] (module comment)."""
    if n is None:
        n = _live(n, T, q.device)
    rc = (L._host or L.host()).delta_step(q, k, v, g, beta, state, out, n, T, slots, norm, scale, eps)
    if rc:
        L.fail("prism_delta_step", rc)


def prefill(q, k, v, g, beta, state, out, cu, T, slots=None, norm=True, scale=None, eps=1e-6):
    """Sequence s is rows cu[s] .. cu[s + 1] - 1 (cu int32 [sequences + 1] on the device, non-decreasing, within 0 .. T),
    continued from its state, which is left as after its last row (module comment).  A sequence may be empty; rows outside
    every sequence are untouched.  What is not finite (an input, or a product past fp32's range) may show in the outputs of
    up to 63 earlier tokens of its sequence as well (they are computed together)."""
    rc = (L._host or L.host()).delta_prefill(q, k, v, g, beta, state, out, cu, T, slots, norm, scale, eps)
    if rc:
        L.fail("prism_delta_prefill", rc)
