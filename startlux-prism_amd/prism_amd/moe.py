"""A mixture-of-experts feed-forward layer in serving: `route` picks each token's experts from the router's logits, `experts`
runs them, for a few tokens (a decode batch), on fp8 weights with block scales.

    out[t] = sum_j weights[t, j] down_e (silu(gate_e x_t) * (up_e x_t)),   e = ids[t, j]

  ids      int32 [>= T, top], weights fp32 [>= T, top], top up to 16
  n        int32 [1] on the device (or None): the live rows of T, read by the kernels; other rows stay untouched

As the other producers: outputs are the caller's buffers, calls go to torch's current stream and can be captured.  The tensors
must be on the current device.
"""
from . import _lib as L
from .quant import _live


def route(logits, ids, weights, n, T, score="softmax", bias=None, renorm=True, scale=1.0):
    """The top = ids.shape[1] experts of each row of logits (fp32 or bf16 [>= T, experts], up to 1024), best first, and their
    weights.  score="softmax": the largest logits, weighted by their softmax over all experts.  score="sigmoid": the largest
    sigmoid(logit) + bias (fp32 [experts] or None; compared in 64 bits), weighted by the sigmoid alone.  Of equal ones the
    lower number comes first.  renorm: the weights divided by the chosen ones' sum; then all times scale.

    An expert whose logit (or its sum with the bias) is -inf or NaN is not chosen; if fewer than top are left, the rest of the
    row is id -1 with weight 0, which `experts` passes over.  So -inf is the mask; a large negative number is a logit as others:
    sigmoids of logits below -709.8 are 0 in 64 bits, and a row whose chosen ones all are has weights 0 / 0 = NaN with renorm
    (score="softmax" has the chosen ones' softmax there).  A logit of +inf makes its row's softmax weights NaN, as does a NaN one with
    renorm=False, where the weights are softmax over all experts."""
    if n is None:
        n = _live(n, T, logits.device)
    rc = (L._host or L.host()).moe_route(logits, ids, weights, n, T, score, bias, renorm, scale)
    if rc:
        L.fail("prism_moe_route", rc)


def experts(x, ids, weights, gate, up, down, out, n, T, epi=0):
    """x bf16 [>= T, H] through the experts that ids names (numbers outside 0 .. experts - 1 take no part; a row with none
    gets zeros; one named twice counts twice).  gate, up: fp8.F8 of [experts, I, H], down of [experts, H, I]; H and I multiples
    of 16, up to 32767 experts; x's rows on whole 16 bytes, at most 2^22 values apart.  epi=0 writes bf16 `out` [>= T, H], rounded once; epi=1 adds into the fp32 residual `out`.

    Weights are multiplied as they stand for and activations as they are, sums in fp32; the hidden values enter the second
    product with 16 bits; the order of the sums depends on T and the sizes.  Made for up to 128 tokens at a time: more go through
    in passes that each read their experts (512 tokens on 8 of 128 experts take 4.6 times as long as 64)."""
    if n is None:
        n = _live(n, T, x.device)
    rc = (L._host or L.host()).moe_experts(x, ids, weights, gate, up, down, out, n, T, epi)
    if rc:
        L.fail("prism_moe_experts", rc)
