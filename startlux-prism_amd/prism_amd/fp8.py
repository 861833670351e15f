"""8-bit floating point projections with block scales: e4m3 weights with one fp32 scale per block of 128 x 128, e4m3
activations with one per row and 128 inputs, the form in which fp8 checkpoints come.

    y[m, j] = sum_b a_s[m, b] w_s[j // 128, b] sum_i a[m, 128 b + i] w[j, 128 b + i]

  F8       a weight (or the experts' weights) in the device layout; pack() quantizes one, from_rows() takes a checkpoint's
           codes and scales, to_rows() gives them back
  a_q      float8_e4m3fn [>= T, 128 ceil(k / 128)], a_s fp32 [>= T, ceil(k / 128)], as quantize_act leaves them: columns from
           k on are zeros
  n        int32 [1] on the device (or None): the live rows of T, read by the kernels; other rows stay untouched

Any n and k.  As the other producers: outputs are the caller's buffers, calls go to torch's current stream and can be
captured.  The tensors must be on the current device.
"""
from typing import NamedTuple

import torch

from . import _lib as L
from .quant import _live

BLOCK = 128


class F8(NamedTuple):
    q: torch.Tensor          # uint8 [ceil(n / 16), ceil(k / 128), 2048]: 16 rows x 128 inputs as the matrix cores take them
    s: torch.Tensor          # fp32 [ceil(n / 128), ceil(k / 128)]; both with experts in front where there are several
    n: int
    k: int

    @property
    def shape(self):
        return (*self.q.shape[:-3], self.n, self.k)

    @property
    def nbytes(self):
        return self.q.numel() + 4 * self.s.numel()


def _blocks(x):
    return -(-x // BLOCK)


def pack(w: torch.Tensor) -> F8:
    """fp32 or bf16 [n, k] or [experts, n, k] on the GPU -> F8: per block of 128 x 128 the scale max(amax, 1e-10) / 448 and the
    nearest codes (ties to even)."""
    if w.dtype not in (torch.float32, torch.bfloat16) or w.dim() not in (2, 3) or 0 in w.shape:
        raise ValueError("fp8.pack: fp32 or bf16 [n, k] or [experts, n, k]")
    n, k = w.shape[-2:]
    lead = w.shape[:-2]
    q = torch.empty(*lead, -(-n // 16), _blocks(k), 2048, dtype=torch.uint8, device=w.device)
    s = torch.empty(*lead, _blocks(n), _blocks(k), dtype=torch.float32, device=w.device)
    st = L.stream_here(w)
    for src, dst, sc in zip(w, q, s) if lead else ((w, q, s),):
        src = src if src.stride(1) == 1 and src.stride(0) >= k else src.contiguous()
        L.call("prism_fp8_pack", L.ptr(src), int(w.dtype == torch.float32), src.stride(0) if n > 1 else k, L.ptr(dst), L.ptr(sc),
               n, k, st)
    return F8(q, s, n, k)


def from_rows(q: torch.Tensor, s: torch.Tensor) -> F8:
    """A checkpoint's weight, float8_e4m3fn (or its uint8 codes) [n, k] and fp32 scales [ceil(n / 128), ceil(k / 128)], or
    [experts, ...] of both, on the GPU -> F8 (a permutation, once at load)."""
    if q.dtype not in (torch.float8_e4m3fn, torch.uint8) or q.dim() not in (2, 3) or 0 in q.shape:
        raise ValueError("fp8.from_rows: q float8_e4m3fn or uint8 [n, k] or [experts, n, k]")
    n, k = q.shape[-2:]
    lead = tuple(q.shape[:-2])
    if s.dtype != torch.float32 or tuple(s.shape) != (*lead, _blocks(n), _blocks(k)) or s.device != q.device:
        raise ValueError(f"fp8.from_rows: s must be fp32 {(*lead, _blocks(n), _blocks(k))} on q's device")
    b = q.view(torch.uint8) if q.dtype != torch.uint8 else q
    pad = (-n % 16, -k % BLOCK)
    if any(pad):
        b = torch.nn.functional.pad(b, (0, pad[1], 0, pad[0]))
    b = b.reshape(-1, (n + 15) // 16, 16, _blocks(k), 2, 4, 16).permute(0, 1, 3, 4, 5, 2, 6)
    return F8(b.reshape(*lead, (n + 15) // 16, _blocks(k), 2048).contiguous(), s.clone().contiguous(), n, k)


def to_rows(w: F8):
    """F8 -> its codes float8_e4m3fn [..., n, k] and scales: the inverse of from_rows."""
    lead = tuple(w.q.shape[:-3])
    nt, kb = w.q.shape[-3:-1]
    b = w.q.reshape(-1, nt, kb, 2, 4, 16, 16).permute(0, 1, 5, 2, 3, 4, 6).reshape(*lead, nt * 16, kb * BLOCK)
    return b[..., :w.n, :w.k].contiguous().view(torch.float8_e4m3fn), w.s.clone()


def quantize_act(x, q, s, n, T):
    """x bf16 or fp32 [>= T, k] -> q, s (module comment): per row and 128 inputs the scale max(amax, 1e-10) / 448 and
    codes nearest x / scale (ties to even), both divisions rounded to fp32 as IEEE has it: bf16 inputs often lie just between
    two codes, and a scale multiplied by 1 / 448 takes the other one there.  q's columns from k on become zeros.  A NaN stays
    one; an infinity gives its 128 inputs the scale infinity, and so a NaN product."""
    if n is None:
        n = _live(n, T, x.device)
    rc = (L._host or L.host()).fp8_quant(x, q, s, n, T)
    if rc:
        L.fail("prism_fp8_quant", rc)


def gemm(a_q, a_s, w: F8, out, n, T, epi=0):
    """epi=0 writes the product, rounded once, into bf16 `out` [>= T, n]; epi=1 adds it into the fp32 residual `out`.

    A block's 128 products go through the fp8 matrix cores, which align each 8 on the largest of them with 13 bits kept below
    it: a product counts up to 2^-13 of the largest of its 8 (1.5e-5 of the result on normal values, 2-norm; bf16's rounding
    is 1.7e-3; in the fp32 residual it is what remains).  Blocks are added in fp32, in an order that depends on T and the sizes.
    a_q's rows lie on whole 16 bytes, they and a_s's at most 2^22 values apart; up to 2^22 - 1 rows."""
    if n is None:
        n = _live(n, T, a_q.device)
    rc = (L._host or L.host()).fp8_gemm(a_q, a_s, w, out, n, T, epi)
    if rc:
        L.fail("prism_fp8_gemm", rc)
