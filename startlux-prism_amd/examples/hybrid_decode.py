"""Two layers of a hybrid decoder in serving, on this library alone: one with the gated delta rule, one with attention over
a paged cache, each between Q8_0 projections.

    python startlux-prism_amd/examples/hybrid_decode.py

Prompts of several sequences go through packed in one pass, then every sequence decodes token by token in one batch.  At
the end all tokens go through once more as prompts, which has to leave the same hidden rows (up to the int8 activations'
occasional other code).  Random weights; the feed-forward halves of the layers are left out.

  linear layer     norm_q8 -> gemm [q | k | v | z | a | b] -> delta.prefill / delta.step -> gated_norm_q8 -> gemm into h
  attention layer  norm_q8 -> gemm [q | k | v] -> kv.append -> kv.attend -> rows_q8 -> gemm into h
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from prism_amd import delta, gguf_formats, kv, quant, w8a8  # noqa: E402

HID, EPS = 1024, 1e-6
HK, HV, DK, DV = 4, 8, 128, 64                # the linear layer's key and value heads
HQ, HKV, DIM, ROT = 8, 2, 128, 64             # the attention layer's heads, their dims and how many of them turn
PAGE, CTX = 16, 256                           # tokens of a page, tokens of a sequence at most


class Cfg:
    v_heads, gdn_dim, eps = HV, DV, EPS


class Layers:
    """Weights, states and cache for up to `seqs` sequences."""

    def __init__(self, seqs, dev, seed=0):
        g = torch.Generator().manual_seed(seed)

        def linear(n, k):
            q8 = gguf_formats.quantize_q8_0(torch.randn(n, k, generator=g) / k ** 0.5)
            return w8a8.weight_from_q8(q8.to(dev), 32)[0]

        def ones(n):
            return (1 + 0.1 * torch.randn(n, generator=g)).to(dev)
        self.dev = dev
        self.lin_norm, self.lin_in = ones(HID), linear(2 * HK * DK + 2 * HV * DV + 2 * HV, HID)
        self.gate_norm, self.lin_out = ones(DV), linear(HID, HV * DV)
        self.rate = (1 + 7 * torch.rand(HV, generator=g)).to(dev)
        self.att_norm, self.att_in = ones(HID), linear((HQ + 2 * HKV) * DIM, HID)
        self.att_out = linear(HID, HQ * DIM)
        self.rope = kv.rope_table(CTX, ROT, device=dev)
        self.state = torch.zeros(seqs, HV, DK, DV, device=dev)
        cols = CTX // PAGE
        self.k_cache, self.v_cache = kv.cache(seqs * cols, PAGE, HKV, DIM, device=dev)
        self.table = torch.randperm(seqs * cols, generator=g).view(seqs, cols).int().to(dev)

    def project(self, x, n, T, w, out=None, into=None):
        """int8 rows x = (q, s) through w: bf16 rows, or added to `into`."""
        if out is None and into is None:
            out = torch.empty(T, w.n, dtype=torch.bfloat16, device=self.dev)
        w8a8.gemm(*x, w, None, out if into is None else into, n, 32, epi=0 if into is None else 1)
        return out

    def rows(self, T, k):
        return torch.empty(T, k, dtype=torch.int8, device=self.dev), torch.empty(T, device=self.dev)

    def run(self, h, seq, pos, cu=None):
        """h fp32 [T, HID] -> the residual rows after both layers.  seq, pos int32 [T]: a row's sequence and position; cu
        int32 [sequences + 1]: prompts packed in the order of their sequences (None: one new token per sequence)."""
        T = h.shape[0]
        n = torch.tensor([T], dtype=torch.int32, device=self.dev)
        h = h.clone()
        # the gated delta rule
        x = self.rows(T, HID)
        quant.norm_q8(h, self.lin_norm, *x, n, T, EPS)
        p = self.project(x, n, T, self.lin_in)
        kd, vd = HK * DK, HV * DV
        q, k = p[:, :kd].unflatten(1, (HK, DK)), p[:, kd:2 * kd].unflatten(1, (HK, DK))
        v, z, at = p[:, 2 * kd:2 * kd + vd].unflatten(1, (HV, DV)), 2 * kd + vd, 2 * kd + 2 * vd
        decay = -self.rate * torch.nn.functional.softplus(p[:, at:at + HV].float() - 3)
        beta = torch.sigmoid(p[:, at + HV:at + 2 * HV].float())
        o = torch.empty(T, HV, DV, device=self.dev)
        if cu is None:
            delta.step(q, k, v, decay, beta, self.state, o, n, T, slots=seq, eps=EPS)
        else:
            delta.prefill(q, k, v, decay, beta, self.state, o, cu, T, eps=EPS)
        x = self.rows(T, vd)
        quant.gated_norm_q8(o, p, z, self.gate_norm, None, *x, n, T, Cfg)
        self.project(x, n, T, self.lin_out, into=h)
        # attention over the cache (a prompt's rows too: each sees the tokens up to its own)
        x = self.rows(T, HID)
        quant.norm_q8(h, self.att_norm, *x, n, T, EPS)
        p = self.project(x, n, T, self.att_in).unflatten(1, (HQ + 2 * HKV, DIM))
        q, k, v = p[:, :HQ], p[:, HQ:HQ + HKV], p[:, HQ + HKV:]
        kv.append(q, k, v, self.rope, pos, self.table, self.k_cache, self.v_cache, q, n, T, seq=seq)
        o = torch.empty(T, HQ, DIM, dtype=torch.bfloat16, device=self.dev)
        kv.attend(q, self.k_cache, self.v_cache, self.table[seq.long()], pos + 1, o, n, T)
        x = self.rows(T, HQ * DIM)
        quant.rows_q8(o.flatten(1), None, *x, n, T)
        self.project(x, n, T, self.att_out, into=h)
        return h


def prompts(layers, rows):
    """rows: per sequence fp32 [tokens, HID].  Returns each sequence's last hidden row."""
    lens = [r.shape[0] for r in rows]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=layers.dev)      # noqa: E731
    seq = ints([i for i, k in enumerate(lens) for _ in range(k)])
    pos = ints([t for k in lens for t in range(k)])
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return layers.run(torch.cat(rows), seq, pos, ints(cu))[[c - 1 for c in cu[1:]]]


def main(lens=(37, 5, 70), steps=6, dev=torch.device("cuda")):
    """The largest relative difference of a sequence's last hidden row between decoding and one pass."""
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn(k + steps, HID, generator=g).to(dev) for k in lens]
    a, b = Layers(len(lens), dev), Layers(len(lens), dev)
    h = prompts(a, [r[:k] for r, k in zip(rows, lens)])
    seq = torch.arange(len(lens), dtype=torch.int32, device=dev)
    pos = torch.tensor(lens, dtype=torch.int32, device=dev)
    for t in range(steps):
        h = a.run(torch.stack([r[k + t] for r, k in zip(rows, lens)]), seq, pos)
        pos += 1
    whole = prompts(b, rows)
    off = ((h - whole).norm(dim=1) / whole.norm(dim=1)).max().item()
    print(f"{len(lens)} sequences, prompts of {list(lens)} tokens, {steps} steps: last rows off by {off:.1e} at most")
    return off


if __name__ == "__main__":
    sys.exit(0 if main() < 2e-2 else 1)
