"""moe.experts in the forms that its rules choose for larger layers: two and four tiles a wave, K of a tile over two and four waves
or none, eight and sixteen columns, each with sums longer than the loads kept in flight, against 64 bits."""
import math

import pytest
import torch

from test_moe_gpu import check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe(dev):
    from prism_amd import moe
    return moe


@pytest.fixture(scope="module")
def fp8(dev):
    from prism_amd import fp8
    return fp8


def make(E, H, I, g, fp8, dev):
    """Codes and scales by name, and the packed weights."""
    rows, packed = [], []
    for n, k in ((I, H), (I, H), (H, I)):
        q = (100 * torch.randn(E, n, k, generator=g, device=dev)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s = (0.5 + 1.5 * torch.rand(E, -(-n // 128), -(-k // 128), generator=g, device=dev)) / (100 * math.sqrt(k))
        rows.append((q, s))
        packed.append(fp8.from_rows(q, s))
    return rows, packed


def plain(x, ids, w, rows):
    """The layer in 64 bits, an expert at a time, and test_moe_gpu's bound on the error of the unrounded sums: (H / 4 + 64) 2^-24 of
    the terms' magnitudes for g and u, 2^-16 of h for silu and the two parts, (I / 4 + 64 + top) 2^-24 for the second sums."""
    E, I, H = rows[0][0].shape
    y = torch.zeros(x.shape[0], H, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(y)
    eh, ei = (H / 4 + 64) * 2.0 ** -24, (I / 4 + 64 + ids.shape[1]) * 2.0 ** -24

    def wide(q, s):
        n, k = q.shape
        return q.double() * s.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    for e in range(E):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        gate, up, down = (wide(q[e], s[e]) for q, s in rows)
        v, wt = x[t].double(), w[t, j].double()[:, None]
        g, u = v @ gate.T, v @ up.T
        dg, du = eh * (v.abs() @ gate.abs().T), eh * (v.abs() @ up.abs().T)
        s = g / (1 + torch.exp(-g))
        h = s * u
        dh = 1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du + 2.0 ** -16 * h.abs()
        y.index_add_(0, t, wt * (h @ down.T))
        tol.index_add_(0, t, wt.abs() * ((dh + ei * h.abs()) @ down.abs().T))
    return y.cpu(), tol.cpu()


# (tokens, experts, top, H, I): tiles a wave and waves a tile (up; down), columns of the down kernel
FORMS = [(33, 40, 6, 2448, 272),     # 1, 4; 4, 1; 16
         (16, 40, 7, 2656, 272),     # 1, 4; 4, 1; 8
         (16, 16, 7, 3088, 784),     # 2, 4; 4, 2; 16
         (11, 16, 4, 3232, 784),     # 1, 4; 4, 2; 8
         (64, 16, 5, 3088, 272),     # 1, 4; 2, 1; 16
         (33, 64, 5, 816, 272),      # 1, 4; 2, 1; 8
         (1, 8, 2, 64, 560),         # 1, 4; 2, 2; 8
         (33, 16, 5, 528, 1552),     # 2, 2; 2, 2; 16
         (11, 8, 6, 1040, 1568),     # 2, 4; 2, 2; 16
         (130, 40, 6, 2448, 272)]    # the first again, and a pass of two tokens


@pytest.mark.parametrize("epi", [0, 1])
@pytest.mark.parametrize("T,E,top,H,I", FORMS)
def test_every_form(moe, fp8, dev, T, E, top, H, I, epi):
    g = torch.Generator(device=dev).manual_seed(T + H)
    rows, packed = make(E, H, I, g, fp8, dev)
    x = torch.randn(T, H, generator=g, device=dev).to(torch.bfloat16)
    w, ids = torch.softmax(torch.randn(T, E, generator=g, device=dev), 1).topk(top, 1)
    ids = ids.int()
    if T > 1:
        ids[T // 2, 0], ids[0, 1] = -1, E
    before = torch.randn(T, H, generator=g, device=dev)
    for live in (T, max(1, T - T // 3)):
        old = before.to(torch.float32 if epi else torch.bfloat16)
        out = old.clone()
        moe.experts(x, ids, w, *packed, out, torch.tensor([live], dtype=torch.int32, device=dev), T, epi=epi)
        y, tol = plain(x[:live], ids[:live], w[:live], rows)
        check(out.cpu()[:live], y, tol, epi, before.cpu()[:live])
        assert torch.equal(out[live:], old[live:])
