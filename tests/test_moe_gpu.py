"""moe.route and moe.experts on the GPU against plain 64-bit forms, and the layer as it is used: router, experts, residual."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe(dev):
    from prism_amd import moe
    return moe


@pytest.fixture(scope="module")
def fp8(dev):
    from prism_amd import fp8
    return fp8


def n_of(v, dev):
    return torch.tensor([v], dtype=torch.int32, device=dev)


def plain_route(x, top, score, bias, renorm, scale):
    """ids and weights of every row, in 64 bits, one row and one choice at a time."""
    ids, ws = torch.full((x.shape[0], top), -1, dtype=torch.int32), torch.zeros(x.shape[0], top, dtype=torch.float64)
    for t in range(x.shape[0]):
        v = x[t].double()
        p = torch.softmax(v, 0) if score == "softmax" else 1 / (1 + torch.exp(-v))
        key = v.clone() if score == "softmax" else p + (0 if bias is None else bias.double())
        key[v == -math.inf] = -math.inf
        key[v.isnan() | key.isnan()] = -math.inf
        for j in range(top):
            best = max(range(len(v)), key=lambda e: (key[e].item(), -e))
            if key[best] == -math.inf:
                break
            ids[t, j], ws[t, j] = best, p[best]
            key[best] = -math.inf
        if renorm and ids[t, 0] >= 0:
            if score == "softmax":                            # (a NaN elsewhere in the row is no part of the chosen ones)
                chosen = v[ids[t][ids[t] >= 0].long()]
                ws[t, :len(chosen)] = torch.softmax(chosen, 0)
            else:
                ws[t] /= ws[t].sum()
    return ids, ws * scale


def run_route(moe, x, top, dev, live=None, **kw):
    T = x.shape[0]
    ids = torch.full((T, top), -7, dtype=torch.int32, device=dev)
    w = torch.full((T, top), -7.0, device=dev)
    kw = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()}
    moe.route(x.to(dev), ids, w, n_of(T if live is None else live, dev), T, **kw)
    return ids.cpu(), w.cpu()


# Weights: the exponent's argument is rounded once (|x - m| up to 40 here: 40 x 2^-24), expf is good to 1 ulp (2^-23), then a sum
# of up to 1024 terms (a tree of at most 16 + 6 additions, 22 x 2^-24), a division and a product (2 x 2^-24): under 80 x 2^-24.
W_REL = 80 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,top", [(1, 1, 1), (3, 4, 4), (5, 63, 2), (9, 64, 6), (17, 65, 8), (6, 128, 8), (11, 200, 5), (4, 256, 16),
                                     (7, 512, 12), (3, 1000, 16), (2, 1024, 1)])
def test_route(moe, dev, dtype, score, T, E, top):
    g = torch.Generator().manual_seed(E + top)
    x = (3 * torch.randn(T, E, generator=g)).to(dtype)
    bias = 0.2 * torch.randn(E, generator=g) if score == "sigmoid" and E % 2 else None
    for renorm, scale in ((True, 1.0), (False, 2.5)):
        ids, w = run_route(moe, x, top, dev, score=score, bias=bias, renorm=renorm, scale=scale, live=max(1, T - 1))
        want_ids, want = plain_route(x.float(), top, score, bias, renorm, scale)
        live = max(1, T - 1)
        assert torch.equal(ids[:live], want_ids[:live])
        assert ((w[:live].double() - want[:live]).abs() <= W_REL * want[:live].abs()).all()
        assert (ids[live:] == -7).all() and (w[live:] == -7).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest(moe, dev, score):
    x = torch.randint(-2, 3, (40, 150), generator=torch.Generator().manual_seed(0)).float()
    x[0], x[1] = 0.0, -0.0
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    ids, _ = run_route(moe, x, 9, dev, score=score)
    assert torch.equal(ids, plain_route(x, 9, score, None, True, 1.0)[0])


def test_route_neighbours_in_64_bits(moe, dev):
    """Sums of sigmoid and bias that fp32 cannot tell apart."""
    x = torch.linspace(-1e-6, 1e-6, 64).repeat(3, 1)
    bias = (0.25 - 1 / (1 + torch.exp(-x[0].double()))).float()
    ids, _ = run_route(moe, x, 8, dev, score="sigmoid", bias=bias)
    assert torch.equal(ids, plain_route(x, 8, "sigmoid", bias, True, 1.0)[0])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_masked(moe, dev, score, renorm):
    """-inf and NaN logits are not chosen; rows that have fewer than top left, or none."""
    x = torch.randn(8, 70, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1] = float("nan")
    x[2, 3:] = -math.inf
    x[3, 1::2] = -math.inf
    x[4, 5] = float("nan")
    x[5] = torch.finfo(torch.float32).min
    x[6, 66:], x[6, :66] = 1.0, -math.inf
    ids, w = run_route(moe, x, 6, dev, score=score, renorm=renorm)
    want_ids, want = plain_route(x, 6, score, None, renorm, 1.0)
    assert torch.equal(ids, want_ids)
    assert (w[ids < 0] == 0).all()
    ok = want_ids >= 0
    assert torch.equal(w[ok].isnan(), want[ok].isnan())
    ok &= ~want.isnan()
    assert ((w.double() - want).abs()[ok] <= W_REL * want[ok]).all()


def test_route_strides(moe, dev):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(12, 300, generator=g)
    ids, w = torch.full((12, 9), -7, dtype=torch.int32, device=dev), torch.full((12, 11), -7.0, device=dev)
    moe.route(wide.to(dev)[:, 3:203], ids[:, 2:7], w[:, 1:6], None, 12)
    want_ids, want = plain_route(wide[:, 3:203], 5, "softmax", None, True, 1.0)
    assert torch.equal(ids.cpu()[:, 2:7], want_ids) and ((w.cpu()[:, 1:6].double() - want).abs() <= W_REL * want).all()
    assert (ids.cpu()[:, [0, 1, 7, 8]] == -7).all() and (w.cpu()[:, [0, 6, 7, 8, 9, 10]] == -7).all()


# ---------------------------------------------------------------------------------------------------------------- experts
def make(E, H, I, seed, fp8, dev):
    g = torch.Generator().manual_seed(seed)
    ws, plain = [], []
    for n, k in ((I, H), (I, H), (H, I)):
        q = (100 * torch.randn(E, n, k, generator=g)).clamp(-448, 448).to(torch.float8_e4m3fn)
        s = (0.5 + 1.5 * torch.rand(E, -(-n // 128), -(-k // 128), generator=g)) / (100 * math.sqrt(k))
        ws.append(fp8.from_rows(q.to(dev), s.to(dev)))
        plain.append(q.double() * s.double().repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k])
    return ws, plain


def plain_experts(x, ids, w, plain):
    """The layer in 64 bits, and a bound on the kernel's error of the unrounded sums: the sums of H products are off by at most
    (H / 4 + 64) 2^-24 of their terms' magnitudes (an MFMA adds its products in groups of at least four), so g and u; |silu'| <=
    1.1; silu itself, the two parts (2^-17) and the products of fp32 another 2^-16 of h; the second sums (I / 4 + 64 + top) 2^-24."""
    gate, up, down = plain
    T, H = x.shape
    E, I, _ = gate.shape
    y, tol = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    eh, ei = (H / 4 + 64) * 2.0 ** -24, (I / 4 + 64 + ids.shape[1]) * 2.0 ** -24
    for t in range(T):
        v = x[t].double()
        for j, e in enumerate(ids[t].tolist()):
            if not 0 <= e < E:
                continue
            g, u = gate[e] @ v, up[e] @ v
            dg, du = eh * (gate[e].abs() @ v.abs()), eh * (up[e].abs() @ v.abs())
            s = g / (1 + torch.exp(-g))
            h = s * u
            dh = 1.1 * dg * u.abs() + s.abs() * du + 1.1 * dg * du + 2.0 ** -16 * h.abs()
            wt = w[t, j].double()
            y[t] += wt * (down[e] @ h)
            tol[t] += wt.abs() * (down[e].abs() @ (dh + ei * h.abs()))
    return y, tol


def check(out, y, tol, epi=0, before=None):
    if epi:
        y = y + before.double()
        tol = tol + 2.0 ** -23 * y.abs() + 2.0 ** -24 * before.double().abs()
    else:
        tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * y.abs() + 2.0 ** -133
    err = (out.double() - y).abs()
    assert (err <= tol).all(), (err / tol.clamp(min=1e-300)).max()


CASES = [(1, 1, 1, 16, 16), (1, 8, 2, 128, 128), (1, 40, 8, 256, 96), (2, 3, 2, 64, 16), (5, 16, 4, 272, 160), (9, 4, 2, 144, 272),
         (16, 64, 8, 512, 128), (33, 8, 1, 160, 400), (40, 5, 5, 128, 144), (70, 300, 3, 96, 48), (128, 16, 8, 64, 80),
         (129, 4, 2, 48, 32), (300, 12, 3, 32, 144), (3, 2, 2, 2064, 1040)]


@pytest.mark.parametrize("epi", [0, 1])
@pytest.mark.parametrize("T,E,top,H,I", CASES)
def test_experts(moe, fp8, dev, T, E, top, H, I, epi):
    ws, plain = make(E, H, I, T + H, fp8, dev)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    w, ids = torch.softmax(torch.randn(T, E, generator=g), 1).topk(top, 1)
    ids = ids.int()
    live = max(1, T - T // 6)
    before = torch.randn(T, H, generator=g)
    out = before.to(dev).to(torch.float32 if epi else torch.bfloat16)
    old = out.cpu().clone()
    moe.experts(x.to(dev), ids.to(dev), w.to(dev), *ws, out, n_of(live, dev), T, epi=epi)
    y, tol = plain_experts(x[:live], ids[:live], w[:live], plain)
    check(out.cpu()[:live], y, tol, epi, before[:live])
    assert torch.equal(out.cpu()[live:], old[live:])


@pytest.mark.parametrize("T,E,top", [(1, 8, 4), (4, 8, 4), (30, 3, 16), (20, 600, 16)])
def test_experts_named_twice_or_not_at_all(moe, fp8, dev, T, E, top):
    """Ids out of range, rows without experts, an expert several times in a row."""
    H, I = 144, 48
    ws, plain = make(E, H, I, 3, fp8, dev)
    g = torch.Generator().manual_seed(E)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    ids = torch.randint(-2, E + 2, (T, top), generator=g).int()
    ids[:, -1] = ids[:, 0]
    ids[T // 2] = -1
    if T > 2:
        ids[1], ids[2] = 1, E
        ids[0, 0] = 2 ** 31 - 1
    w = torch.rand(T, top, generator=g)
    runs = []
    for _ in range(3):
        out = torch.full((T, H), 9.0, dtype=torch.bfloat16, device=dev)
        moe.experts(x.to(dev), ids.to(dev), w.to(dev), *ws, out, None, T)
        runs.append(out.cpu())
    y, tol = plain_experts(x, ids, w, plain)
    check(runs[0], y, tol)
    assert (runs[0][T // 2] == 0).all()
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


@pytest.mark.parametrize("T,E,top", [(129, 4, 4), (131, 600, 2), (140, 300, 8), (255, 20, 1)])
def test_experts_last_pass(moe, fp8, dev, T, E, top):
    """A last pass of few tokens (its pairs found in another way than the first pass's) leaves a token what it gets with other
    tokens behind it; no tensor has a row past the last."""
    H, I = 80, 48
    ws, plain = make(E, H, I, 5, fp8, dev)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(256, H, generator=g).to(torch.bfloat16)
    ids = torch.randint(0, E, (256, top), generator=g).int()
    w = torch.rand(256, top, generator=g)
    outs = []
    for rows in (T, 256):
        out = torch.zeros(rows, H, dtype=torch.bfloat16, device=dev)
        moe.experts(x[:rows].to(dev), ids[:rows].to(dev), w[:rows].to(dev), *ws, out, None, rows)
        outs.append(out.cpu())
    check(outs[0][120:], *plain_experts(x[120:T], ids[120:T], w[120:T], plain))
    assert torch.equal(outs[0], outs[1][:T])


def test_experts_all_tokens_on_one(moe, fp8, dev):
    """More tokens than a tile on one expert, the others idle."""
    E, H, I, T = 20, 128, 64, 100
    ws, plain = make(E, H, I, 4, fp8, dev)
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    ids, w = torch.full((T, 1), 13, dtype=torch.int32), torch.ones(T, 1)
    out = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
    moe.experts(x.to(dev), ids.to(dev), w.to(dev), *ws, out, None, T)
    check(out.cpu(), *plain_experts(x, ids, w, plain))


def test_experts_strides(moe, fp8, dev):
    """Rows that are column ranges of wider buffers, whose other columns hold NaN; outputs at odd places."""
    E, H, I, T, top = 6, 208, 112, 7, 2
    ws, plain = make(E, H, I, 5, fp8, dev)
    g = torch.Generator().manual_seed(6)
    x = torch.full((T, H + 24), float("nan"), dtype=torch.bfloat16)
    x[:, 8:8 + H] = torch.randn(T, H, generator=g).to(torch.bfloat16)
    ids = torch.full((T, 5), 2, dtype=torch.int32)
    ids[:, 1:3] = torch.randint(0, E, (T, top), generator=g).int()
    w = torch.full((T, 4), float("nan"))
    w[:, 2:4] = torch.rand(T, top, generator=g)
    y, tol = plain_experts(x[:, 8:8 + H], ids[:, 1:3], w[:, 2:4], plain)
    for at, width in ((0, H), (4, H + 8), (3, H + 5)):
        out = torch.full((T, width), 5.0, dtype=torch.bfloat16, device=dev)
        moe.experts(x.to(dev)[:, 8:8 + H], ids.to(dev)[:, 1:3], w.to(dev)[:, 2:4], *ws, out[:, at:at + H], None, T)
        check(out.cpu()[:, at:at + H], y, tol)
        assert (out.cpu()[:, :at] == 5).all() and (out.cpu()[:, at + H:] == 5).all()


def test_experts_not_finite(moe, fp8, dev):
    """A NaN or infinity in one token reaches no other, nor one in an expert the tokens that do not name it."""
    E, H, I, T = 4, 160, 48, 6
    ws, plain = make(E, H, I, 7, fp8, dev)
    q, s = fp8.to_rows(ws[2])
    q[3, 5, 7] = float("nan")
    ws[2] = fp8.from_rows(q, s)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    ids = torch.tensor([[0, 1], [1, 2], [3, 0], [2, 0], [1, 0], [2, 1]], dtype=torch.int32)
    w = torch.rand(T, 2, generator=g)
    y, tol = plain_experts(x, ids, w, plain)
    x[1, 9], x[4, 3] = float("nan"), math.inf
    w[5, 1] = 0
    y[5], tol[5] = (v[0] for v in plain_experts(x[5:], ids[5:], w[5:], plain))
    out = torch.zeros(T, H, dtype=torch.bfloat16, device=dev)
    moe.experts(x.to(dev), ids.to(dev), w.to(dev), *ws, out, None, T)
    got = out.cpu()
    assert got[1].isnan().all() and got[4].isnan().any() and got[2, 5].isnan()
    fine = torch.ones(T, H, dtype=torch.bool)
    fine[1], fine[4], fine[2, 5] = False, False, False
    check(got[fine], y[fine], tol[fine])


def layer(moe, fp8, h, x, logits, ws, n, T, top):
    dev = h.device
    ids, w = torch.empty(T, top, dtype=torch.int32, device=dev), torch.empty(T, top, device=dev)
    moe.route(logits, ids, w, n, T)
    moe.experts(x, ids, w, *ws, h, n, T, epi=1)


def test_layer_captured(moe, fp8, dev):
    """Router and experts into the residual, captured once and replayed with new tokens and live rows, eager calls of another
    batch between the replays; and on another stream at the same time."""
    E, H, I, T, top = 24, 256, 96, 20, 4
    ws, plain = make(E, H, I, 9, fp8, dev)
    g = torch.Generator().manual_seed(10)
    x, logits = torch.zeros(T, H, dtype=torch.bfloat16, device=dev), torch.zeros(T, E, device=dev)
    h, n = torch.zeros(T, H, device=dev), n_of(T, dev)
    layer(moe, fp8, h, x, logits, ws, n, T, top)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(moe, fp8, h, x, logits, ws, n, T, top)
    side = torch.cuda.Stream()
    for live in (T, 13, 1, T):
        x.copy_(torch.randn(T, H, generator=g))
        logits.copy_(torch.randn(T, E, generator=g))
        h0 = torch.randn(T, H, generator=g)
        h.copy_(h0)
        n.fill_(live)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            h2 = torch.zeros(3, H, device=dev)
            layer(moe, fp8, h2, x[:3].clone(), logits[:3].clone(), ws, n_of(3, dev), 3, top)
        graph.replay()
        torch.cuda.synchronize()
        ids, w = plain_route(logits.cpu(), top, "softmax", None, True, 1.0)
        y, tol = plain_experts(x.cpu(), ids, w.float(), plain)
        tol = tol + W_REL * y.abs() * 4 + 2.0 ** -20 * y.abs().amax()          # (the router's weights are the kernel's own)
        check(h.cpu()[:live], y[:live], tol[:live], 1, h0[:live])
        assert torch.equal(h.cpu()[live:], h0[live:])
        check(h2.cpu(), y[:3], tol[:3], 1, torch.zeros(3, H))


# -------------------------------------------------------------------------------- route by sigmoids that lie close or coincide
TIED = [  # logits, top, the choice by the 64-bit sigmoids
    ([14, 14, 14.0625], 1, [2]), ([16, 16, 16.125], 1, [2]), ([20, 20, 20.125], 1, [2]), ([1, 1, 1 + 2 ** -23], 1, [2]),
    ([18, 18, 18, 18, 18.125, 19], 3, [5, 4, 0]),                  # as many equal ones as are looked at, a larger one behind
    ([2, 1, 1, 1, 1, 1.0078125], 2, [0, 5]), ([-9, -9, -9, -8.9375], 2, [3, 0]), ([-30, -30, -30, -29.875], 1, [3]),
    ([40, 50, 50], 1, [0]), ([50, 40, 60, 39], 3, [0, 1, 2]),      # sigmoids that are 1 in 64 bits: the lower number
    ([-800, -750, -750, -760], 2, [0, 1]), ([-800, 3, -750], 2, [1, 0]),       # ... that are 0
    ([1e-20, 3e-20, 0, -1e-20, 1], 3, [4, 0, 1]), ([-0.0, 0, 1e-30], 1, [0]),  # ... that are 1 / 2
    ([math.inf, 45, math.inf, 44], 3, [0, 1, 2]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [0, 70, 130, 257, 700])
def test_route_close_sigmoids_without_a_bias(moe, dev, dtype, E):
    """Equal logits in front of a larger one that fp32 sigmoids cannot tell from them, and different logits whose 64-bit sigmoids
    are one number; alone and among experts far below (E: spread over so many)."""
    for x, top, want in TIED:
        v = torch.tensor(x, dtype=torch.float32)
        if not torch.equal(v.to(dtype).float(), v) and 1 + 2 ** -23 in x:
            continue                                               # (no bf16 number)
        at = torch.arange(len(x))
        if E:
            at = (at * (E // len(x))) + 1
            v = torch.full((E,), -math.inf).index_copy(0, at, v)
        rows = v.to(dtype).repeat(5, 1)
        ids, w = run_route(moe, rows, top, dev, score="sigmoid", renorm=False)
        assert torch.equal(ids, at[want].int().repeat(5, 1)), (x, top)
        assert torch.equal(ids, plain_route(rows[:1].float(), top, "sigmoid", None, False, 1.0)[0].repeat(5, 1)), (x, top)
        p = 1 / (1 + torch.exp(-rows.double()))
        want_w = torch.gather(p, 1, ids.long())
        assert ((w.double() - want_w).abs() <= W_REL * want_w + 2.0 ** -149).all(), (x, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [1, 3, 8])
@pytest.mark.parametrize("E", [8, 64, 100, 256])
def test_route_rows_full_of_ties(moe, dev, dtype, top, E):
    """Logits of a few neighbouring values, so that every choice is between equal ones and the next."""
    g = torch.Generator().manual_seed(E * top)
    base = torch.tensor([0.5, 3.0, 9.0, 14.0, 17.0, 19.0, -1.0, -12.0, -40.0])
    bits = base.view(torch.int32)[:, None] + torch.randint(0, 3, (9, E), generator=g, dtype=torch.int32) * (
        65536 if dtype == torch.bfloat16 else 1)
    x = bits.view(torch.float32)
    ids, _ = run_route(moe, x.to(dtype), top, dev, score="sigmoid")
    assert torch.equal(ids, plain_route(x, top, "sigmoid", None, True, 1.0)[0])


@pytest.mark.parametrize("live", [0, -1, -1000, -2 ** 31, -2 ** 31 + 200, 400, 2 ** 31 - 1])
def test_any_live_count(moe, fp8, dev, live):
    """Live counts below zero are none and above T are T, in every pass of a long call."""
    T, E, top, H, I = 300, 6, 2, 48, 32
    ws, plain = make(E, H, I, 13, fp8, dev)
    g = torch.Generator().manual_seed(14)
    x, logits = torch.randn(T, H, generator=g).to(torch.bfloat16), torch.randn(T, E, generator=g)
    ids, w = run_route(moe, logits, top, dev, live=live)
    out = torch.full((T, H), 9.0, dtype=torch.bfloat16, device=dev)
    want_ids, want_w = plain_route(logits, top, "softmax", None, True, 1.0)
    moe.experts(x.to(dev), want_ids.to(dev), want_w.float().to(dev), *ws, out, n_of(live, dev), T)
    if live <= 0:
        assert (ids == -7).all() and (w == -7).all() and (out == 9).all()
    else:
        assert torch.equal(ids, want_ids)
        check(out.cpu(), *plain_experts(x, want_ids, want_w.float(), plain))


def test_route_weights_that_vanish_or_are_not_finite(moe, dev):
    """What finite logits whose sigmoids are 0 in 64 bits, infinite logits and NaN ones leave, beside -inf, the mask."""
    nan, inf, low = float("nan"), math.inf, torch.finfo(torch.float32).min
    x = torch.tensor([[low, low, low, low], [-1e9, -800, -710, low], [-1e9, 0.5, low, -800], [-inf, -inf, 1, -inf], [1, nan, 2, 3],
                      [1, inf, 2, 3]])
    ids, w = run_route(moe, x, 2, dev, score="sigmoid")
    assert ids.tolist() == [[0, 1], [0, 1], [1, 0], [2, -1], [3, 2], [1, 3]]
    assert w[:2].isnan().all() and w[2].tolist() == [1, 0] and w[3].tolist() == [1, 0] and w[4:].isfinite().all()
    ids, w = run_route(moe, x, 2, dev, score="sigmoid", renorm=False)
    assert (w[:2] == 0).all() and w.isfinite().all()
    ids, w = run_route(moe, x, 2, dev)
    assert ids.tolist() == [[0, 1], [2, 1], [1, 3], [2, -1], [3, 2], [1, 3]]
    assert w[0].tolist() == [0.5, 0.5] and w[:5].isfinite().all() and w[5].isnan().all()
    ids, w = run_route(moe, x, 2, dev, renorm=False)
    assert w[0].tolist() == [0.25, 0.25] and w[:4].isfinite().all() and w[4:].isnan().all()
