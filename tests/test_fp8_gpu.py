"""fp8.quantize_act, pack, from_rows and gemm on the GPU against plain 64-bit forms.

Quantizers are exact: the same IEEE division and rounding as torch's.  The product is exact on small integers with power-of-two
scales (every product and sum then is an integer multiple of one unit below 2^24, and no product is more than 2^13 times smaller
than another); on normal values its 2-norm error is bounded by bf16's half step 2^-8 and, per product, by 2^-13 of the largest of
its group of 8 (the MFMA's alignment): 8 products of a group are off by at most 8 x 2^-13 max, and the largest of 8 products is at
most their root sum of squares, so by 2^-10 of the groups' 2-norm."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fp8(dev):
    from prism_amd import fp8
    return fp8


def n_of(v, dev):
    return torch.tensor([v], dtype=torch.int32, device=dev)


def kb(k):
    return -(-k // 128)


def plain_quant(x, k):
    p = torch.zeros(x.shape[0], kb(k) * 128)
    p[:, :k] = x.float()
    b = p.unflatten(1, (-1, 128))
    s = b.abs().amax(2).clamp(min=1e-10) / 448
    return (b / s[..., None]).flatten(1).to(E4), s


def codes(q):
    return q.cpu().view(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,live,k", [(1, 1, 1), (1, 1, 128), (3, 2, 5), (7, 7, 127), (5, 4, 130), (70, 61, 136), (4, 4, 1000),
                                         (300, 257, 2560), (2100, 2100, 2048), (1, 0, 64)])
def test_quantize_is_exact(fp8, dev, dtype, rows, live, k):
    g = torch.Generator().manual_seed(rows * 1000 + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, : k // 2] = 0
    q = torch.full((rows, kb(k) * 128), 1.0, device=dev).to(E4)
    s = torch.full((rows, kb(k)), -1.0, device=dev)
    fp8.quantize_act(x.to(dev), q, s, n_of(live, dev), rows)
    wq, ws = plain_quant(x, k)
    assert torch.equal(s.cpu()[:live], ws[:live]) and (s.cpu()[live:] == -1).all()
    assert torch.equal(codes(q)[:live], codes(wq)[:live]) and (q.float().cpu()[live:] == 1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_ties_and_edges(fp8, dev, dtype):
    """Quotients on and beside the codes' midpoints (amax 448: scale 1), subnormal codes, zeros, the floor of the scale."""
    vals = [448.0] + [c + d for c in (1.0625, 1.1875, 17.0, 416.0, 2 ** -9, 1.5 * 2 ** -9, 2 ** -10, 3 * 2 ** -10)
                      for d in (0, 2 ** -18, -2 ** -18)]
    x = torch.zeros(6, 256)
    x[0, :len(vals)] = torch.tensor(vals)
    x[1] = -x[0]
    x[2, :128] = 1e-12
    x[3, 128:] = torch.linspace(-448, 448, 128)
    x[4, 0] = 3.3e38
    x[5, :128] = torch.linspace(-3, 3, 128)
    x = x.to(dtype)
    q, s = torch.zeros(6, 256, device=dev).to(E4), torch.zeros(6, 2, device=dev)
    fp8.quantize_act(x.to(dev), q, s, None, 6)
    wq, ws = plain_quant(x, 256)
    assert torch.equal(s.cpu(), ws) and torch.equal(codes(q), codes(wq))


def test_quantize_not_finite(fp8, dev):
    """A NaN is a NaN code, its neighbours as without it; an infinity gives its block the scale infinity; no other block or row
    sees either."""
    x = torch.randn(4, 384, generator=torch.Generator().manual_seed(0))
    y = x.clone()
    y[1, 5], y[2, 200] = float("nan"), float("inf")
    out = []
    for v in (x, y):
        q, s = torch.zeros(4, 384, device=dev).to(E4), torch.zeros(4, 3, device=dev)
        fp8.quantize_act(v.to(dev), q, s, None, 4)
        out.append((codes(q), s.cpu(), q.float().cpu()))
    (q0, s0, _), (q1, s1, f1) = out
    same = torch.ones(4, 384, dtype=torch.bool)
    same[1, 5] = False
    same[2, 128:256] = False
    assert torch.equal(q0[same], q1[same]) and f1[1, 5].isnan()
    assert s1[2, 1] == float("inf") and torch.equal(s0[[0, 1, 3]], s1[[0, 1, 3]])
    assert (f1[2, 128:256] * s1[2, 1]).isnan().all()


def test_quantize_strides(fp8, dev):
    """A column range of wider rows, misaligned ones among them; outputs in wider buffers, whose other columns stay."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(9, 700, generator=g).to(torch.bfloat16)
    for at in (0, 8, 3):
        x = wide[:, at:at + 264]
        q, s = torch.zeros(9, 512, device=dev).to(E4), torch.full((9, 5), 7.0, device=dev)
        fp8.quantize_act(wide.to(dev)[:, at:at + 264], q[:, 64:448], s[:, 1:4], None, 9)
        wq, ws = plain_quant(x, 264)
        assert torch.equal(codes(q)[:, 64:448], codes(wq)) and torch.equal(s.cpu()[:, 1:4], ws)
        assert (codes(q)[:, :64] == 0).all() and (codes(q)[:, 448:] == 0).all() and (s.cpu()[:, [0, 4]] == 7).all()


@pytest.mark.parametrize("shape", [(1, 1), (16, 128), (17, 129), (128, 128), (200, 300), (3, 50, 260)])
def test_weights_there_and_back(fp8, dev, shape):
    g = torch.Generator().manual_seed(sum(shape))
    n, k = shape[-2:]
    q = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    s = torch.randn(*shape[:-2], kb(n), kb(k), generator=g)
    w = fp8.from_rows(q.view(E4).to(dev), s.to(dev))
    assert w.shape == tuple(shape) and w.q.shape[-3:] == (-(-n // 16), kb(k), 2048)
    q2, s2 = fp8.to_rows(w)
    assert torch.equal(codes(q2), q) and torch.equal(s2.cpu(), s)
    # the layout, byte by byte: rows past n and inputs past k are zero
    c = w.q.cpu().reshape(-1, -(-n // 16), kb(k), 2, 4, 16, 16)
    full = torch.zeros(c.shape[0], c.shape[1] * 16, c.shape[2] * 128, dtype=torch.uint8)
    full[:, :n, :k] = q.reshape(-1, n, k)
    for r, i in ((0, 0), (n - 1, k - 1), (min(9, n - 1), min(77, k - 1)), (c.shape[1] * 16 - 1, c.shape[2] * 128 - 1)):
        assert torch.equal(c[:, r // 16, i // 128, i % 128 // 64, i % 64 // 16, r % 16, i % 16], full[:, r, i])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (130, 257), (128, 128), (256, 40), (2, 33, 200)])
def test_pack_is_exact(fp8, dev, dtype, shape):
    g = torch.Generator().manual_seed(sum(shape))
    w = (torch.randn(shape, generator=g) * 0.02).to(dtype)
    n, k = shape[-2:]
    f = w.float().reshape(-1, n, k)
    p = torch.zeros(f.shape[0], kb(n) * 128, kb(k) * 128)
    p[:, :n, :k] = f
    b = p.reshape(f.shape[0], kb(n), 128, kb(k), 128)
    s = b.abs().amax((2, 4)).clamp(min=1e-10) / 448
    q = (b / s[:, :, None, :, None]).reshape(p.shape)[:, :n, :k].to(E4)
    q2, s2 = fp8.to_rows(fp8.pack(w.to(dev)))
    assert torch.equal(s2.cpu().reshape(s.shape), s) and torch.equal(codes(q2).reshape(q.shape), codes(q))


# ---------------------------------------------------------------------------------------------------------------- product
def integer_case(M, N, K, seed):
    """Codes that are small integers, scales powers of two: exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    a = torch.zeros(M, kb(K) * 128)
    a[:, :K] = torch.randint(-3, 4, (M, K), generator=g).float()
    w = torch.randint(-3, 4, (N, K), generator=g).float()
    sa = 2.0 ** torch.randint(-2, 3, (M, kb(K)), generator=g)
    sw = 2.0 ** torch.randint(-2, 3, (kb(N), kb(K)), generator=g)
    wide = w.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = (a.double() * sa.double().repeat_interleave(128, 1))[:, :K] @ wide.T
    return a.to(E4), sa, w.to(E4), sw, y


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 5120, 1000), (2, 40, 300), (5, 130, 260), (16, 256, 4000), (17, 100, 128), (31, 64, 512),
          (33, 515, 640), (48, 300, 1500), (64, 129, 2048), (65, 70, 130), (100, 333, 1024), (129, 512, 3000), (200, 1000, 5000),
          (257, 260, 384), (333, 640, 2500), (600, 4100, 256), (1025, 2050, 500)]


@pytest.mark.parametrize("epi", [0, 1])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_is_exact_on_integers(fp8, dev, M, N, K, epi):
    a, sa, w, sw, y = integer_case(M, N, K, M + N + K)
    live = max(1, M - M // 5)
    weight = fp8.from_rows(w.to(dev), sw.to(dev))
    if epi == 0:
        out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=dev)
        want = y.float().to(torch.bfloat16)
    else:
        h = torch.randint(-99, 99, (M, N), generator=torch.Generator().manual_seed(1)).float()
        out = h.to(dev)
        want = (y + h.double()).float()
    before = out.cpu().clone()
    fp8.gemm(a.to(dev), sa.to(dev), weight, out, n_of(live, dev), M, epi=epi)
    assert torch.equal(out.cpu()[:live], want[:live])
    assert torch.equal(out.cpu()[live:], before[live:])


@pytest.mark.parametrize("M,N,K", [(1, 200, 5120), (16, 333, 2000), (40, 512, 4096), (150, 700, 3333), (700, 4096, 1111)])
def test_gemm_on_normal_values(fp8, dev, M, N, K):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g)
    x[:, 7] *= 30
    q, s = plain_quant(x, K)
    weight = fp8.pack((torch.randn(N, K, generator=g) * 0.02).to(dev))
    wq, ws = (t.cpu() for t in fp8.to_rows(weight))
    a = q.double() * s.double().repeat_interleave(128, 1)
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = a[:, :K] @ w.T
    for epi in (0, 1):
        out = torch.zeros(M, N, dtype=torch.float32 if epi else torch.bfloat16, device=dev)
        fp8.gemm(q.to(dev), s.to(dev), weight, out, None, M, epi=epi)
        err = (out.cpu().double() - y).norm() / y.norm()
        assert err <= (0 if epi else 2 ** -8) + 2 ** -10, err
        assert epi == 0 or err <= 1e-4                    # 2^-13 per product with independent signs: 2^-13 sqrt(1 / 3) of it


@pytest.mark.parametrize("M", [3, 40, 130, 520])
def test_gemm_strides(fp8, dev, M):
    """Activations, scales and outputs that are column ranges of wider buffers, also at odd places; what lies beside stays."""
    N, K = 270, 650
    a, sa, w, sw, y = integer_case(M, N, K, M)
    weight = fp8.from_rows(w.to(dev), sw.to(dev))
    wa = torch.full((M, kb(K) * 128 + 160), float("nan"), device=dev).to(E4)
    wa[:, 32:32 + kb(K) * 128] = a.to(dev)
    ws = torch.full((M, kb(K) + 3), float("nan"), device=dev)
    ws[:, 1:1 + kb(K)] = sa.to(dev)
    for at, width in ((0, 272), (4, 280), (1, 277)):
        out = torch.full((M, width), 5.0, dtype=torch.bfloat16, device=dev)
        fp8.gemm(wa[:, 32:32 + kb(K) * 128], ws[:, 1:1 + kb(K)], weight, out[:, at:at + N], None, M)
        assert torch.equal(out.cpu()[:, at:at + N], y.float().to(torch.bfloat16))
        assert (out.cpu()[:, :at] == 5).all() and (out.cpu()[:, at + N:] == 5).all()
    # one row of activations for all
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    fp8.gemm(a[:1].to(dev).expand(M, -1), sa[:1].to(dev).expand(M, -1), weight, out, None, M)
    assert torch.equal(out.cpu(), y[:1].float().to(torch.bfloat16).expand(M, -1))


@pytest.mark.parametrize("M", [4, 50, 300])
def test_gemm_not_finite(fp8, dev, M):
    """A NaN in a row stays in that row, one in a weight's row in that output; rows that are not live are not read."""
    N, K = 160, 384
    a, sa, w, sw, y = integer_case(M, N, K, 5)
    a, w = a.to(dev), w.to(dev)
    a[2, 300] = float("nan")
    w[33, 5] = float("nan")
    sa = sa.to(dev)
    sa[M - 1] = float("nan")
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    fp8.gemm(a, sa, fp8.from_rows(w, sw.to(dev)), out, n_of(M - 1, dev), M)
    got, want = out.cpu(), y.float().to(torch.bfloat16)
    want[2], want[:, 33], want[M - 1] = float("nan"), float("nan"), 0
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("M", [1, 20, 333])
def test_gemm_captured(fp8, dev, M):
    """Captured with its quantizer and replayed on new inputs, eager calls of another size between the replays."""
    N, K = 600, 4096
    g = torch.Generator().manual_seed(M)
    weight = fp8.pack((torch.randn(N, K, generator=g) * 0.02).to(dev))
    x = torch.randn(M, K, generator=g).to(dev)
    q, s = torch.zeros(M, K, device=dev).to(E4), torch.zeros(M, kb(K), device=dev)
    out, n = torch.zeros(M, N, dtype=torch.bfloat16, device=dev), n_of(M, dev)

    def step(o):
        fp8.quantize_act(x, q, s, n, M)
        fp8.gemm(q, s, weight, o, n, M)
    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    for i in range(3):
        x.copy_(torch.randn(M, K, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got, want = out.clone(), torch.zeros_like(out)
        step(want)
        other = torch.zeros(200, N, dtype=torch.bfloat16, device=dev)
        fp8.gemm(torch.ones(200, K, device=dev).to(E4), torch.ones(200, kb(K), device=dev), weight, other, None, 200)
        assert torch.equal(got, want), i
        n.fill_(max(1, M - i))
        out.zero_()
        n.fill_(M)


def test_gemm_on_two_streams(fp8, dev):
    """Calls that need the workspace, in flight on two streams at once."""
    M, N, K = 150, 512, 4096
    ins = [integer_case(M, N, K, i) for i in range(2)]
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    moved = [(a.to(dev), sa.to(dev), fp8.from_rows(w.to(dev), sw.to(dev))) for a, sa, w, sw, _ in ins]
    torch.cuda.synchronize()
    for i in range(6):
        a, sa, w = moved[i % 2]
        with torch.cuda.stream(streams[i % 2]):
            out = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
            fp8.gemm(a, sa, w, out, None, M)
        outs.append(out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out.cpu(), ins[i % 2][4].float().to(torch.bfloat16))
