"""fp8.gemm in every form that its rule chooses (few rows streamed; tiles of 32, 64, 128 and 256 rows; K in parts; activations in
panels), exact on small integers with power-of-two scales; fp8.quantize_act beside every midpoint between codes; calls without
live rows, with more than there are, and from two threads."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fp8(dev):
    from prism_amd import fp8
    return fp8


def kb(k):
    return -(-k // 128)


def case(M, N, K, dev, seed):
    """Integers up to 3 and scales 1/4 .. 4: every sum is a multiple of 1/16 below 2^24 / 16 for K up to 20000 (a block's sum is at
    most 128 x 9 x 16; random signs keep the whole far below), so fp32 holds it exactly.  On the GPU, the product in 64 bits."""
    g = torch.Generator(device=dev).manual_seed(seed)
    a = torch.zeros(M, kb(K) * 128, device=dev)
    a[:, :K] = torch.randint(-3, 4, (M, K), generator=g, device=dev).float()
    w = torch.randint(-3, 4, (N, K), generator=g, device=dev).float()
    sa = 2.0 ** torch.randint(-2, 3, (M, kb(K)), generator=g, device=dev)
    sw = 2.0 ** torch.randint(-2, 3, (kb(N), kb(K)), generator=g, device=dev)
    wide = w.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    y = (a.double() * sa.double().repeat_interleave(128, 1))[:, :K] @ wide.T.contiguous()
    assert y.abs().max() < 2 ** 20
    return a.to(E4), sa, w.to(E4), sw, y


FORMS = [(3, 5000, 130), (20, 8200, 130), (20, 40, 5000), (32, 1300, 9000), (70, 40, 130), (64, 40, 2050), (50, 5000, 9000), (520, 5000, 130),
         (300, 3300, 9000), (130, 8200, 9000), (1030, 5000, 5000), (2060, 3300, 2050), (4100, 40, 5000), (4100, 515, 9000), (4100, 8200, 1000),
         (4100, 3300, 130), (4100, 3300, 9000), (4100, 1000, 17000), (1, 40, 13000), (7, 5000, 5000),
         (12, 3300, 2050), (30, 4100, 2600), (47, 2000, 1300), (64, 3300, 2050)]


@pytest.mark.parametrize("M,N,K", FORMS)
def test_every_form_is_exact_on_integers(fp8, dev, M, N, K):
    a, sa, w, sw, y = case(M, N, K, dev, M + N + K)
    weight = fp8.from_rows(w, sw)
    live = M - M // 9
    n = torch.tensor([live], dtype=torch.int32, device=dev)
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=dev)
    fp8.gemm(a, sa, weight, out, n, M)
    assert torch.equal(out[:live], y[:live].float().to(torch.bfloat16)) and (out[live:] == 7).all()
    h = torch.randint(-99, 99, (M, N), generator=torch.Generator(device=dev).manual_seed(1), device=dev).float()
    out = h.clone()
    fp8.gemm(a, sa, weight, out, n, M, epi=1)
    assert torch.equal(out[:live], (y + h.double()).float()[:live]) and torch.equal(out[live:], h[live:])


@pytest.mark.parametrize("M,N,K", [(40, 300, 700), (300, 3300, 9000), (4100, 515, 9000)])
def test_more_live_rows_than_rows_or_none(fp8, dev, M, N, K):
    a, sa, w, sw, y = case(M, N, K, dev, 3)
    weight = fp8.from_rows(w, sw)
    for live in (M + 1000, 0, -5):
        n = torch.tensor([live], dtype=torch.int32, device=dev)
        out = torch.full((M + 2, N), 7.0, dtype=torch.bfloat16, device=dev)
        fp8.gemm(a, sa, weight, out, n, M)
        rows = min(max(live, 0), M)
        assert torch.equal(out[:rows], y[:rows].float().to(torch.bfloat16)) and (out[rows:] == 7).all()


@pytest.mark.parametrize("K", [640, 9000])
def test_rows_of_wide_buffers(fp8, dev, K):
    """Rows further apart than a tile's offsets would hold together, and 4100 rows that are one."""
    M, N = 2060, 1300
    a, sa, w, sw, y = case(M, N, K, dev, 9)
    weight = fp8.from_rows(w, sw)
    wide = torch.zeros(M, 65536 + 128 * kb(K), dtype=torch.uint8, device=dev).view(E4)
    wide[:, 32768:32768 + 128 * kb(K)] = a
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    fp8.gemm(wide[:, 32768:32768 + 128 * kb(K)], sa, weight, out, None, M)
    assert torch.equal(out, y.float().to(torch.bfloat16))
    out.zero_()
    fp8.gemm(a[5:6].expand(M, -1), sa[5:6].expand(M, -1), weight, out, None, M)
    assert torch.equal(out, y[5:6].float().to(torch.bfloat16).expand(M, -1))


def test_more_rows_than_a_grid_dimension(fp8, dev):
    from prism_amd import moe
    M, N, K = 70000, 40, 300
    a, sa, w, sw, y = case(M, N, K, dev, 11)
    out = torch.zeros(M, N, dtype=torch.bfloat16, device=dev)
    fp8.gemm(a, sa, fp8.from_rows(w, sw), out, None, M)
    assert torch.equal(out, y.float().to(torch.bfloat16))
    x = torch.randn(M, 40, device=dev)
    ids, wt = torch.zeros(M, 2, dtype=torch.int32, device=dev), torch.zeros(M, 2, device=dev)
    moe.route(x, ids, wt, None, M)
    assert torch.equal(ids.long(), x.topk(2, 1)[1])


def test_two_threads(fp8, dev):
    """Calls that use the workspace, from two threads on their own streams."""
    ins = [case(300, 3300, 9000, dev, i) for i in range(2)]
    ws = [fp8.from_rows(i[2], i[3]) for i in ins]
    outs = [[torch.zeros(300, 3300, dtype=torch.bfloat16, device=dev) for _ in range(5)] for _ in range(2)]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for o in outs[i]:
                    fp8.gemm(ins[i][0], ins[i][1], ws[i], o, None, 300)
        except Exception as e:                                   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not errors
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, ins[i][4].float().to(torch.bfloat16))


def test_quantize_beside_every_midpoint(fp8, dev):
    """fp32 values a few places beside the midpoints of all neighbouring codes times scales of every kind: the codes are the IEEE
    quotient's."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(E4).float()
    mids = (codes[:-1] + codes[1:]) / 2
    g = torch.Generator().manual_seed(0)
    rows = []
    for _ in range(120):
        amax = (0.5 + torch.rand(1, generator=g)) * 2.0 ** torch.randint(-30, 30, (1,), generator=g)
        s = amax / 448
        base = mids * s
        bits = base.view(torch.int32)[:, None] + torch.arange(-6, 7, dtype=torch.int32)[None]
        v = bits.view(torch.float32).flatten()
        v = torch.where(torch.rand(v.shape, generator=g) < 0.5, -v, v)
        v = torch.cat([v, torch.zeros(-len(v) % 127)]).view(-1, 127)
        rows.append(torch.cat([amax.expand(v.shape[0], 1), v.clamp(-amax.item(), amax.item())], 1))
    x = torch.cat(rows)
    T = x.shape[0]
    q, s = torch.zeros(T, 128, device=dev).to(E4), torch.zeros(T, 1, device=dev)
    fp8.quantize_act(x.to(dev), q, s, None, T)
    ws = x.abs().amax(1, keepdim=True).clamp(min=1e-10) / 448
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu().view(torch.uint8), (x / ws).to(E4).view(torch.uint8))


def test_nothing_live_in_any_call(dev):
    from prism_amd import fp8, moe
    n = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.randn(200, 256, device=dev).to(torch.bfloat16)
    q, s = torch.full((200, 256), 2.0, device=dev).to(E4), torch.full((200, 2), 2.0, device=dev)
    fp8.quantize_act(x, q, s, n, 200)
    ids, w = torch.full((200, 4), 5, dtype=torch.int32, device=dev), torch.full((200, 4), 2.0, device=dev)
    for score in ("softmax", "sigmoid"):
        moe.route(torch.randn(200, 9, device=dev), ids, w, n, 200, score=score)
    ws = [fp8.pack(torch.randn(9, *nk, device=dev)) for nk in ((48, 256), (48, 256), (256, 48))]
    for T in (3, 200):
        out = torch.full((T, 256), 2.0, dtype=torch.bfloat16, device=dev)
        moe.experts(x, ids, w, *ws, out, n, T)
        assert (out == 2).all()
    assert (q.float() == 2).all() and (s == 2).all() and (ids == 5).all() and (w == 2).all()
