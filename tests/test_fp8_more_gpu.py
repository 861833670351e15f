"""fp8.quantize_act where a thread takes several units and the grid goes round again; fp8.gemm on a single block of 128 inputs, on
unsplit 128 x 128 tiles with the activations in panels, and captured calls whose live count changes between replays."""
import pytest
import torch

from test_fp8_kernels_gpu import case, kb

pytestmark = pytest.mark.gpu
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fp8(dev):
    from prism_amd import fp8
    return fp8


def n_of(v, dev):
    return torch.tensor([v], dtype=torch.int32, device=dev)


# 32 units (a row's 128 inputs) a workgroup: from 2048 workgroups on two units a thread, at most 4096 workgroups, so that past
# 262144 units (131072 where k % 16 leaves no whole loads) each goes round again
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,live,k", [(4100, 4099, 2560), (8191, 8191, 4352), (8191, 7001, 4352), (8191, 8190, 2190), (70001, 69999, 128),
                                         (300007, 262147, 16)])
def test_quantize_many_units(fp8, dev, dtype, rows, live, k):
    g = torch.Generator(device=dev).manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g, device=dev) * torch.exp(3 * torch.randn(rows, 1, generator=g, device=dev))
    x = x.to(dtype)
    q = torch.full((rows, kb(k) * 128), 1.0, device=dev).to(E4)
    s = torch.full((rows, kb(k)), -1.0, device=dev)
    fp8.quantize_act(x, q, s, n_of(live, dev), rows)
    q, s, x = q.cpu().view(torch.uint8), s.cpu(), x.cpu()[:live].float()             # (the quotients on the CPU: IEEE divisions)
    b = torch.nn.functional.pad(x, (0, kb(k) * 128 - k)).unflatten(1, (-1, 128))
    ws = b.abs().amax(2).clamp(min=1e-10) / 448
    assert torch.equal(s[:live], ws) and (s[live:] == -1).all()
    assert torch.equal(q[:live], (b / ws[..., None]).flatten(1).to(E4).view(torch.uint8))
    assert (q[live:] == 0x38).all()                                                   # (the code of 1)


# the forms: tiles of 32, 64, 64, 128, 128, 256 and 256 rows; then 128 rows, unsplit, in panels (whole stores of rows and single ones)
@pytest.mark.parametrize("M,N,K", [(20, 8200, 128), (65, 40, 128), (100, 1001, 1), (300, 8200, 128), (520, 5000, 100), (1030, 8200, 128),
                                   (4100, 5000, 64), (344, 11512, 3850), (4588, 1061, 3962)])
def test_single_blocks_and_panels(fp8, dev, M, N, K):
    a, sa, w, sw, y = case(M, N, K, dev, M + N + K)
    weight = fp8.from_rows(w, sw)
    live = M - M // 9
    n = n_of(live, dev)
    out = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=dev)
    fp8.gemm(a, sa, weight, out, n, M)
    assert torch.equal(out[:live], y[:live].float().to(torch.bfloat16)) and (out[live:] == 7).all()
    h = torch.randint(-99, 99, (M, N), generator=torch.Generator(device=dev).manual_seed(1), device=dev).float()
    out = h.clone()
    fp8.gemm(a, sa, weight, out, n, M, epi=1)
    assert torch.equal(out[:live], (y + h.double()).float()[:live]) and torch.equal(out[live:], h[live:])


@pytest.mark.parametrize("epi", [0, 1])
@pytest.mark.parametrize("M,N,K", [(1, 600, 4096), (8, 5000, 2000), (20, 40, 5000), (64, 600, 4096), (333, 600, 4096), (300, 3300, 9000),
                                   (344, 11512, 3850)])
def test_captured_live_counts(fp8, dev, M, N, K, epi):
    """The quantizer and the product captured once and replayed with other live counts and inputs, eager calls between: the live rows
    are an eager call's, the rows behind stay."""
    g = torch.Generator(device=dev).manual_seed(M)
    weight = fp8.pack(torch.randn(N, K, generator=g, device=dev) * 0.02)
    x = torch.randn(M, K, generator=g, device=dev)
    q, s = torch.zeros(M, kb(K) * 128, device=dev).to(E4), torch.zeros(M, kb(K), device=dev)
    out, n = torch.zeros(M, N, dtype=torch.float32 if epi else torch.bfloat16, device=dev), n_of(M, dev)

    def step(q, s, o):
        fp8.quantize_act(x, q, s, n, M)
        fp8.gemm(q, s, weight, o, n, M, epi=epi)
    step(q, s, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, s, out)
    for live in (M // 2, M, 1, 0, (M + 1) // 2, M + 5, -3):
        x.copy_(torch.randn(M, K, generator=g, device=dev))
        n.fill_(live)
        h = torch.randn(M, N, generator=g, device=dev).to(out.dtype)
        out.copy_(h)
        q.view(torch.uint8).fill_(0x38)
        s.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        rows = min(max(live, 0), M)
        q2, s2, want = torch.full_like(q.view(torch.uint8), 0x38).view(E4), torch.full_like(s, -1.0), h.clone()
        step(q2, s2, want)
        assert torch.equal(out, want) and torch.equal(out[rows:], h[rows:]), live
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2), live
        assert (q.view(torch.uint8)[rows:] == 0x38).all() and (s[rows:] == -1).all()
        assert rows == 0 or not torch.equal(out[:rows], h[:rows])
