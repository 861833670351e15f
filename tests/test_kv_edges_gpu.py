"""prism_amd.kv on the GPU where its kernels can go wrong: scores past fp32's range."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("lens", [[1], [5, 40, 0, 130], [700], [3, 1025, 128, 129]])
def test_attend_scores_of_minus_infinity(dev, lens, dim):
    """Keys of the type's lowest value under queries of 4 give scores of -inf.  Where all of a sequence's are, its rows are
    NaN, as the softmax of fp32 scores is; beside one finite score they have no weight; without tokens rows are 0.  Short
    sequences (one unit) and split ones."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(sum(lens) + dim)
    T, hq, hkv, page = len(lens), 4, 2, 16
    cols = -(-max(lens) // page)
    kc, vc = (torch.zeros(T * cols, page, hkv, dim, dtype=torch.bfloat16) for _ in range(2))
    vc.copy_(torch.randn(vc.shape, generator=g))
    kc[..., 0] = torch.finfo(torch.bfloat16).min
    table = torch.arange(T * cols, dtype=torch.int32).view(T, cols)
    finite = [(i, n // 3) for i, n in enumerate(lens) if n]          # in cache head 1: one token's score is 0
    for i, t in finite:
        kc[int(table[i, t // page]), t % page, 1, 0] = 0.0
    q = torch.zeros(T, hq, dim, dtype=torch.bfloat16)
    q[:, :, 0] = 4.0
    out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device=dev)
    kv.attend(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), out,
              None, T)
    out = out.cpu()
    for i, n in enumerate(lens):
        if n == 0:
            assert (out[i] == 0).all()
            continue
        t = n // 3
        assert torch.isnan(out[i, :2]).all()
        assert torch.equal(out[i, 2:], vc[int(table[i, t // page]), t % page, 1].expand(2, dim))
