"""kv.attend's softmax weights reach the values unbiased: over millions of outputs the mean error against 64 bits is that of
the outputs' rounding alone.

Values of [1.5, 2) keep every output in that range, where a bf16 step is 2^-7 = h and the rounding error of an output is
uniform in +-h / 2, standard deviation h / sqrt(12); its mean over n outputs is within 6 h / sqrt(12 n) of zero.  Errors of
fp32 sums have either sign; 8 2^-24 are allowed for what of them is common.  Weights cut to 16 bits would show as a mean
of about -1e-5, three times the bound.  The scores are exact (queries with one element that is not zero)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("tokens", [32, 200])
def test_attend_does_not_lean(dev, dtype, tokens):
    from prism_amd import kv
    g = torch.Generator(device=dev).manual_seed(tokens)
    T, hq, hkv, dim, page = 512, 64, 4, 256, 32
    cols = -(-tokens // page)
    kc, vc = kv.cache(T * cols, page, hkv, dim, dtype=dtype, device=dev)
    k = torch.zeros(T * cols, page, hkv, dim, device=dev)
    k[..., 0] = 4 * torch.rand(T * cols, page, hkv, generator=g, device=dev)
    kc.copy_(k.to(dtype))
    v = (1.5 + 0.5 * torch.rand(T * cols, page, hkv, dim, generator=g, device=dev)).to(torch.bfloat16).float()
    vc.copy_(v.clamp(max=1.875 if dtype == E4M3 else 2 - 2.0 ** -7).to(dtype))
    table = torch.arange(T * cols, dtype=torch.int32, device=dev).view(T, cols)
    q = torch.zeros(T, hq, dim, dtype=torch.bfloat16, device=dev)
    q[:, :, 0] = 2 * torch.rand(T, hq, generator=g, device=dev) - 1
    out = torch.empty_like(q)
    kv.attend(q, kc, vc, table, torch.full((T,), tokens, dtype=torch.int32, device=dev), out, None, T, scale=1.0)

    total, count = 0.0, 0
    for h in range(hkv):
        k = kc[:, :, h, 0].float().reshape(T, cols * page)[:, :tokens].double()
        x = vc[:, :, h].float().reshape(T, cols * page, dim)[:, :tokens].double()
        hs = slice(h * hq // hkv, (h + 1) * hq // hkv)
        w = torch.softmax(q[:, hs, 0].double()[:, :, None] * k[:, None], 2)
        want = torch.matmul(w, x)
        total += float((out[:, hs].double() - want).sum())
        count += want.numel()
    h = 2.0 ** -7
    assert abs(total / count) <= 6 * h / (12 * count) ** 0.5 + 8 * 2.0 ** -24
