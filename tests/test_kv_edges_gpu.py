"""prism_amd.kv on the GPU where its kernels can go wrong: scores past fp32's range, clones, empty calls, caches of two
memory orders."""
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


def test_clones_keep_what_they_were_made_of(dev):
    """Caches and outputs that are copy-on-write clones: the tensors they were made of stay as they are, the caches that
    attend reads stay shared."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(5)
    kc, vc = kv.cache(4, 16, 2, 64, device=dev)
    q, k, v = (torch.randn(3, h, 64, generator=g).to(torch.bfloat16).to(dev) for h in (4, 2, 2))
    turned, out = torch.zeros_like(q), torch.zeros_like(q)
    table = torch.arange(3, dtype=torch.int32, device=dev).view(3, 1)
    ones = torch.ones(3, dtype=torch.int32, device=dev)
    lk, lv, lt, lo = (torch._lazy_clone(x) for x in (kc, vc, turned, out))
    kv.append(q, k, v, None, ones - 1, table, lk, lv, lt, None, 3)
    assert (kc == 0).all() and (vc == 0).all() and (turned == 0).all()
    assert torch.equal(lk[:3, 0], k) and torch.equal(lv[:3, 0], v) and torch.equal(lt, q)
    rk, rv = torch._lazy_clone(lk), torch._lazy_clone(lv)
    kv.attend(q, rk, rv, table, ones, lo, None, 3)
    assert (out == 0).all() and torch.equal(lo, v.repeat_interleave(2, 1))
    assert torch._C._is_cow_tensor(rk) and torch._C._is_cow_tensor(rv)


def test_calls_without_rows(dev):
    """T = 0 with tensors of no rows does nothing."""
    from prism_amd import kv
    kc, vc = kv.cache(4, 16, 2, 64, device=dev)
    bf = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=dev)             # noqa: E731
    ints = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)              # noqa: E731
    n = torch.zeros(1, dtype=torch.int32, device=dev)
    kv.append(bf(0, 4, 64), bf(0, 2, 64), bf(0, 2, 64), torch.empty(9, 32, device=dev), ints(0), ints(1, 4), kc, vc,
              bf(0, 4, 64), n, 0)
    kv.attend(bf(0, 4, 64), kc, vc, ints(0, 4), ints(0), bf(0, 4, 64), n, 0)
    assert (kc == 0).all() and (vc == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_caches_of_different_orders(dev, dtype):
    """Keys by the page's heads and values by token rows, and the other way round: append and attend give the bits of
    caches of one order (fewer than 16 sequences: the order does not choose the form)."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(7)
    T, hq, hkv, dim, page, cols = 5, 8, 4, 128, 32, 9
    lens = torch.tensor([1, 40, 288, 100, 64], dtype=torch.int32, device=dev)
    table = torch.randperm(T * cols, generator=g).view(T, cols).int().to(dev)
    shape = (T * cols, page, hkv, dim)
    old = [torch.randn(shape, generator=g).to(dtype).to(dev) for _ in range(2)]
    q, k, v = (torch.randn(T, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    rope = kv.rope_table(cols * page, 64, device=dev)

    def order(x, by_head):
        c = torch.empty(shape[0], hkv, page, dim, dtype=dtype, device=dev).transpose(1, 2) if by_head else \
            torch.empty(shape, dtype=dtype, device=dev)
        c.copy_(x)
        return c

    def run(k_by_head, v_by_head):
        kc, vc = order(old[0], k_by_head), order(old[1], v_by_head)
        turned, out = torch.empty_like(q), torch.empty_like(q)
        kv.append(q, k, v, rope, lens - 1, table, kc, vc, turned, None, T)
        kv.attend(turned, kc, vc, table, lens, out, None, T)
        return [x.contiguous().view(torch.uint8) for x in (kc, vc, turned, out)]
    want = run(True, True)
    for ways in ((True, False), (False, True), (False, False)):
        assert all(torch.equal(a, b) for a, b in zip(run(*ways), want))
