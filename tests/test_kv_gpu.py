"""prism_amd.kv on the GPU: append bit for bit against the formula's fp32 steps, attend against 64-bit softmax attention.

attend's tolerance, per output with o the exact value and vm the head's largest |v| (u = 2^-24): the bf16 rounding of o,
2^-8 |o|, plus 2 E vm for the weights' relative error E, once in the sum and once in the normaliser.  E collects the
score's error (D + 4) u times scale sum |q k| (products exact, D additions, two scalings), the exponential's and its
argument's 2^-21, the two truncated bf16 parts' 2^-15, and the sums over the tokens, 4 (tokens + 32) u."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def make_cache(g, pages, page, heads, dim, dtype, layout):
    shape = (pages, heads, page, dim) if layout == "head" else (pages, page, heads, dim)
    x = torch.randn(*shape, generator=g)
    x = x.to(dtype) if dtype == torch.bfloat16 else (x * 40).to(dtype)
    return x.transpose(1, 2) if layout == "head" else x


def bits(x):
    return x.contiguous().view(torch.uint8)


def to_dev(x, dev):
    """The tensor on the device with its strides (Tensor.to keeps those of dense tensors)."""
    y = x.to(dev)
    assert y.stride() == x.stride()
    return y


# -------------------------------------------------------------------------------------------------------------- append
def rotated(x, rope, pos, pairs):
    """fp32 [T, heads, dim]; every product and sum rounded to fp32, as torch's elementwise operations on the CPU are."""
    y = x.float().clone()
    if rope is None:
        return y
    half = rope.shape[1] // 2
    c, s = rope[pos, None, :half], rope[pos, None, half:]
    i, j = (slice(0, half), slice(half, 2 * half)) if pairs == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    a, b = y[..., i].clone(), y[..., j].clone()
    y[..., i] = a * c - b * s
    y[..., j] = b * c + a * s
    return y


def stored(x, dtype, scale):
    if dtype == torch.bfloat16:
        return x.to(dtype)
    return (x if scale is None else x / scale[:, None]).clamp(-448, 448).to(dtype)


@pytest.mark.parametrize("T,live,hq,hkv,dim,rot,page,dtype,layout,pairs,scaled", [
    (1, 1, 32, 8, 128, 128, 16, torch.bfloat16, "token", "half", False),
    (5, 3, 24, 4, 256, 64, 64, E4M3, "head", "half", True),
    (7, 7, 8, 8, 64, 32, 32, E4M3, "token", "adjacent", False),
    (130, 129, 5, 1, 64, 64, 16, torch.bfloat16, "head", "adjacent", False),
    (33, 33, 0, 2, 128, 96, 256, torch.bfloat16, "token", "half", False),       # no queries
    (9, 9, 7, 1, 128, 0, 16, E4M3, "head", "half", True),                       # no rotation
    (700, 650, 40, 8, 128, 16, 64, torch.bfloat16, "token", "half", False),
])
def test_append_bits(dev, T, live, hq, hkv, dim, rot, page, dtype, layout, pairs, scaled):
    from prism_amd import kv
    g = torch.Generator().manual_seed(T * 1000 + dim)
    seqs = min(4, T)
    cols = -(-(T + 40) // page) + 1
    pages = seqs * cols + 3
    kc, vc = (make_cache(g, pages, page, hkv, dim, dtype, layout) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:seqs * cols].view(seqs, cols).int()
    proj = (torch.randn(T, (hq + 2 * hkv) * dim + 8, generator=g) * 3).to(torch.bfloat16)
    proj[0, 3], proj[0, (hq + hkv) * dim + 1] = float("inf"), float("nan")
    seq = torch.arange(T).remainder(seqs).int()
    pos = (torch.arange(T) // seqs + 17).int()
    rope = kv.rope_table(cols * page, rot, 1e6, "cpu") if rot else None
    sc = [0.01 + 0.02 * torch.rand(hkv, generator=g) for _ in range(2)] if scaled else [None, None]

    def parts(p):
        at = lambda i, n: p[:, i * dim:(i + n) * dim].unflatten(1, (n, dim))   # noqa: E731
        return at(0, hq) if hq else None, at(hq, hkv), at(hq + hkv, hkv)
    q, k, v = parts(proj)
    want_k, want_v = kc.clone(), vc.clone()
    t = slice(0, live)
    where = (table[seq[t].long(), pos[t].long() // page].long(), pos[t].long() % page)
    want_k[where] = stored(rotated(k[t], rope, pos[t].long(), pairs), dtype, sc[0])
    want_v[where] = stored(v[t].float(), dtype, sc[1])

    d = to_dev(proj, dev)
    dq, dk, dv = parts(d)
    out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device=dev) if hq else None
    kd, vd = to_dev(kc, dev), to_dev(vc, dev)
    kv.append(dq, dk, dv, None if rope is None else rope.to(dev), pos.to(dev), table.to(dev), kd, vd, out,
              torch.tensor([live], dtype=torch.int32, device=dev), T, seq=seq.to(dev), pairs=pairs,
              k_scale=None if sc[0] is None else sc[0].to(dev), v_scale=None if sc[1] is None else sc[1].to(dev))

    def same(got, want):
        got, want = got.cpu().float(), want.float()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, 5.0, 6e38, -6e38), torch.nan_to_num(want, 5.0, 6e38, -6e38))
    same(kd, want_k)
    same(vd, want_v)
    if hq:
        same(out[:live], rotated(q[t], rope, pos[t].long(), pairs).to(torch.bfloat16))
        assert (out[live:] == 7).all()


def test_append_skips_tokens_without_a_place(dev):
    """Negative positions, positions past the table or the rotations, sequences and pages out of range: nothing is
    written for them; their neighbours are.  q_out may be q."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(3)
    hq, hkv, dim, page, pages, cols = 2, 1, 64, 16, 6, 3
    kc, vc = (make_cache(g, pages, page, hkv, dim, torch.bfloat16, "token") for _ in range(2))
    table = torch.tensor([[0, 2, -1], [4, 77, 5]], dtype=torch.int32)
    rope = kv.rope_table(40, dim, 1e4, "cpu")
    cases = [(0, 3, True), (0, -1, False), (0, 47, False), (1, 48, False), (1, 20, False), (0, 33, False), (2, 1, False),
             (-1, 1, False), (1, 39, True), (1, 41, False), (0, 17, True)]
    T = len(cases)
    seq, pos = (torch.tensor([c[i] for c in cases], dtype=torch.int32) for i in (0, 1))
    q, k, v = (torch.randn(T, h, dim, generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
    want_k, want_v, want_q = kc.clone(), vc.clone(), q.clone()
    for i, (s, p, there) in enumerate(cases):
        if there:
            at = (int(table[s, p // page]), p % page)
            r = torch.tensor([p])
            want_k[at] = rotated(k[i:i + 1], rope, r, "half")[0].to(torch.bfloat16)
            want_v[at] = v[i]
            want_q[i] = rotated(q[i:i + 1], rope, r, "half")[0].to(torch.bfloat16)
    qd, kd, vd = q.to(dev), kc.to(dev), vc.to(dev)
    kv.append(qd, k.to(dev), v.to(dev), rope.to(dev), pos.to(dev), table.to(dev), kd, vd, qd, None, T, seq=seq.to(dev))
    assert torch.equal(kd.cpu(), want_k) and torch.equal(vd.cpu(), want_v) and torch.equal(qd.cpu(), want_q)


# -------------------------------------------------------------------------------------------------------------- attend
def exact_attend(q, kc, vc, table, lens, scale, window, ks, vs):
    """(out, bound of the absolute error before the output's rounding), float64."""
    T, hq, dim = q.shape
    page, hkv = kc.shape[1], kc.shape[2]
    out, tol = torch.zeros(T, hq, dim, dtype=torch.float64), torch.zeros(T, hq, 1, dtype=torch.float64)
    for i in range(T):
        n = min(max(int(lens[i]), 0), table.shape[1] * page)
        lo = max(0, n - window) if window else 0
        if n == 0:
            continue
        t = torch.arange(lo, n)
        at = table[i, t // page].long()
        for h in range(hkv):
            k, v = kc[at, t % page, h].double(), vc[at, t % page, h].double()
            if ks is not None:
                k, v = k * ks[h].double(), v * vs[h].double()
            hs = slice(h * hq // hkv, (h + 1) * hq // hkv)
            x = q[i, hs].double()
            out[i, hs] = torch.softmax(x @ k.T * scale, 1) @ v
            mag = (x.abs() @ k.abs().T).amax(1, keepdim=True) * scale
            e = (dim + 4) * 2.0 ** -24 * mag + 2.0 ** -21 + 2.0 ** -15 + 4 * (n - lo + 32) * 2.0 ** -24
            tol[i, hs] = 2 * e * v.abs().max()
    return out, tol


def check_attend(dev, lens, hq, hkv, dim, page, dtype, layout, window=0, scale=None, live=None, scaled=False, seed=0,
                 q_std=1.5, extra=8):
    from prism_amd import kv
    g = torch.Generator().manual_seed(seed + 17 * dim + len(lens))
    T = len(lens)
    live = T if live is None else live
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    kc, vc = (make_cache(g, pages, page, hkv, dim, dtype, layout) for _ in range(2))
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((T, max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    # rows of the cache that hold no visible token hold NaN
    for c in (kc, vc):
        used = torch.zeros(pages, page, dtype=torch.bool)
        for i, n in enumerate(lens):
            t = torch.arange(max(0, n - window) if window else 0, n)
            used[table[i, t // page].long(), t % page] = True
        if dtype == E4M3:
            c.view(torch.uint8)[~used] = 0x7f
        else:
            c[~used] = float("nan")
    ks, vs = ((0.01 + 0.02 * torch.rand(hkv, generator=g) for _ in range(2)) if scaled else (None, None))
    proj = (q_std * torch.randn(T, (hq + 2) * dim, generator=g)).to(torch.bfloat16)
    q = proj[:, dim:(hq + 1) * dim].unflatten(1, (hq, dim))
    s = dim ** -0.5 if scale is None else scale
    want, tol = exact_attend(q[:live], kc, vc, table, lens, s, window, ks, vs)

    dproj = proj.to(dev)
    out = torch.full((T, hq + 1, dim), 7.0, dtype=torch.bfloat16, device=dev)[:, :hq]
    args = (dproj[:, dim:(hq + 1) * dim].unflatten(1, (hq, dim)), to_dev(kc, dev), to_dev(vc, dev), table.to(dev),
            torch.tensor(lens, dtype=torch.int32, device=dev), out,
            torch.tensor([live], dtype=torch.int32, device=dev), T)
    kw = dict(scale=scale, window=window, k_scale=None if ks is None else ks.to(dev),
              v_scale=None if vs is None else vs.to(dev))
    kv.attend(*args, **kw)
    got = out.cpu()
    assert (got[live:] == 7).all()
    err = (got[:live].double() - want).abs()
    bound = 2.0 ** -8 * want.abs() + tol
    assert (err <= bound).all(), (float((err - bound).max()), torch.nonzero(err > bound)[:4].tolist())
    for i, n in enumerate(lens[:live]):
        if n == 0:
            assert (got[i] == 0).all()
    out.fill_(7.0)
    kv.attend(*args, **kw)
    assert torch.equal(bits(out.cpu()), bits(got))               # the same bits again


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 255, 257, 700]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_attend_lengths(dev, dim, dtype, layout):
    check_attend(dev, EDGES, 6, 2, dim, 16, dtype, layout, scaled=dtype == E4M3)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (5, 1), (28, 4), (16, 1), (17, 1), (40, 2), (64, 1)])
def test_attend_heads(dev, hq, hkv):
    check_attend(dev, [77, 300, 1], hq, hkv, 128, 32, torch.bfloat16, "head")


@pytest.mark.parametrize("page", [16, 64, 256, 1024])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attend_long_and_ragged(dev, page, dtype):
    """One long sequence beside short ones: split and joined, and not."""
    check_attend(dev, [5000, 3, 0, 1025, 130], 8, 2, 128, page, dtype, "token", scaled=dtype == E4M3)
    check_attend(dev, [20011], 8, 2, 64, page, dtype, "head")


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 4096])
def test_attend_window(dev, window):
    check_attend(dev, [0, 1, 16, 17, 99, 100, 101, 500, 5003], 6, 2, 128, 16, torch.bfloat16, "token", window=window)


def test_attend_live_rows_and_many_sequences(dev):
    g = torch.Generator().manual_seed(8)
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    check_attend(dev, lens, 4, 2, 64, 32, torch.bfloat16, "head", live=131)


@pytest.mark.parametrize("hq,hkv,dim,window", [(8, 4, 64, 0), (4, 4, 128, 0), (64, 4, 64, 33), (28, 4, 128, 0), (24, 8, 256, 700),
                                               (12, 12, 64, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attend_batches_over_token_rows(dev, hq, hkv, dim, window, dtype):
    """Sixteen sequences and more over caches whose heads lie side by side, taken four at a time; some end a part, some
    are empty, some are past the live rows."""
    lens = [0, 1, 31, 32, 33, 2100, 64, 0, 0, 97, 1024, 15, 16, 17, 129, 1, 500, 0, 800]
    check_attend(dev, lens, hq, hkv, dim, 16, dtype, "token", window=window, live=18, scaled=dtype == E4M3)


def test_attend_peaked_scores(dev):
    """Scores of hundreds: one token takes nearly all of the weight, the running maximum moves often."""
    check_attend(dev, [900, 64], 4, 1, 128, 16, torch.bfloat16, "token", scale=1.0, q_std=4.0)


def test_attend_extreme_values(dev):
    """Keys of the type's lowest value give a uniform or a one-token softmax, never NaN; infinite and NaN values show
    only where their token is visible."""
    from prism_amd import kv
    dim, page = 64, 16
    kc, vc = (torch.zeros(3, page, 1, dim, dtype=torch.bfloat16) for _ in range(2))
    low = torch.finfo(torch.bfloat16).min
    kc[0, :4, 0, 0] = low                                        # scores -3e38 (times 1 / 8): still finite
    vc[0, :4, 0] = torch.arange(4.0)[:, None]
    kc[1, 0, 0, 0] = low                                         # one token far below the other
    vc[1, 0, 0], vc[1, 1, 0] = 9.0, 2.0
    vc[2, 0, 0], vc[2, 1, 0] = 1.0, float("inf")
    table = torch.tensor([[0], [1], [2], [2]], dtype=torch.int32)
    q = torch.zeros(4, 1, dim, dtype=torch.bfloat16)
    q[:, 0, 0] = 1.0
    out = torch.empty(4, 1, dim, dtype=torch.bfloat16, device=dev)
    kv.attend(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), torch.tensor([4, 2, 1, 2], dtype=torch.int32, device=dev),
              out, None, 4)
    out = out.cpu().float()
    assert (out[0] == 1.5).all() and (out[1] == 2.0).all() and (out[2] == 1.0).all() and torch.isinf(out[3]).all()


def test_attend_length_past_the_table(dev):
    """More tokens than the table has room for count as what it holds."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(1)
    kc, vc = (make_cache(g, 4, 16, 2, 64, torch.bfloat16, "token").to(dev) for _ in range(2))
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=dev)
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16).to(dev)
    a, b = (torch.empty(1, 4, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for out, n in ((a, 32), (b, 2 ** 31 - 1)):
        kv.attend(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device=dev), out, None, 1)
    assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["token", "head"])
def test_offsets_beyond_32_bits(dev, layout):
    """The last pages of caches of over 2^32 bytes, written and read."""
    from prism_amd import kv
    pages, page, hkv, dim, T = 36000, 64, 8, 128, 3
    kc, vc = (torch.empty((pages, hkv, page, dim) if layout == "head" else (pages, page, hkv, dim), dtype=torch.bfloat16,
                          device=dev) for _ in range(2))
    if layout == "head":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    assert kc.numel() * 2 > 2 ** 32
    g = torch.Generator().manual_seed(2)
    lens = [70, 1, 128]
    table = torch.tensor([[pages - 1, pages - 2], [pages - 3, -1], [33000, 0]], dtype=torch.int32)
    seq = torch.tensor([i for i, n in enumerate(lens) for _ in range(n)], dtype=torch.int32)
    pos = torch.tensor([t for n in lens for t in range(n)], dtype=torch.int32)
    k, v = (torch.randn(len(seq), hkv, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    kv.append(None, k.to(dev), v.to(dev), None, pos.to(dev), table.to(dev), kc, vc, None, None, len(seq), seq=seq.to(dev))
    rows = table[seq.long(), pos.long() // page].long().to(dev), (pos.long() % page).to(dev)
    assert torch.equal(kc[rows].cpu(), k) and torch.equal(vc[rows].cpu(), v)
    q = torch.randn(T, 16, dim, generator=g).to(torch.bfloat16)
    out = torch.empty(T, 16, dim, dtype=torch.bfloat16, device=dev)
    kv.attend(q.to(dev), kc, vc, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), out, None, T)
    some = sorted(set(table.flatten().tolist()) - {-1})
    small = {p: i for i, p in enumerate(some)}
    kt, vt = (c[torch.tensor(some, device=dev)].cpu() for c in (kc, vc))
    tab = torch.tensor([[small.get(p, -1) for p in r] for r in table.tolist()], dtype=torch.int32)
    want, tol = exact_attend(q, kt, vt, tab, lens, dim ** -0.5, 0, None, None)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + tol).all()


def test_captured_on_another_stream(dev):
    """append and attend captured on a side stream: every replay gives the eager call's bits, with other lengths and
    other eager work between the replays."""
    from prism_amd import kv
    g = torch.Generator().manual_seed(4)
    T, hq, hkv, dim, page = 3, 8, 2, 128, 16
    kc, vc = kv.cache(64, page, hkv, dim, device=dev)
    first = torch.randn(kc.shape, generator=g).to(torch.bfloat16).to(dev)
    kc.copy_(first)
    vc.copy_(first.flip(0))
    table = torch.randperm(64, generator=g)[:60].view(3, 20).int().to(dev)
    q, k, v = (torch.randn(T, h, dim, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    rope = kv.rope_table(320, dim, device=dev)
    pos = torch.zeros(T, dtype=torch.int32, device=dev)
    n = torch.tensor([T], dtype=torch.int32, device=dev)
    lens, turned, out = pos + 1, torch.empty_like(q), torch.empty_like(q)

    def both():
        kv.append(q, k, v, rope, pos, table, kc, vc, turned, n, T)
        torch.add(pos, 1, out=lens)
        kv.attend(turned, kc, vc, table, lens, out, n, T)
    both()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        both()
    for step in ([0, 5, 300], [200, 17, 319], [319, 0, 16], [1, 2, 3]):
        pos.copy_(torch.tensor(step, dtype=torch.int32))
        both()
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(out), bits(want))
