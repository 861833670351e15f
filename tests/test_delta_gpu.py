"""prism_amd.delta on the GPU against the recurrence in 64 bits.

Tolerances.  Both forms compute in fp32 (u = 2^-24) or as finely.  A token's update is a contraction of the state's
error (a <= 1, |I - beta k k^T| <= 1 for unit keys and 0 <= beta <= 1), and adds at most (DK + 16) u of the column's
length |S| plus |v|; after L tokens, and for an output of the state's last value, the error of any element is below
(L + 2) (DK + 16) u (max |S column| + max |v|).  That bound is of signs that all agree; rounding errors of independent
signs give about sqrt(DK) u = 7e-7 per output relative to the tensor's norm and the contraction keeps them from adding up,
so the relative error of each whole tensor is held to 1.5e-6 as well."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def recurrence(q, k, v, g, beta, state, spans, slots, norm, scale, eps=1e-6):
    """float64 (out [T, HV, DV], state) with the rows of no sequence NaN."""
    q, k, v, g, beta, state = (x.double().clone() for x in (q, k, v, g, beta, state))
    if norm:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + eps)
    q = q * scale
    head = torch.arange(v.shape[1]) // (v.shape[1] // q.shape[1])
    out = torch.full(v.shape, float("nan"), dtype=torch.float64)
    for (begin, end), slot in zip(spans, slots):
        if not 0 <= slot < state.shape[0]:
            continue
        s = state[slot]
        for t in range(begin, end):
            s *= torch.exp(g[t])[:, None, None]
            kt = k[t, head]
            u = beta[t][:, None] * (v[t] - (kt[:, None] @ s)[:, 0])
            s += kt[:, :, None] * u[:, None]
            out[t] = (q[t, head][:, None] @ s)[:, 0]
    return out, state


def inputs(T, hk, hv, dk, dv, states, seed):
    g = torch.Generator().manual_seed(seed)
    proj = torch.randn(T, 2 * hk * dk + hv * dv + 8, generator=g).to(torch.bfloat16)
    decay = -(1 + 15 * torch.rand(hv, generator=g)) * torch.nn.functional.softplus(torch.randn(T, hv, generator=g) - 4)
    beta = torch.sigmoid(2 * torch.randn(T, hv, generator=g))
    state = 0.3 * torch.randn(states, hv, dk, dv, generator=g)
    return proj, decay, beta, state


def split(proj, hk, hv, dk, dv):
    at = hk * dk
    return (proj[:, :at].unflatten(1, (hk, dk)), proj[:, at:2 * at].unflatten(1, (hk, dk)),
            proj[:, 2 * at:2 * at + hv * dv].unflatten(1, (hv, dv)))


def compare(out, state, want_out, want_state, spans, v, dk, initial):
    longest = max([e - b for b, e in spans] + [1])
    size = max(float(want_state.norm(dim=2).max()), float(initial.norm(dim=2).max())) + float(v.abs().max())
    bound = (longest + 2) * (dk + 16) * U * size
    rows = ~torch.isnan(want_out)
    for got, want in ((out.cpu().double()[rows], want_out[rows]), (state.cpu().double(), want_state)):
        if want.numel():
            assert torch.isfinite(got).all()
            assert float((got - want).abs().max()) <= bound
            assert float((got - want).norm()) <= 1.5e-6 * float(want.norm())


def run_step(dev, T, live, hk, hv, dk, dv, norm=True, scale=None, seed=0, edit=None, slots=None, states=None):
    from prism_amd import delta
    states = T + 2 if states is None else states
    proj, g, beta, state = inputs(T, hk, hv, dk, dv, states, seed)
    if not norm:
        proj *= dk ** -0.5
    if edit:
        edit(split(proj, hk, hv, dk, dv), g, beta, state)
    order = torch.randperm(states, generator=torch.Generator().manual_seed(seed))[:T].int() if slots is None else slots
    q, k, v = split(proj, hk, hv, dk, dv)
    spans = [(i, i + 1) for i in range(live)]
    want = recurrence(q, k, v, g, beta, state, spans, order.tolist(), norm, dk ** -0.5 if scale is None else scale)
    dq, dk_, dv_ = split(proj.to(dev), hk, hv, dk, dv)
    ds = state.to(dev)
    out = torch.full((T, hv, dv), float("nan"), device=dev)
    delta.step(dq, dk_, dv_, g.to(dev), beta.to(dev), ds, out, torch.tensor([live], dtype=torch.int32, device=dev), T,
               slots=order.to(dev), norm=norm, scale=scale)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want[0]))          # the other rows untouched
    compare(out, ds, *want, spans, v, dk, state)
    mine = [int(s) for s in order[:live] if 0 <= s < states]
    rest = [i for i in range(states) if i not in mine]
    assert torch.equal(ds.cpu()[rest], state[rest])


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("T,live,hk,hv", [(1, 1, 16, 48), (3, 2, 4, 4), (48, 40, 2, 4), (130, 130, 1, 3)])
def test_step(dev, T, live, hk, hv, dk, dv):
    run_step(dev, T, live, hk, hv, dk, dv, seed=T + dk)


def test_step_without_norm_and_with_scale(dev):
    run_step(dev, 5, 5, 2, 6, 128, 128, norm=False, scale=0.37, seed=9)


def test_step_slots_out_of_range(dev):
    run_step(dev, 4, 4, 2, 2, 64, 64, slots=torch.tensor([3, -1, 4, 0], dtype=torch.int32), states=4)


def test_step_edge_gates(dev):
    """Decay 1, a decay that clears the state (-inf), beta 0 and 1, a key and a query of zeros."""
    def edit(qkv, g, beta, state):
        q, k, v = qkv
        g[0], g[1], beta[2], beta[3] = 0.0, float("-inf"), 0.0, 1.0
        k[4], q[5] = 0, 0
    run_step(dev, 6, 6, 2, 4, 128, 128, edit=edit)


def run_prefill(dev, lens, hk, hv, dk, dv, norm=True, scale=None, seed=0, edit=None, tail=0, slots=None):
    from prism_amd import delta
    T = sum(lens) + tail
    states = len(lens) + 1
    proj, g, beta, state = inputs(T, hk, hv, dk, dv, states, seed)
    if not norm:
        proj *= dk ** -0.5
    if edit:
        edit(split(proj, hk, hv, dk, dv), g, beta, state)
    cu = [sum(lens[:i]) for i in range(len(lens) + 1)]
    spans = list(zip(cu, cu[1:]))
    order = torch.randperm(states, generator=torch.Generator().manual_seed(seed))[:len(lens)].int() if slots is None \
        else torch.tensor(slots, dtype=torch.int32)
    q, k, v = split(proj, hk, hv, dk, dv)
    want = recurrence(q, k, v, g, beta, state, spans, order.tolist(), norm, dk ** -0.5 if scale is None else scale)
    dq, dk_, dv_ = split(proj.to(dev), hk, hv, dk, dv)
    ds = state.to(dev)
    out = torch.full((T, hv, dv), float("nan"), device=dev)
    args = (dq, dk_, dv_, g.to(dev), beta.to(dev), ds, out, torch.tensor(cu, dtype=torch.int32, device=dev), T)
    delta.prefill(*args, slots=order.to(dev), norm=norm, scale=scale)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want[0]))
    compare(out, ds, *want, spans, v, dk, state)
    mine = [int(s) for s, n in zip(order, lens) if n and 0 <= s < states]
    rest = [i for i in range(states) if i not in mine]
    assert torch.equal(ds.cpu()[rest], state[rest])
    first = out.clone(), ds.clone()
    ds.copy_(state)
    delta.prefill(*args, slots=order.to(dev), norm=norm, scale=scale)
    assert torch.equal(torch.nan_to_num(first[0]), torch.nan_to_num(out)) and torch.equal(first[1], ds)    # same bits


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("lens", [[1], [2], [31], [63], [64], [65], [200], [0, 1, 0, 130, 64, 5, 0]])
def test_prefill_lengths(dev, lens, dk, dv):
    run_prefill(dev, lens, 2, 4, dk, dv, seed=sum(lens) + dk + dv)


@pytest.mark.parametrize("hk,hv", [(1, 1), (1, 5), (4, 12), (16, 48)])
def test_prefill_heads(dev, hk, hv):
    run_prefill(dev, [70, 3], hk, hv, 128, 128, seed=hv)


def test_prefill_long(dev):
    run_prefill(dev, [1500, 17], 1, 2, 128, 128, seed=3)


def test_prefill_many_sequences_and_rows_of_none(dev):
    run_prefill(dev, [3, 70, 0, 1, 64, 129, 2, 90] * 3, 1, 2, 64, 64, seed=5, tail=9)


def test_prefill_without_norm_and_with_scale(dev):
    run_prefill(dev, [150], 2, 2, 128, 128, norm=False, scale=0.37, seed=9)


def test_prefill_skips_slots_out_of_range(dev):
    run_prefill(dev, [70, 5, 66], 1, 2, 64, 64, seed=2, slots=[1, 9, 0])
    run_prefill(dev, [70, 5, 66], 1, 2, 64, 64, seed=2, slots=[-1, 2, 3])


@pytest.mark.parametrize("gate", ["none", "clear", "strong", "mixed"])
def test_prefill_edge_gates(dev, gate):
    """No decay at all; states cleared in the middle of a chunk (-inf) with gentle decays around it; decays that leave
    nothing; all of them together, with betas of 0 and 1 and zero keys and queries."""
    def edit(qkv, g, beta, state):
        q, k, v = qkv
        if gate in ("none", "mixed"):
            g[10:100] = 0.0
            beta[20:60:3], beta[21:60:3] = 0.0, 1.0
            k[33], q[40] = 0, 0
        if gate in ("clear", "mixed"):
            g[5], g[64], g[130], g[131] = (float("-inf"),) * 4
        if gate in ("strong", "mixed"):
            g[140:150] = -1000.0
            g[150:170] = -30.0
    run_prefill(dev, [190], 2, 4, 128, 128, edit=edit, seed=6)


def test_prefill_repeated_keys(dev):
    """Keys all alike with beta 1 and no decay: the chunk's triangular system at its worst conditioned."""
    def edit(qkv, g, beta, state):
        qkv[1][:] = qkv[1][:1].clone()
        g[:], beta[:] = 0.0, 1.0
    run_prefill(dev, [130], 1, 2, 128, 128, edit=edit, seed=7)


def test_prefill_continues_a_prompt(dev):
    """A prompt in two calls, cut inside a chunk, and then token by token, gives what one call gives (within both
    calls' tolerance)."""
    from prism_amd import delta
    T, hk, hv, dk, dv = 100, 2, 4, 128, 128
    proj, g, beta, state = (x.to(dev) for x in inputs(T, hk, hv, dk, dv, 1, 11))
    q, k, v = split(proj, hk, hv, dk, dv)
    one, two = state.clone(), state.clone()
    a, b = (torch.empty(T, hv, dv, device=dev) for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)     # noqa: E731
    delta.prefill(q, k, v, g, beta, one, a, ints(0, T), T)
    for lo, hi in ((0, 37), (37, 90)):
        delta.prefill(q[lo:hi], k[lo:hi], v[lo:hi], g[lo:hi], beta[lo:hi], two, b[lo:hi], ints(0, hi - lo), hi - lo)
    for t in range(90, T):
        delta.step(q[t:t + 1], k[t:t + 1], v[t:t + 1], g[t:t + 1], beta[t:t + 1], two, b[t:t + 1], None, 1)
    assert float((a - b).norm()) <= 3e-6 * float(a.norm()) and float((one - two).norm()) <= 3e-6 * float(one.norm())


def test_captured_on_another_stream(dev):
    """step and prefill captured on a side stream: every replay gives the eager call's bits."""
    from prism_amd import delta
    T, hk, hv, dk, dv = 90, 2, 4, 64, 128
    proj, g, beta, state = (x.to(dev) for x in inputs(T, hk, hv, dk, dv, 3, 12))
    q, k, v = split(proj, hk, hv, dk, dv)
    cu = torch.tensor([0, 80, 90], dtype=torch.int32, device=dev)
    n = torch.tensor([2], dtype=torch.int32, device=dev)
    work, out, last = state.clone(), torch.zeros(T, hv, dv, device=dev), torch.zeros(2, hv, dv, device=dev)

    def both():
        delta.prefill(q, k, v, g, beta, work, out, cu, T)
        delta.step(q[:2], k[:2], v[:2], g[:2], beta[:2], work, last, n, 2)
    both()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        both()
    for cut in (80, 3, 90, 64):
        cu.copy_(torch.tensor([0, cut, 90], dtype=torch.int32))
        work.copy_(state)
        both()
        torch.cuda.synchronize()
        want = work.clone(), out.clone(), last.clone()
        work.copy_(state)
        out.zero_(), last.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(work, want[0]) and torch.equal(out, want[1]) and torch.equal(last, want[2])
