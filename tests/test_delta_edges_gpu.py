"""prism_amd.delta on the GPU where its forms can go wrong: normalising without an eps, values of very different sizes or
not finite, clones, empty calls, many sequences, strides with gaps.  Checks and tolerances are test_delta_gpu's."""
import pytest
import torch

from test_delta_gpu import compare, inputs, recurrence, split

pytestmark = pytest.mark.gpu


def check_prefill(dev, lens, hk, hv, dk, dv, seed=0, eps=1e-6, lead=0, tail=0):
    """Prompts of these lengths after `lead` rows of none, `tail` rows of none behind; every state and row of out checked."""
    from prism_amd import delta
    T, states = lead + sum(lens) + tail, len(lens) + 1
    proj, g, beta, state = inputs(T, hk, hv, dk, dv, states, seed)
    cu = [lead + sum(lens[:i]) for i in range(len(lens) + 1)]
    spans = list(zip(cu, cu[1:]))
    slots = torch.randperm(states, generator=torch.Generator().manual_seed(seed))[:len(lens)].int()
    q, k, v = split(proj, hk, hv, dk, dv)
    want = recurrence(q, k, v, g, beta, state, spans, slots.tolist(), True, dk ** -0.5, eps)
    dq, dk_, dv_ = split(proj.to(dev), hk, hv, dk, dv)
    ds, out = state.to(dev), torch.full((T, hv, dv), float("nan"), device=dev)
    delta.prefill(dq, dk_, dv_, g.to(dev), beta.to(dev), ds, out, torch.tensor(cu, dtype=torch.int32, device=dev), T,
                  slots=slots.to(dev), eps=eps)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want[0]))
    compare(out, ds, *want, spans, v, dk, state)


@pytest.mark.parametrize("eps", [0.0, 1e-60])                    # (the second is 0 in fp32)
@pytest.mark.parametrize("lens", [[1], [5], [64], [65], [77], [130], [70, 0, 3, 129, 64, 31]])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
def test_prefill_without_eps(dev, lens, eps, dk, dv):
    """Lengths that leave a chunk unfilled: the rows past its end have no length to divide by."""
    check_prefill(dev, lens, 2, 4, dk, dv, seed=sum(lens), eps=eps)


@pytest.mark.parametrize("what,factor", [("value", 2.0 ** 20), ("value", 2.0 ** 40), ("value", 2.0 ** 70), ("key", 2.0 ** 20)])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
def test_prefill_tokens_keep_their_own_size(dev, what, factor, dk, dv):
    """One token far above the others, and the state cleared some tokens later: the tokens before the one and from the
    clearing on are held to the bounds of their own sizes, as if the large one were not there.  (A large key makes the
    update no contraction: its state is cleared at once, and its own token is not held to anything.)"""
    from prism_amd import delta
    T, hk, hv, big, clear = 190, 2, 4, 100, 140 if what == "value" else 101
    norm = what == "value"
    proj, g, beta, state = inputs(T, hk, hv, dk, dv, 1, 21)
    if not norm:
        proj *= dk ** -0.5
    q, k, v = split(proj, hk, hv, dk, dv)
    (v if what == "value" else k)[big] *= factor
    g[clear] = float("-inf")
    want_out, want_state = recurrence(q, k, v, g, beta, state, [(0, T)], [0], norm, dk ** -0.5)
    dq, dk_, dv_ = split(proj.to(dev), hk, hv, dk, dv)
    ds, out = state.to(dev), torch.empty(T, hv, dv, device=dev)
    delta.prefill(dq, dk_, dv_, g.to(dev), beta.to(dev), ds, out, torch.tensor([0, T], dtype=torch.int32, device=dev), T,
                  norm=norm)
    for begin, end in ((0, big), (clear, T)) + (((big, clear),) if norm else ()):
        part = torch.full_like(want_out, float("nan"))
        part[begin:end] = want_out[begin:end]
        compare(out, ds, part, want_state, [(begin, end)], v[begin:end], dk, state)


@pytest.mark.parametrize("form", ["step", "prefill"])
def test_clones_keep_what_they_were_made_of(dev, form):
    """States and outputs that are copy-on-write clones: the tensors they were made of stay as they are."""
    from prism_amd import delta
    T, hk, hv, dk, dv = 20, 2, 4, 64, 64
    proj, g, beta, state = (x.to(dev) for x in inputs(T, hk, hv, dk, dv, T, 31))
    q, k, v = split(proj, hk, hv, dk, dv)
    out = torch.zeros(T, hv, dv, device=dev)
    s, o = torch._lazy_clone(state), torch._lazy_clone(out)
    before = state.clone()
    if form == "step":
        delta.step(q, k, v, g, beta, s, o, None, T)
    else:
        delta.prefill(q, k, v, g, beta, s, o, torch.tensor([0, T], dtype=torch.int32, device=dev), T)
    assert torch.equal(state, before) and (out == 0).all()
    assert not torch.equal(s, state) and (o != 0).any()


@pytest.mark.parametrize("T,slots", [(0, 3), (0, 0), (5, 0)])
def test_calls_without_rows_or_states(dev, T, slots):
    """No rows, no prompts, or no state that a sequence could have: nothing is done."""
    from prism_amd import delta
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)             # noqa: E731
    f = lambda *s: torch.zeros(*s, device=dev)                                    # noqa: E731
    state, out = f(slots, 4, 64, 128) + 2, f(T, 4, 128) + 3
    args = (bf(T, 2, 64), bf(T, 2, 64), bf(T, 4, 128), f(T, 4), f(T, 4), state, out)
    delta.step(*args, torch.tensor([T], dtype=torch.int32, device=dev), T)
    delta.prefill(*args, torch.tensor([0, T], dtype=torch.int32, device=dev), T)
    delta.prefill(*args, torch.zeros(1, dtype=torch.int32, device=dev), T)
    assert (state == 2).all() and (out == 3).all()


def test_prefill_more_sequences_than_a_wave_has_lanes(dev):
    """130 short and empty prompts, some of more than a chunk and some past the 64th, rows of none on both sides."""
    lens = [(7 * i * i + 3 * i) % 9 for i in range(130)]
    lens[3], lens[63], lens[64], lens[90], lens[129] = 70, 129, 65, 64, 200
    check_prefill(dev, lens, 1, 2, 64, 64, seed=41, lead=5, tail=3)


@pytest.mark.parametrize("lead", [1, 5, 63, 64, 70])
def test_prefill_rows_before_the_first_sequence(dev, lead):
    check_prefill(dev, [130, 0, 7, 64], 1, 2, 64, 128, seed=lead, lead=lead, tail=2)


@pytest.mark.parametrize("form", ["step", "prefill"])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128)])
def test_rows_and_slots_with_gaps(dev, form, dk, dv):
    """out between other columns, padded state slots, gates as column ranges of wider rows: the same bits as from whole
    tensors, and nothing beside them written."""
    from prism_amd import delta
    hk, hv, T, seqs = 2, 4, 90, 3
    proj, g, beta, state = (x.to(dev) for x in inputs(T, hk, hv, dk, dv, T, 51))
    q, k, v = split(proj, hk, hv, dk, dv)
    count = torch.tensor([T] if form == "step" else [0, 60, 61, T], dtype=torch.int32, device=dev)
    call = delta.step if form == "step" else delta.prefill
    states = T if form == "step" else seqs

    want_s, want_o = state[:states].clone(), torch.zeros(T, hv, dv, device=dev)
    call(q, k, v, g, beta, want_s, want_o, count, T)

    wide_o = torch.full((T, hv + 2, dv + 8), 7.0, device=dev)
    size = hv * dk * dv
    wide_s = torch.full((states, size + 12), 7.0, device=dev)
    s = wide_s.as_strided((states, hv, dk, dv), (size + 12, dk * dv, dv, 1))
    s.copy_(state[:states])
    gates = torch.cat([torch.full((T, 3), 9.0, device=dev), g, beta, torch.full((T, 2), 9.0, device=dev)], 1)
    o = wide_o[:, 1:hv + 1, 4:dv + 4]
    call(q, k, v, gates[:, 3:hv + 3], gates[:, hv + 3:2 * hv + 3], s, o, count, T)
    assert torch.equal(o, want_o) and torch.equal(s, want_s)
    o.fill_(7.0)
    assert (wide_o == 7).all() and (wide_s[:, size:] == 7).all()


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("where", ["v", "k", "state", "g"])
def test_prefill_values_that_are_not_finite_stay_in_their_sequence_and_head(dev, bad, where):
    """Other sequences, other heads and earlier chunks of the same sequence keep their bits; the sequence's later rows and
    its state show it."""
    from prism_amd import delta
    hk, hv, dk, dv, T = 2, 4, 128, 64, 300
    proj, g, beta, state = (x.to(dev) for x in inputs(T, hk, hv, dk, dv, 3, 61))
    cu = torch.tensor([0, 90, 240, T], dtype=torch.int32, device=dev)

    def run():
        q, k, v = split(proj, hk, hv, dk, dv)
        s, o = state.clone(), torch.zeros(T, hv, dv, device=dev)
        delta.prefill(q, k, v, g, beta, s, o, cu, T)
        return o, s
    want_o, want_s = run()
    _, k, v = split(proj, hk, hv, dk, dv)
    t, first = 160, 154                                          # sequence 1, its second chunk (rows 154 .. 217)
    if where == "v":
        v[t, 2, 5] = bad
    elif where == "k":
        k[t, 1, 5] = bad
    elif where == "g":
        g[t, 2] = bad if bad != bad else float("nan")
    else:
        state[1, 2, 3, 4], first = bad, 90
    heads = [2, 3] if where == "k" else [2]                      # (a key head's value heads)
    o, s = run()
    clean = torch.ones(T, hv, dtype=torch.bool, device=dev)
    clean[first:240, heads] = False
    assert torch.equal(o[clean], want_o[clean])
    rest = torch.ones(3, hv, dtype=torch.bool, device=dev)
    rest[1, heads] = False
    assert torch.equal(s[rest], want_s[rest])
    assert not torch.isfinite(o[t, 2]).all() and not torch.isfinite(s[1, 2]).all()
