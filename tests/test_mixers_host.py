"""The token mixers' host path on the CPU: what it does to the tensors before the call is refused for want of a GPU."""
import os

import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from prism_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libprism_amd.so not built (run __graft_entry__.build())")


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def calls():
    """name -> (function, arguments, the outputs among them)"""
    from prism_amd import delta, kv
    kc, vc = kv.cache(4, 16, 2, 64, device="cpu")
    f = torch.zeros
    rec = dict(q=_bf(5, 2, 64), k=_bf(5, 2, 64), v=_bf(5, 4, 128), g=f(5, 4), beta=f(5, 4), state=f(6, 4, 64, 128),
               out=f(5, 4, 128), T=5)
    return {
        "append": (kv.append, dict(q=_bf(3, 4, 64), k=_bf(3, 2, 64), v=_bf(3, 2, 64), rope=f(9, 32), pos=_i32(3),
                                   table=_i32(3, 4), k_cache=kc, v_cache=vc, q_out=_bf(3, 4, 64), n=_i32(1), T=3),
                   ("q_out", "k_cache", "v_cache")),
        "attend": (kv.attend, dict(q=_bf(3, 4, 64), k_cache=kc, v_cache=vc, table=_i32(3, 4), lens=_i32(3),
                                   out=_bf(3, 4, 64), n=_i32(1), T=3), ("out",)),
        "step": (delta.step, dict(rec, n=_i32(1)), ("state", "out")),
        "prefill": (delta.prefill, dict(rec, cu=_i32(3)), ("state", "out")),
    }


@pytest.mark.parametrize("name", ["append", "attend", "step", "prefill"])
def test_outputs_that_are_copy_on_write_clones(name):
    """Every output is given memory of its own before its pointer is taken, and no input is."""
    fn, args, outputs = calls()[name]
    lazy = {k: torch._lazy_clone(x) if torch.is_tensor(x) else x for k, x in args.items()}
    with pytest.raises(RuntimeError):                            # no GPU tensors
        fn(**lazy)
    for k, x in lazy.items():
        if torch.is_tensor(x):
            assert torch._C._is_cow_tensor(x) == (k not in outputs), k


@pytest.mark.parametrize("name", ["append", "attend", "step", "prefill"])
def test_expanded_outputs_are_refused(name):
    """An output of which several rows, heads or pages are one place is refused; inputs may be expanded."""
    fn, args, outputs = calls()[name]
    for k, x in args.items():
        if not torch.is_tensor(x):
            continue
        for d in range(x.dim() - 1):
            if x.shape[d] > 1:
                wide = {**args, k: x.narrow(d, 0, 1).expand(x.shape)}
                with pytest.raises(ValueError if k in outputs else RuntimeError):
                    fn(**wide)
