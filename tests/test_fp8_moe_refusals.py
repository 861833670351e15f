"""What fp8 and moe refuse, on the CPU: the C entries' codes (placeholders that are never dereferenced) and the Python layer's
TypeError / ValueError before any call; outputs that are expanded or copy-on-write clones."""
import os
import re
import struct

import pytest
import torch

QUANT, GEMM = struct.Struct("10q"), struct.Struct("15q")
ROUTE, EXPERTS = struct.Struct("14q d"), struct.Struct("23q")
OK, SHAPE, ALIGN, ARG = 0, 1, 2, 3
P, U = 0x100000, 0x100001
E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    from prism_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libprism_amd.so not built (run __graft_entry__.build())")
    return _lib.lib()


def packed(layout, *fields):
    return layout.pack(*(0 if f is None else f for f in fields))


def test_packed_layouts_match_the_header():
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "prism_amd.h")).read()
    count = {name: sum(len(f.split(",")) for f in body.split(";") if f.strip())
             for body, name in re.findall(r"typedef struct \{([^{}]*?)\} (prism_\w+);", src, re.S)}
    for layout, name in ((QUANT, "fp8_quant"), (GEMM, "fp8_gemm"), (ROUTE, "moe_route"), (EXPERTS, "moe_experts")):
        assert layout.size == 8 * count[f"prism_{name}_args"], name


def test_quant_codes(lib):
    def call(x=P, f32=0, x_ld=256, q=P, q_ld=256, s=P, s_ld=2, n=P, T=0, k=256):
        return lib.prism_fp8_quant(packed(QUANT, x, f32, x_ld, q, q_ld, s, s_ld, n, T, k), None)
    assert lib.prism_fp8_quant(None, None) == ARG
    assert call() == OK
    assert call(x=None) == ARG and call(q=None) == ARG and call(s=None) == ARG and call(n=None) == ARG and call(f32=2) == ARG
    assert call(T=-1) == SHAPE and call(k=0) == SHAPE and call(k=2 ** 21) == SHAPE
    assert call(T=2, q_ld=248) == SHAPE and call(T=2, s_ld=1) == SHAPE
    assert call(q=P + 4) == ALIGN and call(q_ld=260) == ALIGN


def test_gemm_codes(lib):
    def call(a=P, a_ld=256, sa=P, as_ld=2, w=P, ws=P, out=P, o_ld=64, n=P, T=0, N=64, K=256, epi=0, wsp=None, wsp_bytes=0):
        return lib.prism_fp8_gemm(packed(GEMM, a, a_ld, sa, as_ld, w, ws, out, o_ld, n, T, N, K, epi, wsp, wsp_bytes), None)
    assert lib.prism_fp8_gemm(None, None) == ARG
    assert call() == OK
    for name in ("a", "sa", "w", "ws", "out", "n"):
        assert call(**{name: None}) == ARG, name
    assert call(epi=2) == ARG and call(T=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE and call(K=2 ** 21) == SHAPE
    assert call(T=2, o_ld=63) == SHAPE and call(a_ld=2 ** 23) == SHAPE
    assert call(a=U) == ALIGN and call(w=U) == ALIGN and call(a_ld=264) == ALIGN and call(out=U) == ALIGN and call(epi=1, out=P + 2) == ALIGN
    need = lib.prism_fp8_gemm_workspace_bytes(150, 512, 4096)
    assert need > 0 and lib.prism_fp8_gemm_workspace_bytes(1, 512, 4096) == 0 == lib.prism_fp8_gemm_workspace_bytes(0, 512, 4096)
    big = dict(T=150, N=512, K=4096, a_ld=4096, as_ld=32, o_ld=512)
    assert call(**big) == ARG and call(**big, wsp=P, wsp_bytes=need - 1) == ARG and call(**big, wsp=U, wsp_bytes=need) == ALIGN


def test_pack_codes(lib):
    def call(w=P, f32=1, ld=64, c=P, s=P, n=32, k=64):
        return lib.prism_fp8_pack(w, f32, ld, c, s, n, k, None)
    assert call(w=None) == ARG and call(c=None) == ARG and call(s=None) == ARG and call(f32=3) == ARG
    assert call(n=0) == SHAPE and call(k=0) == SHAPE and call(ld=63) == SHAPE and call(n=2 ** 21) == SHAPE and call(c=P + 8) == ALIGN


def test_route_codes(lib):
    def call(x=P, f32=1, x_ld=64, bias=None, ids=P, ids_ld=4, w=P, w_ld=4, n=P, T=0, E=64, top=4, sig=0, renorm=1, scale=1.0):
        return lib.prism_moe_route(packed(ROUTE, x, f32, x_ld, bias, ids, ids_ld, w, w_ld, n, T, E, top, sig, renorm, scale),
                                   None)
    assert lib.prism_moe_route(None, None) == ARG
    assert call() == OK and call(sig=1, bias=P) == OK
    assert call(x=None) == ARG and call(ids=None) == ARG and call(w=None) == ARG and call(n=None) == ARG
    assert call(f32=2) == ARG and call(sig=2) == ARG and call(renorm=2) == ARG and call(bias=P) == ARG
    assert call(T=-1) == SHAPE and call(E=0) == SHAPE and call(E=1025) == SHAPE and call(top=0) == SHAPE
    assert call(top=17) == SHAPE and call(E=3) == SHAPE and call(T=2, ids_ld=3) == SHAPE and call(T=2, w_ld=3) == SHAPE
    assert call(x=U) == ALIGN and call(ids=U) == ALIGN and call(w=U) == ALIGN


def test_experts_codes(lib):
    def call(x=P, x_ld=64, ids=P, ids_ld=2, w=P, w_ld=2, gate=P, gs=P, up=P, us=P, down=P, ds=P, out=P, o_ld=64, n=P, T=0, E=8,
             top=2, H=64, I=32, epi=0, wsp=None, wsp_bytes=0):
        return lib.prism_moe_experts(packed(EXPERTS, x, x_ld, ids, ids_ld, w, w_ld, gate, gs, up, us, down, ds, out, o_ld, n, T, E,
                                            top, H, I, epi, wsp, wsp_bytes), None)
    assert lib.prism_moe_experts(None, None) == ARG
    assert call() == OK
    for name in ("x", "ids", "w", "gate", "gs", "up", "us", "down", "ds", "out", "n"):
        assert call(**{name: None}) == ARG, name
    assert call(epi=2) == ARG
    assert call(T=-1) == SHAPE and call(E=0) == SHAPE and call(E=32768) == SHAPE and call(top=0) == SHAPE and call(top=17) == SHAPE
    assert call(H=8) == SHAPE and call(I=40) == SHAPE and call(H=72) == SHAPE and call(T=2, o_ld=63) == SHAPE
    assert call(I=2 ** 20, top=16) == SHAPE                      # a pass's hidden values would pass 31-bit offsets
    assert call(x=U) == ALIGN and call(x_ld=68) == ALIGN and call(gate=U) == ALIGN and call(up=U) == ALIGN and call(down=U) == ALIGN
    assert call(out=U) == ALIGN and call(out=P + 2, epi=1) == ALIGN
    need = lib.prism_moe_experts_workspace_bytes(3, 2, 64, 32)
    assert need > 0 and lib.prism_moe_experts_workspace_bytes(0, 2, 64, 32) == 0
    assert call(T=3) == ARG and call(T=3, wsp=P, wsp_bytes=need - 1) == ARG and call(T=3, wsp=U, wsp_bytes=need) == ALIGN


# ----------------------------------------------------------------------------------------------------------- the Python layer
def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _e4(*shape):
    return torch.zeros(*shape).to(E4)


def calls():
    """name -> (function, arguments, the outputs among them)"""
    from prism_amd import fp8, moe
    f = torch.zeros

    def w(n, k, *e):
        return fp8.from_rows(_e4(*e, n, k), f(*e, -(-n // 128), -(-k // 128)))
    return {
        "quant": (fp8.quantize_act, dict(x=_bf(3, 200), q=_e4(3, 256), s=f(3, 2), n=_i32(1), T=3), ("q", "s")),
        "gemm": (fp8.gemm, dict(a_q=_e4(3, 256), a_s=f(3, 2), w=w(40, 200), out=_bf(3, 40), n=_i32(1), T=3), ("out",)),
        "route": (moe.route, dict(logits=f(3, 20), ids=_i32(3, 4), weights=f(3, 4), n=_i32(1), T=3), ("ids", "weights")),
        "experts": (moe.experts, dict(x=_bf(3, 160), ids=_i32(3, 2), weights=f(3, 2), gate=w(48, 160, 5), up=w(48, 160, 5),
                                      down=w(160, 48, 5), out=_bf(3, 160), n=_i32(1), T=3), ("out",)),
    }


NAMES = ["quant", "gemm", "route", "experts"]


@pytest.mark.parametrize("name", NAMES)
def test_good_arguments_pass_the_checks(lib, name):
    """... and are refused only for want of a GPU; buffers may have more rows than T, and T may be 0."""
    fn, args, _ = calls()[name]
    for T in (3, 2, 0):
        with pytest.raises(RuntimeError, match="GPU"):
            fn(**{**args, "T": T})


@pytest.mark.parametrize("name", NAMES)
def test_wrong_tensors(lib, name):
    fn, args, outputs = calls()[name]
    for k, x in args.items():
        if k == "T":
            bad = ["3", None, 4]                                 # more rows than the buffers have
        elif not torch.is_tensor(x):
            bad = [x.q, (x.q, x.s, x.n), x._replace(n=x.n + 16), x._replace(k=x.k + 128), x._replace(q=x.q[..., :1024]),
                   x._replace(s=x.s.half()), x._replace(s=x.s[..., :0]), x._replace(q=x.q.transpose(-1, -2)), x._replace(n=0)]
        elif k == "n":
            bad = [x.float(), 3]
        else:
            bad = [x.double(), x[0], x[:2], x[:, :-1], torch.cat([x, x], 1)[:, ::2], "x"]
            if k in ("logits", "ids", "x"):                      # (their widths are the call's sizes)
                bad = [b for i, b in enumerate(bad) if i != 3 or name == "experts" and k == "x"]
        for b in bad:
            with pytest.raises((TypeError, ValueError)):
                fn(**{**args, k: b})
    with pytest.raises(TypeError):
        fn(**{**args, "bogus": 1})


def test_wrong_values(lib):
    c = calls()
    fn, a, _ = c["gemm"]
    for bad in (dict(epi=2), dict(epi="x"), dict(epi=1), dict(T=-1, a_q=_e4(0, 256))):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            fn(**{**a, **bad})
    fn, a, _ = c["route"]
    for bad in (dict(score="tanh"), dict(score=None), dict(bias=torch.zeros(20)), dict(bias=torch.zeros(19), score="sigmoid"),
                dict(ids=_i32(3, 21), weights=torch.zeros(3, 21)), dict(ids=_i32(3, 17), weights=torch.zeros(3, 17)),
                dict(ids=_i32(3, 0), weights=torch.zeros(3, 0)), dict(logits=torch.zeros(3, 1025)), dict(scale="x"),
                dict(ids=_i32(3, 5))):
        with pytest.raises((TypeError, ValueError)):
            fn(**{**a, **bad})
    fn, a, _ = c["experts"]
    for bad in (dict(epi=1), dict(gate=a["down"]), dict(down=a["gate"]), dict(ids=_i32(3, 17), weights=torch.zeros(3, 17)),
                dict(ids=_i32(3, 3))):
        with pytest.raises((TypeError, ValueError)):
            fn(**{**a, **bad})
    from prism_amd import fp8

    def w(n, k):
        return fp8.from_rows(_e4(5, n, k), torch.zeros(5, -(-n // 128), -(-k // 128)))
    with pytest.raises(ValueError, match="16"):
        fn(**{**a, "gate": w(40, 160), "up": w(40, 160), "down": w(160, 40)})
    one = fp8.from_rows(_e4(48, 160), torch.zeros(1, 2))
    with pytest.raises(ValueError):
        fn(**{**a, "gate": one})


def test_weights_refused(lib):
    from prism_amd import fp8
    for q, s in ((torch.zeros(3, 4), torch.zeros(1, 1)), (_e4(4), torch.zeros(1, 1)), (_e4(130, 4), torch.zeros(1, 1)),
                 (_e4(3, 4), torch.zeros(1, 1).double()), (_e4(2, 3, 4), torch.zeros(1, 1)), (_e4(0, 4), torch.zeros(0, 1))):
        with pytest.raises(ValueError):
            fp8.from_rows(q, s)
    for w in (torch.zeros(3, 4).half(), torch.zeros(4), torch.zeros(0, 4)):
        with pytest.raises(ValueError):
            fp8.pack(w)
    with pytest.raises(RuntimeError, match="GPU"):
        fp8.pack(torch.zeros(3, 4))


def test_weights_layout():
    """from_rows on the CPU: to_rows gives the bytes back, at sizes that are no whole tiles."""
    from prism_amd import fp8
    for shape in ((1, 1), (17, 129), (40, 300), (3, 33, 128)):
        q = torch.randint(0, 256, shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
        s = torch.randn(*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128))
        w = fp8.from_rows(q, s)
        q2, s2 = fp8.to_rows(w)
        assert torch.equal(q2.view(torch.uint8), q) and torch.equal(s2, s) and w.shape == tuple(shape)
        assert w.q.long().sum() == q.long().sum()                # the padding is zeros


@pytest.mark.parametrize("name", NAMES)
def test_outputs_that_are_copy_on_write_clones(lib, name):
    fn, args, outputs = calls()[name]
    lazy = {k: torch._lazy_clone(x) if torch.is_tensor(x) else x for k, x in args.items()}
    with pytest.raises(RuntimeError):
        fn(**lazy)
    for k, x in lazy.items():
        if torch.is_tensor(x):
            assert torch._C._is_cow_tensor(x) == (k not in outputs), k


@pytest.mark.parametrize("name", NAMES)
def test_expanded_outputs_are_refused(lib, name):
    fn, args, outputs = calls()[name]
    for k, x in args.items():
        if not torch.is_tensor(x) or k == "n":
            continue
        wide = {**args, k: x.narrow(0, 0, 1).expand(x.shape)}
        with pytest.raises(ValueError if k in outputs else RuntimeError):
            fn(**wide)
