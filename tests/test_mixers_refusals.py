"""What the token mixers refuse, on the CPU: the C entries' codes for bad pointers, sizes and alignment (placeholders that
are never dereferenced), and the Python layer's TypeError / ValueError before any call."""
import os
import struct
import types

import pytest
import torch

# the C entries' structs: 8-byte fields, floating ones as doubles
L = types.SimpleNamespace(_APPEND=struct.Struct("19q 12q 5q 5q"), _ATTEND=struct.Struct("19q 6q 4q d 2q"),
                          _ARGS=struct.Struct("9q 4q 4q 3q q 7q 2d 2q"))
OK, SHAPE, ALIGN, ARG = 0, 1, 2, 3
P, U = 0x100000, 0x100001


@pytest.fixture(scope="module")
def lib():
    from prism_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("libprism_amd.so not built (run __graft_entry__.build())")
    return _lib.lib()


def packed(layout, *fields):
    return layout.pack(*(0 if f is None else f for f in fields))


def test_packed_layouts_match_the_header():
    """The layouts above have as many 8-byte fields as the header's structs declare."""
    import re
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "prism_amd.h")).read()
    count = {}
    for body, name in re.findall(r"typedef struct \{(.*?)\} (prism_\w+);", src, re.S):
        count[name] = sum(count["prism_kv_cache"] if f.split()[0] == "prism_kv_cache" else len(f.split(","))
                          for f in body.split(";") if f.strip())
    for layout, name in ((L._APPEND, "prism_kv_append_args"), (L._ATTEND, "prism_kv_attend_args"),
                         (L._ARGS, "prism_delta_args")):
        assert layout.size == 8 * count[name], name


def test_append_codes(lib):
    def call(q=P, k=P, rope=P, rot=64, ldr=64, adjacent=0, pos=P, kc=P, tok=128, e4m3=0, ks=None, cols=4, pages=8,
             page=16, T=1, HQ=2, D=64, ldk=128, qo=P):
        return lib.prism_kv_append(packed(
            L._APPEND, kc, 4096, tok, 64, P, 4096, tok, 64, e4m3, ks, None, P, 4, 2, cols, pages, page, 2, D,
            q, 256, 64, k, ldk, 64, P, 128, 64, qo, 128, 64, rope, ldr, 100, rot, adjacent, pos, None, P, T, HQ), None)
    assert lib.prism_kv_append(None, None) == ARG
    assert call(T=0) == OK and call(T=0, HQ=0, q=None, qo=None) == OK and call(T=0, rot=0, rope=None, ldr=0) == OK
    assert call(k=None) == ARG and call(q=None) == ARG and call(rope=None) == ARG and call(pos=None) == ARG
    assert call(adjacent=2) == ARG and call(e4m3=2) == ARG and call(ks=P) == ARG      # a bf16 cache has no scales
    assert call(D=96) == SHAPE and call(rot=24) == SHAPE and call(rot=80) == SHAPE and call(ldr=32) == SHAPE
    assert call(page=8) == SHAPE and call(page=48) == SHAPE and call(pages=0) == SHAPE and call(cols=5) == SHAPE
    assert call(T=-1) == SHAPE and call(tok=(1 << 26) + 8) == SHAPE
    assert call(k=U) == ALIGN and call(kc=U) == ALIGN and call(tok=132) == ALIGN and call(ldk=130) == ALIGN
    assert call(e4m3=1, tok=136) == ALIGN                        # 8 bytes: not a whole 16-byte unit


def test_attend_codes(lib):
    def call(q=P, lens=P, out=P, T=1, HQ=4, D=64, window=0, ws=P, ws_bytes=1 << 20, cols=16, page=16, ldq=256, ldo=256):
        return lib.prism_kv_attend(packed(
            L._ATTEND, P, 4096, 128, 64, P, 4096, 128, 64, 0, None, None, P, cols, T, cols, 8, page, 2, D,
            q, ldq, 64, out, ldo, 64, lens, P, HQ, window, 0.125, ws, ws_bytes), None)
    assert lib.prism_kv_attend(None, None) == ARG
    assert call(T=0) == OK
    assert call(q=None) == ARG and call(lens=None) == ARG and call(ws=None) == ARG and call(ws_bytes=64) == ARG
    assert call(HQ=3) == SHAPE and call(HQ=0) == SHAPE and call(D=32) == SHAPE and call(window=-1) == SHAPE
    assert call(T=65536) == SHAPE and call(T=-1) == SHAPE and call(page=24) == SHAPE and call(cols=1 << 27) == SHAPE
    assert call(q=U) == ALIGN and call(out=U) == ALIGN and call(ldq=260) == ALIGN and call(ldo=258) == ALIGN
    assert call(ws=U) == ALIGN
    b = lib.prism_kv_attend_workspace_bytes
    assert b(1, 8, 2, 128, 4, 16) == 0 and b(0, 8, 2, 128, 64, 16) == 0 and b(1, 9, 2, 128, 64, 16) == 0
    assert b(3, 8, 2, 128, 64, 16) > 0


def test_delta_codes(lib):
    def call(q=P, state=P, n=P, T=1, HK=2, HV=4, DK=128, DV=128, norm=1, nslots=2, stride=None, ldv=512, fn="step", seqs=1,
             ws=None, ws_bytes=0):
        return getattr(lib, "prism_delta_" + fn)(packed(
            L._ARGS, q, 256, 128, P, 256, 128, P, ldv, 128, P, 4, P, 4, state, HV * DK * DV if stride is None else stride,
            nslots, None, P, 512, 128, n, seqs, T, HK, HV, DK, DV, norm, 1.0, 1e-6, ws, ws_bytes), None)
    for fn in ("step", "prefill"):
        assert getattr(lib, "prism_delta_" + fn)(None, None) == ARG
        assert call(T=0, fn=fn) == OK
        assert call(q=None, fn=fn) == ARG and call(n=None, fn=fn) == ARG and call(norm=2, fn=fn) == ARG
        assert call(DK=96, fn=fn) == SHAPE and call(DV=256, fn=fn) == SHAPE and call(HV=5, fn=fn) == SHAPE
        assert call(HK=0, fn=fn) == SHAPE and call(T=-1, fn=fn) == SHAPE and call(stride=100, fn=fn) == SHAPE
        assert call(ldv=(1 << 24) + 8, fn=fn) == SHAPE
        assert call(q=U, fn=fn) == ALIGN and call(state=U, fn=fn) == ALIGN and call(ldv=516, fn=fn) == ALIGN
    b = lib.prism_delta_prefill_workspace_bytes
    need = b(1000, 1, 2, 4, 128, 128)
    assert need > 0 and b(1, 1, 2, 4, 128, 128) == 0 and b(1000, 1, 2, 4, 96, 128) == 0 and b(0, 1, 2, 4, 128, 128) == 0
    assert call(fn="prefill", T=1000) == ARG and call(fn="prefill", T=1000, ws=P, ws_bytes=need - 1) == ARG
    assert call(fn="prefill", T=1000, ws=U, ws_bytes=need) == ALIGN
    assert call(fn="prefill", T=1000, seqs=-1) == SHAPE and call(fn="prefill", T=1000, seqs=0) == OK


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_kv_python_checks(lib):
    from prism_amd import kv
    kc, vc = kv.cache(4, 16, 2, 64, device="cpu")
    assert kc.shape == (4, 16, 2, 64) and kc.stride(2) == 16 * 64
    good = dict(q=_bf(3, 4, 64), k=_bf(3, 2, 64), v=_bf(3, 2, 64), rope=torch.zeros(9, 32), pos=_i32(3), table=_i32(3, 4),
                k_cache=kc, v_cache=vc, q_out=_bf(3, 4, 64), n=None, T=3)

    def bad(error, **kw):
        with pytest.raises(error):
            kv.append(**{**good, **kw})
    bad(TypeError, k=torch.zeros(3, 2, 64))
    bad(TypeError, pos=torch.zeros(3, dtype=torch.int64))
    bad(TypeError, v_cache=vc.to(torch.float8_e4m3fn))
    bad(TypeError, rope=torch.zeros(9, 32, dtype=torch.float64))
    bad(ValueError, T=4)
    bad(ValueError, k=_bf(3, 4, 64))
    bad(ValueError, q_out=None)
    bad(ValueError, q=_bf(3, 64, 4).transpose(1, 2))             # no unit stride in dim
    bad(ValueError, rope=torch.zeros(9, 40))
    bad(ValueError, rope=torch.zeros(9, 80))
    bad(ValueError, pairs="quarter")
    bad(ValueError, pos=_i32(2))
    bad(ValueError, seq=_i32(2))
    bad(ValueError, k_scale=torch.ones(2))                       # a bf16 cache
    bad(ValueError, n=torch.zeros(1, dtype=torch.int64))
    k8, v8 = kv.cache(4, 16, 2, 64, dtype=torch.float8_e4m3fn, device="cpu")
    bad(ValueError, k_cache=k8, v_cache=v8, k_scale=torch.ones(3))
    bad(ValueError, k_cache=kc[:, :8], v_cache=vc[:, :8])        # a page of 8
    bad(ValueError, k_cache=_bf(4, 16, 2, 96), v_cache=_bf(4, 16, 2, 96))
    bad(RuntimeError)                                            # all well but for the device: no GPU tensors

    ok = dict(q=_bf(3, 4, 64), k_cache=kc, v_cache=vc, table=_i32(3, 4), lens=_i32(3), out=_bf(3, 4, 64), n=None, T=3)

    def no(error, **kw):
        with pytest.raises(error):
            kv.attend(**{**ok, **kw})
    no(ValueError, q=_bf(3, 3, 64), out=_bf(3, 3, 64))
    no(ValueError, table=_i32(2, 4))
    no(ValueError, lens=_i32(2))
    no(ValueError, window=-1)
    no(ValueError, out=_bf(3, 4, 128))
    no(TypeError, out=torch.zeros(3, 4, 64))
    no(TypeError, lens=torch.zeros(3, dtype=torch.int64))


def test_delta_python_checks(lib):
    from prism_amd import delta
    f = torch.zeros
    good = dict(q=_bf(5, 2, 64), k=_bf(5, 2, 64), v=_bf(5, 4, 128), g=f(5, 4), beta=f(5, 4), state=f(6, 4, 64, 128),
                out=f(5, 4, 128), T=5)

    def bad(error, fn=delta.step, **kw):
        for fn, extra in ((delta.step, {"n": None}), (delta.prefill, {"cu": _i32(3)})):
            with pytest.raises(error):
                fn(**{**good, **extra, **kw})
    bad(TypeError, q=f(5, 2, 64))
    bad(TypeError, g=_bf(5, 4))
    bad(TypeError, state=_bf(6, 4, 64, 128))
    bad(ValueError, T=6)
    bad(ValueError, v=_bf(5, 3, 128))
    bad(ValueError, k=_bf(5, 2, 128))
    bad(ValueError, beta=f(5, 8)[:, ::2])
    bad(ValueError, state=f(6, 4, 128, 64))
    bad(ValueError, state=f(6, 4, 128, 64).transpose(2, 3))
    bad(ValueError, out=f(5, 4, 64))
    bad(ValueError, slots=_i32(1))
    bad(RuntimeError)                                            # no GPU tensors
    with pytest.raises(ValueError):
        delta.prefill(**good, cu=_i32(2, 2))
    with pytest.raises(TypeError):
        delta.prefill(**good, cu=torch.zeros(3, dtype=torch.int64))
