"""CPU: what the C entries of the attention-side layers refuse, before any HIP call, and what they accept as nothing to do."""
import ctypes

import pytest

P = 4096                                   # an aligned address that is never read: every call below returns before a launch
ARG, SHAPE, UNSUPPORTED, WORKSPACE = -1, -2, -4, -5


@pytest.fixture(scope="module")
def L():
    from yolo_amd import _lib
    return _lib.lib()


def linear(L, **kw):
    a = dict(dtype=1, x=P, x_ld=8, w=P, w_ld=8, bias=None, bias_dtype=0, res=None, res_ld=0, out=P, out_ld=16, M=0, N=16, K=8, act=0)
    a.update(kw)
    return L.yolo_linear(*a.values(), None)


def test_linear(L):
    assert linear(L) == 0                                                         # M = 0
    assert linear(L, x=None, out=None) == 0
    for kw, code, text in ((dict(dtype=2), ARG, b"dtype"), (dict(bias_dtype=7), ARG, b"bias dtype"), (dict(act=5), ARG, b"activation"), (dict(act=-1), ARG, b"activation"),
                           (dict(M=-1), ARG, b"size"), (dict(N=0), ARG, b"size"), (dict(K=0), ARG, b"size"), (dict(M=1, x=None), ARG, b"null"),
                           (dict(M=1, w=None), ARG, b"null"), (dict(M=1, out=None), ARG, b"null"), (dict(M=1, x_ld=7), ARG, b"stride"), (dict(M=1, w_ld=7), ARG, b"stride"),
                           (dict(M=1, out_ld=15), ARG, b"stride"), (dict(M=1, res=P, res_ld=15), ARG, b"stride"), (dict(M=1, x=P + 1), ARG, b"aligned"),
                           (dict(M=1, dtype=0, out=P + 2), ARG, b"aligned"), (dict(M=1, bias=P + 2, bias_dtype=0), ARG, b"aligned"),
                           (dict(M=1, K=(1 << 30) + 1, x_ld=1 << 31, w_ld=1 << 31), UNSUPPORTED, b"2^30"),
                           (dict(M=1 << 40, N=1 << 20, out_ld=1 << 20), UNSUPPORTED, b"tiles")):
        assert linear(L, **kw) == code and text in L.yolo_last_error(), (kw, L.yolo_last_error())


def strides(*v):
    return (ctypes.c_int64 * 3)(*v)


def qk(L, **kw):
    a = dict(dtype=1, B=0, D=64, q=P, qs=strides(64, 64, 64), Lq=1, Hq=1, qw=None, qp=P, qo=P, k=None, ks=None, Lk=0, Hk=0, kw=None, kp=None, ko=None, wd=0,
             f=P, R=64, axes=1, p64=0, qb=0, kb=0, il=0, eps=1e-6)
    a.update(kw)
    return L.yolo_qk_norm_rope(*a.values(), None)


def test_qk_norm_rope(L):
    assert qk(L) == 0 and qk(L, B=2, Lq=0, q=None) == 0
    kk = dict(k=P, ks=strides(64, 64, 64), Lk=3, Hk=1, kp=P, ko=P)
    for kw, code, text in ((dict(dtype=3), ARG, b"dtype"), (dict(wd=2), ARG, b"weight dtype"), (dict(B=-1), ARG, b"size"), (dict(Hq=0), ARG, b"size"),
                           (dict(k=P, Hk=0), ARG, b"size"), (dict(D=257), UNSUPPORTED, b"head size"), (dict(D=0), UNSUPPORTED, b"head size"),
                           (dict(eps=0.0), ARG, b"eps"), (dict(eps=float("nan")), ARG, b"eps"), (dict(R=63), ARG, b"rotary"), (dict(R=66), ARG, b"rotary"), (dict(R=0), ARG, b"rotary"),
                           (dict(axes=3), ARG, b"axes"), (dict(R=62, axes=2), ARG, b"axes"), (dict(B=1, q=None), ARG, b"null"), (dict(B=1, qo=None), ARG, b"null"),
                           (dict(B=1, qs=None), ARG, b"null"), (dict(B=1, qp=None), ARG, b"positions"), (dict(kk, B=1, Lq=0, kp=None), ARG, b"positions"),
                           (dict(kk, B=1, Lq=0, ko=None), ARG, b"null"), (dict(B=1, q=P + 1), ARG, b"aligned"), (dict(B=1 << 16, Lq=1 << 15), UNSUPPORTED, b"2^31")):
        assert qk(L, **kw) == code and text in L.yolo_last_error(), (kw, L.yolo_last_error())


def attention(L, **kw):
    s = strides(64, 64, 64)
    a = dict(dtype=1, q=P, qs=s, k=P, ks=s, v=P, vs=s, lens=None, mask=None, B=0, Lq=1, Lk=1, Hq=4, Hk=2, D=64, scale=0.125, out=P, ws=None, wsn=0)
    a.update(kw)
    return L.yolo_cross_attention(*a.values(), None)


def test_cross_attention(L):
    assert attention(L) == 0 and attention(L, B=3, Lq=0, q=None, out=None) == 0
    for kw, code, text in ((dict(dtype=2), ARG, b"dtype"), (dict(B=-1), ARG, b"size"), (dict(Lk=-1), ARG, b"size"), (dict(Hk=0), ARG, b"size"), (dict(Hq=0), ARG, b"size"),
                           (dict(Hq=5), SHAPE, b"share"), (dict(D=0), UNSUPPORTED, b"head size"), (dict(D=257), UNSUPPORTED, b"head size"), (dict(B=1, q=None), ARG, b"null"),
                           (dict(B=1, k=None), ARG, b"null"), (dict(B=1, v=None), ARG, b"null"), (dict(B=1, out=None), ARG, b"null"), (dict(B=1, vs=None), ARG, b"null"),
                           (dict(B=1, q=P + 1), ARG, b"aligned"), (dict(B=1, lens=P + 2), ARG, b"aligned"), (dict(B=1 << 16, Lq=1 << 15), UNSUPPORTED, b"2^31")):
        assert attention(L, **kw) == code and text in L.yolo_last_error(), (kw, L.yolo_last_error())
    for bad in (dict(B=-1), dict(Hq=5), dict(D=300)):
        a = dict(dtype=1, B=1, Lq=1, Lk=100, Hq=4, Hk=2, D=64)
        a.update(bad)
        assert L.yolo_cross_attention_workspace_bytes(*a.values()) == 0


def test_launches_past_the_runtime_limit_are_refused(L):
    """The runtime counts the threads of a launch in 32 bits: sizes that need more are the documented refusal, not a failed launch."""
    for kw in (dict(M=1 << 30, N=1, out_ld=1), dict(M=1 << 30, N=256, out_ld=256), dict(M=1 << 30, N=256, out_ld=256, dtype=0),
               dict(M=1 << 30, N=256, out_ld=256, x_ld=9), dict(M=1 << 30, N=33, out_ld=33, x_ld=1 << 22)):
        assert linear(L, **kw) == UNSUPPORTED and b"tiles" in L.yolo_last_error(), (kw, L.yolo_last_error())
    wide = dict(qs=strides(1 << 20, 256, 8), D=8, R=8)
    for kw in (dict(wide, B=1 << 12, Lq=1 << 12, Hq=32), dict(B=1 << 12, Lq=1 << 12, Hq=64, D=256, R=256), dict(wide, B=1 << 12, Lq=1 << 12, Hq=32, D=4, R=4, dtype=0)):
        assert qk(L, **kw) == UNSUPPORTED and b"workgroups" in L.yolo_last_error(), (kw, L.yolo_last_error())
    for kw in (dict(B=1 << 10, Lq=1 << 13, Hq=8, Hk=8, Lk=0), dict(B=1 << 10, Lq=1 << 13, Hq=8, Hk=8, D=7), dict(B=1 << 26, Hq=1, Hk=1),
               dict(B=1 << 24, Hq=1, Hk=1, D=128), dict(B=1 << 24, Hq=1, Hk=1, D=256), dict(B=1 << 24, Hq=8, Hk=8, dtype=0), dict(B=1 << 23, Hq=1, Hk=1, D=256)):
        assert attention(L, **kw) == UNSUPPORTED and b"workgroups" in L.yolo_last_error(), (kw, L.yolo_last_error())


def test_no_row_kernel_that_no_call_reaches(L):
    """A row of at most 256 elements is 32 pairs of 16-byte pieces in float32 and 16 in bfloat16: the library has no bfloat16 kernel of 32 lanes."""
    from yolo_amd import _lib
    with open(_lib.LIB_PATH, "rb") as f:
        built = f.read()
    assert b"qk_norm_rope_kernelILb0ELi32E" in built and b"qk_norm_rope_kernelILb1ELi16E" in built
    assert b"qk_norm_rope_kernelILb1ELi32E" not in built


def test_objects_depend_on_the_makefile():
    """A changed flag (such as the one against packed float32 arithmetic) compiles every source again."""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "yolo_amd", "csrc")
    plan = subprocess.run(["make", "-n", "-W", "Makefile"], cwd=csrc, check=True, capture_output=True, text=True).stdout
    for f in sorted(os.listdir(csrc)):
        if f.endswith(".hip"):
            assert "-c " + f in plan, f
