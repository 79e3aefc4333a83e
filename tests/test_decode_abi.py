"""Argument checks of the cached-decoding entries: status codes before any device
work (pointers are fake and never dereferenced; no GPU needed)."""
import ctypes

import pytest

import b2q

FAKE = 1 << 20  # aligned, non-null
OK, ARG, UNSUP, ALIGN, WS, TOO = 0, 1, 2, 3, 4, 7


def plan(**kw):
    a = dict(cached=FAKE, new=FAKE, B=4, ps=16, free=FAKE, nf=8, table=FAKE, W=8, ldt=32, mt=64, slots=FAKE, pos=FAKE,
             cu=FAKE, kv=FAKE, counts=FAKE)
    a.update(kw)
    return b2q.lib().b2q_kv_cache_plan(a["cached"], a["new"], a["B"], a["ps"], a["free"], a["nf"], a["table"], a["W"],
                                       a["ldt"], a["mt"], a["slots"], a["pos"], a["cu"], a["kv"], a["counts"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(B=-1), ARG), (dict(nf=-1), ARG), (dict(W=-1), ARG), (dict(mt=-1), ARG), (dict(ldt=28), ARG),
    (dict(cached=None), ARG), (dict(new=None), ARG), (dict(free=None), ARG), (dict(table=None), ARG),
    (dict(slots=None), ARG), (dict(pos=None), ARG), (dict(cu=None), ARG), (dict(kv=None), ARG), (dict(counts=None), ARG),
    (dict(ps=8), UNSUP), (dict(ps=24), UNSUP), (dict(ps=512), UNSUP), (dict(ps=0), UNSUP),
    (dict(B=16385), TOO), (dict(mt=1 << 31), TOO), (dict(nf=1 << 31), TOO), (dict(W=1 << 31, ldt=1 << 40), TOO),
    (dict(slots=FAKE + 8), ALIGN), (dict(pos=FAKE + 4), ALIGN), (dict(cu=FAKE + 2), ALIGN), (dict(ldt=34), ALIGN),
    (dict(table=FAKE + 1), ALIGN),
])
def test_plan_checks(b2q_mod, kw, expect):
    assert plan(**kw) == expect


def rope(**kw):
    a = dict(qkv=FAKE, T=4, Hq=4, Hkv=2, D=64, ld=8 * 64 * 4, norm=0, gq=None, gk=None, eps=1e-6, pos=FAKE, ps_=4, axes=3,
             sec=(16, 8, 8), inv=FAKE, inter=0, ty=1, q=FAKE, ldq=512, kc=FAKE, vc=FAKE, slots=FAKE, np_=4, ps=16)
    a.update(kw)
    sec = (ctypes.c_int32 * 4)(*a["sec"]) if a["sec"] is not None else None
    return b2q.lib().b2q_qkv_rope_cache(a["qkv"], a["T"], a["Hq"], a["Hkv"], a["D"], a["ld"], a["norm"], a["gq"], a["gk"],
                                        a["eps"], a["pos"], a["ps_"], a["axes"], sec, a["inv"], a["inter"], a["ty"],
                                        a["q"], a["ldq"], a["kc"], a["vc"], a["slots"], a["np_"], a["ps"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(T=-1), ARG), (dict(Hq=0, Hkv=0), ARG), (dict(Hkv=-1), ARG), (dict(norm=2), ARG), (dict(inter=3), ARG),
    (dict(norm=1, eps=-1.0), ARG), (dict(norm=1, eps=float("nan")), ARG), (dict(axes=4), ARG), (dict(axes=-1), ARG),
    (dict(sec=None), ARG), (dict(sec=(20, 8, 8)), ARG), (dict(sec=(20, -4, 8)), ARG), (dict(ld=8 * 64 * 4 - 16), ARG),
    (dict(ldq=504), ARG), (dict(ps_=3), ARG), (dict(qkv=None), ARG), (dict(q=None), ARG), (dict(kc=None), ARG),
    (dict(vc=None), ARG), (dict(slots=None), ARG), (dict(pos=None), ARG), (dict(inv=None), ARG),
    (dict(D=32), UNSUP), (dict(D=96), UNSUP), (dict(ty=0), UNSUP), (dict(ps=8), UNSUP), (dict(ps=48), UNSUP),
    (dict(T=1 << 31, ps_=1 << 31), TOO), (dict(Hq=5000, ld=1 << 30, ldq=1 << 30), TOO),
    (dict(qkv=FAKE + 8), ALIGN), (dict(ld=8 * 64 * 4 + 8), ALIGN), (dict(q=FAKE + 4), ALIGN), (dict(ldq=516), ALIGN),
    (dict(kc=FAKE + 2), ALIGN), (dict(norm=1, gq=FAKE + 4), ALIGN), (dict(slots=FAKE + 4), ALIGN),
    (dict(T=0), OK),
])
def test_rope_checks(b2q_mod, kw, expect):
    assert rope(**kw) == expect


def attn(**kw):
    a = dict(ty=1, q=FAKE, ldq=512, cu=FAKE, B=2, T=8, mn=4, k=FAKE, v=FAKE, np_=9, ps=16, table=FAKE, W=8, ldt=32, kv=FAKE,
             mk=128, Hq=4, Hkv=2, D=64, scale=0.125, causal=1, window=0, sinks=0, o=FAKE, ldo=512, ws=FAKE, wsb=1 << 40)
    a.update(kw)
    return b2q.lib().b2q_attention_paged(a["ty"], a["q"], a["ldq"], a["cu"], a["B"], a["T"], a["mn"], a["k"], a["v"], a["np_"],
                                         a["ps"], a["table"], a["W"], a["ldt"], a["kv"], a["mk"], a["Hq"], a["Hkv"], a["D"],
                                         a["scale"], a["causal"], a["window"], a["sinks"], a["o"], a["ldo"], a["ws"],
                                         a["wsb"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(B=-1), ARG), (dict(T=-1), ARG), (dict(mn=-1), ARG), (dict(mk=-1), ARG), (dict(Hq=3), ARG), (dict(Hkv=0), ARG),
    (dict(window=-1), ARG), (dict(sinks=-1), ARG), (dict(causal=2), ARG), (dict(causal=0, window=5), ARG),
    (dict(scale=float("inf")), ARG), (dict(scale=float("nan")), ARG), (dict(np_=-1), ARG), (dict(W=-1), ARG),
    (dict(ldq=508), ARG), (dict(ldo=256), ARG), (dict(ldt=28), ARG), (dict(q=None), ARG), (dict(o=None), ARG),
    (dict(cu=None), ARG), (dict(kv=None), ARG), (dict(table=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG),
    (dict(ty=0), UNSUP), (dict(ty=8), UNSUP), (dict(D=32), UNSUP), (dict(D=256), UNSUP), (dict(ps=8), UNSUP),
    (dict(ps=100), UNSUP), (dict(B=65536), TOO), (dict(T=1 << 31), TOO), (dict(mn=1 << 31), TOO),
    (dict(W=1 << 28, ldt=1 << 40), TOO), (dict(q=FAKE + 8), ALIGN), (dict(ldq=520), ALIGN), (dict(o=FAKE + 2), ALIGN),
    (dict(k=FAKE + 8), ALIGN), (dict(ws=FAKE + 16), ALIGN), (dict(ldt=34), ALIGN),
    (dict(mk=100000, W=8000, ldt=32000, wsb=16), WS), (dict(mk=100000, W=8000, ldt=32000, ws=None), WS),
    (dict(B=0), OK), (dict(T=0), OK), (dict(mn=0), OK),
])
def test_attention_checks(b2q_mod, kw, expect):
    assert attn(**kw) == expect


def test_attention_workspace_size(b2q_mod):
    f = b2q.attention_paged_workspace_bytes
    assert f(2, 2, 1, 100, 8, 2, 128) == 0          # one stretch: nothing to join
    big = f(2, 2, 1, 100000, 8, 2, 128)
    assert big > 0 and big % 256 == 0
    assert f(2, 2, 1, 100000, 8, 2, 128, True, 64, 4) == 0   # the window bounds what a row sees
    assert f(2, 2, 1, 100000, 8, 3, 128) == 0       # invalid sizes
    assert f(-1, 2, 1, 100000, 8, 2, 128) == 0


def test_attention_rows_times_heads_are_bounded(b2q_mod):
    # T * Hq past 2^31: the partial outputs of such a call would not fit the byte counts
    f = b2q.attention_paged_workspace_bytes
    assert f(1, 1 << 26, 1, 1 << 30, 64, 1, 128) == 0
    assert attn(T=1 << 26, mn=1, Hq=64, Hkv=1, ldq=1 << 14, ldo=1 << 14) == TOO


def vec(**kw):
    a = dict(wt=2, w=FAKE, n=64, k=1024, xt=0, x=FAKE, m=4, ldx=4096, bias=None, gate=None, resid=None, ldr=0, y=FAKE,
             ldy=256)
    a.update(kw)
    return b2q.lib().b2q_mul_vec(a["wt"], a["w"], a["n"], a["k"], a["xt"], a["x"], a["m"], a["ldx"], a["bias"], a["gate"],
                                 a["resid"], a["ldr"], a["y"], a["ldy"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(n=-1), ARG), (dict(m=-1), ARG), (dict(k=0), ARG), (dict(k=1000), ARG), (dict(wt=12, k=1056, ldx=8192), ARG),
    (dict(gate=FAKE), ARG), (dict(ldx=4092), ARG), (dict(ldy=252), ARG), (dict(resid=FAKE + 4096, ldr=128), ARG),
    (dict(resid=FAKE, ldr=512), ARG), (dict(w=None), ARG), (dict(x=None), ARG), (dict(y=None), ARG),
    (dict(wt=8), UNSUP), (dict(wt=1), UNSUP), (dict(xt=2), UNSUP), (dict(m=9), TOO), (dict(n=1 << 31, ldy=1 << 34), TOO),
    (dict(w=FAKE + 16), ALIGN), (dict(x=FAKE + 2), ALIGN), (dict(xt=1, x=FAKE + 1), ALIGN), (dict(ldx=4098), ALIGN),
    (dict(y=FAKE + 2), ALIGN), (dict(bias=FAKE + 1), ALIGN), (dict(m=0), OK), (dict(n=0), OK),
])
def test_mul_vec_checks(b2q_mod, kw, expect):
    assert vec(**kw) == expect
