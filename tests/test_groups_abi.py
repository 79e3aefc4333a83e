"""Argument checks of the entries for rows that go by group and for drafted tokens: status codes before any device
work (pointers are fake and never dereferenced; no GPU needed)."""
import pytest

import b2q

FAKE = 1 << 20  # aligned, non-null
OK, ARG, UNSUP, ALIGN, WS, TOO = 0, 1, 2, 3, 4, 7
BIG = 1 << 40


def route(**kw):
    a = dict(ty=0, x=FAKE, T=4, E=8, ld=32, bias=FAKE, top=2, sc=0, rn=1, scale=1.0, ids=FAKE, w=FAKE, order=FAKE, off=FAKE,
             ws=FAKE, wsb=BIG)
    a.update(kw)
    return b2q.lib().b2q_moe_route(a["ty"], a["x"], a["T"], a["E"], a["ld"], a["bias"], a["top"], a["sc"], a["rn"], a["scale"],
                                   a["ids"], a["w"], a["order"], a["off"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(T=-1), ARG), (dict(E=0), ARG), (dict(top=0), ARG), (dict(top=9), ARG), (dict(ld=28), ARG), (dict(sc=2), ARG),
    (dict(sc=-1), ARG), (dict(rn=2), ARG), (dict(scale=float("inf")), ARG), (dict(scale=float("nan")), ARG),
    (dict(x=None), ARG), (dict(ids=None), ARG), (dict(w=None), ARG), (dict(order=None), ARG), (dict(off=None), ARG),
    (dict(ty=8), UNSUP), (dict(ty=2), UNSUP), (dict(E=1025, ld=5000), TOO), (dict(E=64, ld=256, top=33), TOO),
    (dict(T=1 << 30), TOO), (dict(x=FAKE + 2), ALIGN), (dict(ty=1, x=FAKE + 1), ALIGN), (dict(ld=34), ALIGN),
    (dict(bias=FAKE + 2), ALIGN), (dict(ids=FAKE + 1), ALIGN), (dict(w=FAKE + 3), ALIGN), (dict(order=FAKE + 2), ALIGN),
    (dict(off=FAKE + 2), ALIGN), (dict(ws=FAKE + 2), ALIGN), (dict(T=5000, ws=None), WS), (dict(T=5000, wsb=8), WS),
])
def test_route_checks(b2q_mod, kw, expect):
    assert route(**kw) == expect


def rows(**kw):
    a = dict(ids=FAKE, S=9, G=4, order=FAKE, off=FAKE, ws=FAKE, wsb=BIG)
    a.update(kw)
    return b2q.lib().b2q_group_rows(a["ids"], a["S"], a["G"], a["order"], a["off"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(S=-1), ARG), (dict(G=0), ARG), (dict(ids=None), ARG), (dict(order=None), ARG), (dict(off=None), ARG),
    (dict(G=1025), TOO), (dict(S=(1 << 30) + 1), TOO), (dict(ids=FAKE + 2), ALIGN), (dict(order=FAKE + 1), ALIGN),
    (dict(off=FAKE + 2), ALIGN), (dict(S=100000, ws=None), WS), (dict(S=100000, wsb=100), WS),
])
def test_group_rows_checks(b2q_mod, kw, expect):
    assert rows(**kw) == expect


def mmid(**kw):
    a = dict(wt=1, w=FAKE, E=4, n=16, k=64, ldw=128, lde=2048, x=FAKE, xr=10, ldx=128, order=FAKE, off=FAKE, S=20, pr=2,
             bias=FAKE, glu=0, yt=1, y=FAKE, ldy=32)
    a.update(kw)
    return b2q.lib().b2q_mul_mat_id(a["wt"], a["w"], a["E"], a["n"], a["k"], a["ldw"], a["lde"], a["x"], a["xr"], a["ldx"],
                                    a["order"], a["off"], a["S"], a["pr"], a["bias"], a["glu"], a["yt"], a["y"], a["ldy"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(E=0), ARG), (dict(n=-1), ARG), (dict(k=0), ARG), (dict(k=60), ARG), (dict(wt=2, k=48, ldx=128), ARG), (dict(xr=-1), ARG),
    (dict(S=-1), ARG), (dict(pr=0), ARG), (dict(glu=2), ARG), (dict(xr=9), ARG), (dict(ldw=112), ARG), (dict(lde=-16), ARG), (dict(lde=0), ARG),
    (dict(ldx=112), ARG), (dict(ldy=30), ARG), (dict(w=None), ARG), (dict(x=None), ARG), (dict(order=None), ARG),
    (dict(off=None), ARG), (dict(y=None), ARG), (dict(wt=8), UNSUP), (dict(wt=12), UNSUP), (dict(wt=0), UNSUP),
    (dict(yt=30), UNSUP), (dict(wt=30, yt=1), UNSUP), (dict(wt=2, yt=30), UNSUP), (dict(E=1025), TOO),
    (dict(n=1 << 30, ldy=1 << 31), TOO), (dict(n=1 << 22, E=1024, ldy=1 << 23), TOO), (dict(k=1 << 29, ldw=1 << 30, ldx=1 << 30), TOO),
    (dict(S=(1 << 30) + 1, xr=1 << 30), TOO), (dict(w=FAKE + 8), ALIGN), (dict(wt=2, w=FAKE + 16), ALIGN), (dict(ldw=136), ALIGN),
    (dict(lde=2056), ALIGN), (dict(x=FAKE + 8), ALIGN), (dict(ldx=136), ALIGN), (dict(order=FAKE + 2), ALIGN),
    (dict(off=FAKE + 1), ALIGN), (dict(bias=FAKE + 2), ALIGN), (dict(y=FAKE + 1), ALIGN), (dict(ldy=33), ALIGN),
    (dict(S=0), OK), (dict(n=0), OK), (dict(S=0, xr=0), OK),
])
def test_mul_mat_id_checks(b2q_mod, kw, expect):
    assert mmid(**kw) == expect


def join(**kw):
    a = dict(yt=1, y=FAKE, ldy=32, w=FAKE, ids=FAKE, T=4, top=2, n=16, ot=0, r=FAKE, ldr=64, o=FAKE * 2, ldo=64)
    a.update(kw)
    return b2q.lib().b2q_moe_combine(a["yt"], a["y"], a["ldy"], a["w"], a["ids"], a["T"], a["top"], a["n"], a["ot"], a["r"], a["ldr"],
                                     a["o"], a["ldo"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(T=-1), ARG), (dict(top=0), ARG), (dict(n=-1), ARG), (dict(y=None), ARG), (dict(w=None), ARG), (dict(o=None), ARG),
    (dict(ldy=30), ARG), (dict(ldo=60), ARG), (dict(ldr=60), ARG), (dict(r=FAKE * 2, ldr=128), ARG), (dict(yt=8), UNSUP),
    (dict(ot=2), UNSUP), (dict(n=(1 << 21) + 1, ldy=1 << 23, ldo=1 << 24, ldr=1 << 24), TOO), (dict(T=1 << 30), TOO),
    (dict(y=FAKE + 1), ALIGN), (dict(ldy=33), ALIGN), (dict(w=FAKE + 2), ALIGN), (dict(ids=FAKE + 2), ALIGN), (dict(o=FAKE + 2), ALIGN),
    (dict(ldo=66), ALIGN), (dict(r=FAKE + 2), ALIGN), (dict(ldr=66), ALIGN), (dict(T=0), OK), (dict(n=0), OK),
])
def test_combine_checks(b2q_mod, kw, expect):
    assert join(**kw) == expect


def lora(**kw):
    a = dict(xt=1, x=FAKE, T=8, k=64, ldx=128, a=FAKE, b=FAKE, G=3, r=16, n=32, sc=FAKE, order=FAKE, off=FAKE, yt=0, res=FAKE, ldr=128,
             y=FAKE, ldy=128, ws=FAKE, wsb=BIG)
    a.update(kw)
    return b2q.lib().b2q_lora_add(a["xt"], a["x"], a["T"], a["k"], a["ldx"], a["a"], a["b"], a["G"], a["r"], a["n"], a["sc"],
                                  a["order"], a["off"], a["yt"], a["res"], a["ldr"], a["y"], a["ldy"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(T=-1), ARG), (dict(k=0), ARG), (dict(k=60), ARG), (dict(G=0), ARG), (dict(r=0), ARG), (dict(r=12), ARG), (dict(n=-1), ARG),
    (dict(ldx=112), ARG), (dict(ldr=124), ARG), (dict(ldy=124), ARG), (dict(ldy=256), ARG), (dict(x=None), ARG), (dict(a=None), ARG),
    (dict(b=None), ARG), (dict(order=None), ARG), (dict(off=None), ARG), (dict(res=None), ARG), (dict(y=None), ARG),
    (dict(xt=0), UNSUP), (dict(yt=30), UNSUP), (dict(xt=30, yt=1), UNSUP), (dict(r=136), TOO), (dict(G=1025), TOO),
    (dict(T=(1 << 30) + 1), TOO), (dict(n=1 << 31, ldr=1 << 33, ldy=1 << 33), TOO), (dict(x=FAKE + 8), ALIGN), (dict(ldx=136), ALIGN),
    (dict(a=FAKE + 8), ALIGN), (dict(b=FAKE + 8), ALIGN), (dict(sc=FAKE + 2), ALIGN), (dict(order=FAKE + 2), ALIGN),
    (dict(off=FAKE + 2), ALIGN), (dict(res=FAKE + 2), ALIGN), (dict(ldr=130, y=2 * FAKE), ALIGN), (dict(y=FAKE + 2), ALIGN),
    (dict(ws=FAKE + 16), ALIGN), (dict(T=5000, ws=None), WS), (dict(T=5000, wsb=100), WS), (dict(T=0), OK), (dict(n=0), OK),
])
def test_lora_checks(b2q_mod, kw, expect):
    assert lora(**kw) == expect


@pytest.mark.parametrize("call", [
    lambda: mmid(),                                                       # x itself
    lambda: mmid(y=FAKE - 32 * 19),                                       # its last row on x's first
    lambda: mmid(y=FAKE + 128 * 9 + 126),                                 # its first row on x's last value
    lambda: mmid(y=FAKE + 100, ldy=128),                                  # columns of one table that share some
    lambda: join(o=FAKE + 32, ldo=64),
    lambda: join(o=FAKE, ldo=64),
    lambda: join(r=2 * FAKE + 64),                                        # a row further
    lambda: join(r=2 * FAKE + 32, ldr=96, ldo=96),
    lambda: lora(xt=1, yt=1, ldy=64, ldr=64),                             # x is y
    lambda: lora(y=2 * FAKE, res=2 * FAKE + 128),
    lambda: lora(y=2 * FAKE, res=2 * FAKE - 64, ldy=160, ldr=160),
])
def test_results_on_operands_are_refused(b2q_mod, call):
    assert call() == ARG


def verify(**kw):
    a = dict(ty=0, t=FAKE, ldt=400, g=FAKE, ldg=400, d=FAKE, cu=FAKE, B=3, D=6, V=100, u=FAKE, v=FAKE, acc=FAKE, tok=FAKE)
    a.update(kw)
    return b2q.lib().b2q_draft_verify(a["ty"], a["t"], a["ldt"], a["g"], a["ldg"], a["d"], a["cu"], a["B"], a["D"], a["V"], a["u"],
                                      a["v"], a["acc"], a["tok"], None)


@pytest.mark.parametrize("kw,expect", [
    (dict(B=-1), ARG), (dict(D=-1), ARG), (dict(V=0), ARG), (dict(t=None), ARG), (dict(d=None), ARG), (dict(cu=None), ARG),
    (dict(u=None), ARG), (dict(v=None), ARG), (dict(acc=None), ARG), (dict(tok=None), ARG), (dict(ldt=396), ARG), (dict(ldg=396), ARG),
    (dict(ty=12), UNSUP), (dict(B=(1 << 20) + 1), TOO), (dict(D=(1 << 30) + 1), TOO), (dict(V=(1 << 28) + 1, ldt=1 << 31, ldg=1 << 31), TOO),
    (dict(t=FAKE + 2), ALIGN), (dict(ldt=402), ALIGN), (dict(g=FAKE + 2), ALIGN), (dict(ldg=402), ALIGN), (dict(d=FAKE + 2), ALIGN),
    (dict(cu=FAKE + 2), ALIGN), (dict(u=FAKE + 2), ALIGN), (dict(v=FAKE + 1), ALIGN), (dict(acc=FAKE + 2), ALIGN),
    (dict(tok=FAKE + 2), ALIGN), (dict(B=0), OK),
])
def test_verify_checks(b2q_mod, kw, expect):
    assert verify(**kw) == expect


def test_workspace_sizes(b2q_mod):
    L = b2q.lib()
    assert L.b2q_moe_route_workspace_bytes(10, 64, 4) == 0            # one launch, nothing to keep
    assert L.b2q_moe_route_workspace_bytes(10000, 64, 4) % (65 * 4) == 0 < L.b2q_moe_route_workspace_bytes(10000, 64, 4)
    assert L.b2q_moe_route_workspace_bytes(10000, 64, 65) == 0        # invalid sizes
    assert L.b2q_group_rows_workspace_bytes(100, 64) == 0 < L.b2q_group_rows_workspace_bytes(100000, 64)
    assert L.b2q_group_rows_workspace_bytes(100000, 0) == 0
    assert L.b2q_lora_add_workspace_bytes(8, 64, 8, 16) == 0 < L.b2q_lora_add_workspace_bytes(5000, 64, 8, 16)
    assert L.b2q_lora_add_workspace_bytes(5000, 64, 8, 12) == 0
