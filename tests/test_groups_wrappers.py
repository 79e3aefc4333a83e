"""What the Python wrappers of the calls for rows that go by group and for drafted tokens refuse before anything reaches
the library, and what they pass on.  The library is a stand-in that records the calls; no GPU needed."""
import types

import pytest
import torch

import b2q

F32, F16, BF16, I32, I64 = torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int64


@pytest.fixture
def lib_calls(monkeypatch):
    calls = []
    fake = lambda name: lambda *a: (calls.append((name, a)), 0)[1]  # noqa: E731
    names = ("b2q_moe_route", "b2q_group_rows", "b2q_mul_mat_id", "b2q_moe_combine", "b2q_lora_add", "b2q_draft_verify")
    monkeypatch.setattr(b2q, "_lib", types.SimpleNamespace(**{n: fake(n) for n in names}))
    monkeypatch.setattr(b2q, "_raw_stream", lambda *a: 0)
    for n in ("_route_ws_bytes", "_group_ws_bytes", "_lora_ws_bytes"):
        monkeypatch.setattr(b2q, n, lambda *a: 0)
    monkeypatch.setattr(b2q, "_packed4_bytes", lambda wtype, n, k: n * k * 9 // 16)
    return calls


def z(*shape, dt=F32):
    return torch.zeros(*shape, dtype=dt)


def route(T=5, E=8, **kw):
    a = dict(logits=z(T, E), top=2)
    a.update(kw)
    return b2q.moe_route(**a)


def mmid(E=4, n=16, k=64, rows=6, per_row=2, glu=False, **kw):
    a = dict(wtype=b2q.TYPE_F16, w=z(E, 2 * n if glu else n, k, dt=F16), n=n, k=k, x=z(rows, k, dt=F16),
             order=z(rows * per_row, dt=I32), offsets=z(E + 1, dt=I32), per_row=per_row, glu=glu)
    a.update(kw)
    return b2q.mul_mat_id(**a)


def join(T=4, top=2, n=16, **kw):
    a = dict(y=z(T * top, n, dt=F16), weights=z(T, top), ids=z(T, top, dt=I32))
    a.update(kw)
    return b2q.moe_combine(**a)


def lora(T=6, G=3, r=16, k=64, n=32, **kw):
    a = dict(resid=z(T, n), x=z(T, k, dt=F16), a=z(G, r, k, dt=F16), b=z(G, n, r, dt=F16), scales=z(G), order=z(T, dt=I32),
             offsets=z(G + 1, dt=I32))
    a.update(kw)
    return b2q.lora_add(**a)


def verify(B=3, D=5, V=20, **kw):
    a = dict(target=z(D + B, V), draft_probs=z(D, V), drafts=z(D, dt=I32), cu_drafts=z(B + 1, dt=I32), u=z(D), v=z(B))
    a.update(kw)
    return b2q.draft_verify(**a)


def refused(lib_calls, call, **kw):
    with pytest.raises((AssertionError, KeyError)):
        call(**kw)
    assert not lib_calls


@pytest.mark.parametrize("call,name", [(route, "b2q_moe_route"), (mmid, "b2q_mul_mat_id"), (join, "b2q_moe_combine"),
                                       (lora, "b2q_lora_add"), (verify, "b2q_draft_verify")])
def test_plain_calls_are_taken(lib_calls, call, name):
    call()
    assert [c[0] for c in lib_calls] == [name]


@pytest.mark.parametrize("kw", [
    dict(logits=z(5, 8, dt=I32)), dict(logits=z(8, 5).t()), dict(logits=z(8).expand(5, 8)), dict(top=0), dict(top=9),
    dict(bias=z(7)), dict(bias=z(8, dt=F16)), dict(bias=z(16)[::2]), dict(scoring="relu"),
])
def test_route_refuses(lib_calls, kw):
    refused(lib_calls, route, **kw)


@pytest.mark.parametrize("ids", [z(6, dt=I64), z(6), z(12, dt=I32)[::2]])
def test_group_rows_refuses(lib_calls, ids):
    refused(lib_calls, lambda: b2q.group_rows(ids, 3))


@pytest.mark.parametrize("kw", [
    dict(x=z(6, 32, dt=F16)), dict(x=z(6, 64, dt=BF16)), dict(x=z(6, 64)), dict(x=z(64, 6, dt=F16).t()),
    dict(x=z(64, dt=F16).expand(6, 64)), dict(w=z(4, 16, 32, dt=F16)), dict(w=z(4, 32, 64, dt=F16)), dict(w=z(4, 16, 64)),
    dict(w=z(3, 16, 64, dt=F16)), dict(w=z(16, 64, dt=F16).expand(4, 16, 64)), dict(w=z(4, 64, 16, dt=F16).transpose(1, 2)), dict(order=z(12, dt=I64)),
    dict(order=z(24, dt=I32)[::2]), dict(offsets=z(5, dt=I64)), dict(bias=z(63)), dict(bias=z(64, dt=F16)),
    dict(out=z(12, 8, dt=F16)), dict(out=z(11, 16, dt=F16)), dict(out=z(16, 12, dt=F16).t()), dict(out=z(12, 16), out_dtype=F16),
    dict(out=z(16, dt=F16).expand(12, 16)), dict(out_dtype=I32), dict(wtype=b2q.TYPE_BF16), dict(glu=True, w=z(4, 16, 64, dt=F16)),
    dict(wtype=b2q.TYPE_Q4_0, w=z(100, dt=torch.uint8)),
    dict(wtype=b2q.TYPE_Q4_0, w=z(4 * 16 * 64, dt=torch.uint8), x=z(6, 64, dt=BF16)),
])
def test_mul_mat_id_refuses(lib_calls, kw):
    refused(lib_calls, mmid, **kw)


def test_mul_mat_id_passes_strides(lib_calls):
    w = z(4, 20, 80, dt=F16)[:, :16, :64]
    x = z(6, 72, dt=F16)[:, :64]
    mmid(w=w, x=x, out=z(12, 24, dt=F16)[:, :16])
    a = lib_calls[0][1]
    assert a[5:7] == (160, 3200) and a[8:10] == (6, 144) and a[18] == 48


@pytest.mark.parametrize("kw", [
    dict(y=z(7, 16, dt=F16)), dict(y=z(8, 16, dt=I32)), dict(y=z(16, 8, dt=F16).t()), dict(weights=z(4, 2, dt=F16)),
    dict(weights=z(2, 4).t()), dict(ids=z(4, 3, dt=I32)), dict(ids=z(4, 2, dt=I64)), dict(resid=z(4, 15)), dict(resid=z(3, 16)),
    dict(resid=z(4, 16), out_dtype=F16), dict(out=z(4, 15, dt=F16)), dict(out=z(16, 4).t()),
    dict(resid=z(4, 16, dt=F16), out=z(4, 16)), dict(y=z(16, dt=F16).expand(8, 16)), dict(out=z(16).expand(4, 16)),
    dict(resid=z(16).expand(4, 16)), dict(resid=z(16).expand(4, 16), out=z(4, 16)),
])
def test_combine_refuses(lib_calls, kw):
    refused(lib_calls, join, **kw)


@pytest.mark.parametrize("kw", [
    dict(x=z(6, 64)), dict(x=z(6, 56, dt=F16)), dict(x=z(64, dt=F16).expand(6, 64)), dict(x=z(64, 6, dt=F16).t()),
    dict(a=z(3, 16, 64, dt=BF16)), dict(a=z(3, 64, 16, dt=F16).transpose(1, 2)), dict(b=z(3, 31, 16, dt=F16)), dict(b=z(2, 32, 16, dt=F16)),
    dict(b=z(3, 32, 8, dt=F16)), dict(scales=z(2)), dict(scales=z(3, dt=F16)), dict(order=z(5, dt=I32)), dict(order=z(6, dt=I64)),
    dict(offsets=z(3, dt=I32)), dict(resid=z(5, 32)), dict(resid=z(6, 32, dt=I32)), dict(resid=z(32, 6).t()),
    dict(resid=z(32).expand(6, 32)), dict(out=z(6, 32, dt=F16)), dict(out=z(6, 31)), dict(out=z(5, 32)), dict(out=z(32).expand(6, 32)),
])
def test_lora_refuses(lib_calls, kw):
    refused(lib_calls, lora, **kw)


@pytest.mark.parametrize("kw", [
    dict(target=z(7, 20)), dict(target=z(20, 8).t()), dict(target=z(8, 20, dt=I32)), dict(target=z(20).expand(8, 20)),
    dict(draft_probs=z(5, 19)), dict(draft_probs=z(4, 20)), dict(draft_probs=z(5, 20, dt=F16)), dict(draft_probs=z(20).expand(5, 20)),
    dict(draft_probs=z(20, 5).t()), dict(drafts=z(5, dt=I64)), dict(drafts=z(10, dt=I32)[::2]), dict(cu_drafts=z(4, dt=I64)),
    dict(u=z(4)), dict(u=z(5, dt=F16)), dict(v=z(4)), dict(v=z(3, dt=torch.float64)),
])
def test_verify_refuses(lib_calls, kw):
    refused(lib_calls, verify, **kw)


def test_operands_on_the_host_are_refused(monkeypatch):
    """Without the stand-in for the stream: tensors of the host never reach the library."""
    monkeypatch.setattr(b2q, "_lib", types.SimpleNamespace())
    for n in ("_route_ws_bytes", "_group_ws_bytes", "_lora_ws_bytes"):
        monkeypatch.setattr(b2q, n, lambda *a: 0)
    for call in (route, mmid, join, lora, verify, lambda: b2q.group_rows(z(3, dt=I32), 2)):
        with pytest.raises((AssertionError, AttributeError)):
            call()
