"""What the Python wrappers of the cached-decoding calls refuse before anything reaches the library: operands whose
size, type or strides are not those that the kernels would read and write.  The library is a stand-in that records the
calls; no GPU needed."""
import types

import pytest
import torch

import b2q

F32, F16, BF16, I32, I64 = torch.float32, torch.float16, torch.bfloat16, torch.int32, torch.int64


@pytest.fixture
def lib_calls(monkeypatch):
    calls = []
    fake = lambda name: lambda *a: (calls.append((name, a)), 0)[1]  # noqa: E731
    names = ("b2q_kv_cache_plan", "b2q_qkv_rope_cache", "b2q_attention_paged", "b2q_mul_vec")
    monkeypatch.setattr(b2q, "_lib", types.SimpleNamespace(**{n: fake(n) for n in names}))
    monkeypatch.setattr(b2q, "_raw_stream", lambda *a: 0)
    monkeypatch.setattr(b2q, "_paged_ws_bytes", lambda *a: 0)
    return calls


def plan(B=3, W=8, T=40, **kw):
    a = dict(cached=torch.zeros(B, dtype=I32), new=torch.zeros(B, dtype=I32), page_size=16,
             free_pages=torch.zeros(9, dtype=I32), block_table=torch.zeros(B, W, dtype=I32), max_tokens=T)
    a.update(kw)
    return b2q.kv_cache_plan(**a)


def rope(T=4, Hq=4, Hkv=2, D=64, **kw):
    a = dict(qkv=torch.zeros(T, (Hq + 2 * Hkv) * D), Hq=Hq, Hkv=Hkv, D=D, positions=torch.zeros(2, T, dtype=I32),
             sections=(8, 8), inv_freq=torch.zeros(16), slots=torch.zeros(T, dtype=I64),
             k_cache=torch.zeros(5, Hkv, 16, D, dtype=F16), v_cache=torch.zeros(5, Hkv, 16, D, dtype=F16))
    a.update(kw)
    return b2q.qkv_rope_cache(**a)


def attention(T=6, B=3, W=8, Hq=4, Hkv=2, D=64, **kw):
    a = dict(q=torch.zeros(T, Hq * D, dtype=F16), k_cache=torch.zeros(5, Hkv, 16, D, dtype=F16),
             v_cache=torch.zeros(5, Hkv, 16, D, dtype=F16), block_table=torch.zeros(B, W, dtype=I32),
             kv_len=torch.zeros(B, dtype=I32), cu_new=torch.zeros(B + 1, dtype=I32), max_new=2, max_kv=128, Hq=Hq)
    a.update(kw)
    return b2q.attention_paged(**a)


def accepted(lib_calls, name, call, **kw):
    call(**kw)
    assert len(lib_calls) == 1 and lib_calls[0][0] == name
    return lib_calls[0][1]


def refused(lib_calls, call, **kw):
    with pytest.raises(AssertionError):
        call(**kw)
    assert not lib_calls


# ------------------------------------------------------------------------------------------------- block tables
def table(kind, B=3, W=8):
    if kind == "expanded":          # one row for all requests: rows 0 bytes apart
        return torch.zeros(W, dtype=I32).expand(B, W)
    if kind == "overlapping":       # rows that begin inside one another
        return torch.zeros(B * W, dtype=I32).as_strided((B, W), (W - 3, 1))
    if kind == "columns":
        return torch.zeros(W, B, dtype=I32).t()
    if kind == "wide":
        return torch.zeros(B, W + 5, dtype=I32)[:, 2:2 + W]
    return torch.zeros(B, W, dtype=I32)


@pytest.mark.parametrize("kind", ["expanded", "overlapping", "columns"])
@pytest.mark.parametrize("call", [plan, attention])
def test_tables_whose_rows_overlap_are_refused(lib_calls, call, kind):
    refused(lib_calls, call, block_table=table(kind))


@pytest.mark.parametrize("kind,stride", [("plain", 32), ("wide", 52)])
def test_tables_that_are_taken(lib_calls, kind, stride):
    assert accepted(lib_calls, "b2q_kv_cache_plan", plan, block_table=table(kind))[8] == stride
    lib_calls.clear()
    assert accepted(lib_calls, "b2q_attention_paged", attention, block_table=table(kind))[13] == stride


def test_a_table_of_one_request_may_have_any_stride(lib_calls):
    t = torch.zeros(8, dtype=I32).expand(1, 8)
    assert accepted(lib_calls, "b2q_kv_cache_plan", plan, B=1, block_table=t)[8] >= 32
    lib_calls.clear()
    assert accepted(lib_calls, "b2q_attention_paged", attention, B=1, block_table=t)[13] >= 32


# ------------------------------------------------------------------------------------------- operands of the rope call
D_, HQ, HKV = 64, 4, 2


@pytest.mark.parametrize("kw", [
    dict(gamma_q=torch.ones(D_)), dict(gamma_k=torch.ones(D_)),                          # one head's gamma for all
    dict(gamma_q=torch.ones(HQ * D_ + 1)), dict(gamma_k=torch.ones(HKV * D_).half()), dict(gamma_q=torch.ones(HQ * D_, dtype=BF16)),
    dict(gamma_q=torch.ones(HQ * D_, 2)[:, 0]), dict(gamma_k=torch.ones(D_).expand(HKV, D_)),
    dict(out=torch.zeros(3, HQ * D_, dtype=F16)), dict(out=torch.zeros(4, HQ * D_ - 8, dtype=F16)),
    dict(out=torch.zeros(HQ * D_, 4, dtype=F16).t()), dict(out=torch.zeros(4, HQ * D_)),
])
def test_rope_operands_that_do_not_fit_are_refused(lib_calls, kw):
    refused(lib_calls, rope, norm=True, **kw)


def test_rope_operands_that_fit(lib_calls):
    kw = dict(gamma_q=torch.ones(HQ, D_), gamma_k=torch.ones(HKV * D_), out=torch.zeros(4, HQ * D_ + 8, dtype=F16)[:, :HQ * D_])
    args = accepted(lib_calls, "b2q_qkv_rope_cache", rope, norm=True, **kw)
    assert args[7] == kw["gamma_q"].data_ptr() and args[8] == kw["gamma_k"].data_ptr() and args[18] == 2 * (HQ * D_ + 8)
    lib_calls.clear()
    accepted(lib_calls, "b2q_qkv_rope_cache", rope, norm=False, gamma_q=torch.ones(3))  # not read without the norm
    lib_calls.clear()
    accepted(lib_calls, "b2q_qkv_rope_cache", rope, T=1, out=torch.zeros(1, HQ * D_, dtype=F16))


# ---------------------------------------------------------------------------------------------- operands of mul_vec
def vec(m=3, n=40, k=512, wtype=b2q.TYPE_Q4_0, packed=None, x=None, **kw):
    size = b2q.lib_packed_bytes(wtype, n, k)
    packed = torch.zeros(size, dtype=torch.uint8) if packed is None else packed(size)
    return b2q.mul_vec(wtype, packed, n, k, torch.zeros(m, k) if x is None else x, **kw)


@pytest.fixture
def packed_sizes(monkeypatch):
    """Sizes of the packed layouts as the library gives them (on the stand-in they are what a test says)."""
    sizes = lambda wtype, n, k: n * k // 2 + n * k // 32 * 2 + (256 if wtype == b2q.TYPE_Q4_0 else 0)  # noqa: E731
    monkeypatch.setattr(b2q, "_packed4_bytes", sizes, raising=False)
    monkeypatch.setattr(b2q, "lib_packed_bytes", sizes, raising=False)


@pytest.mark.parametrize("wtype", [b2q.TYPE_Q4_0, b2q.TYPE_Q4_K])
@pytest.mark.parametrize("kw", [
    dict(bias=torch.zeros(39)), dict(bias=torch.zeros(40, dtype=F16)), dict(bias=torch.zeros(40, 2)[:, 0]),
    dict(bias=torch.zeros(3, 40)), dict(gate=torch.zeros(1), resid=torch.zeros(3, 40)),
    dict(gate=torch.zeros(40, dtype=BF16), resid=torch.zeros(3, 40)), dict(resid=torch.zeros(40)), dict(resid=torch.zeros(2, 40)),
    dict(resid=torch.zeros(3, 40, dtype=F16)), dict(resid=torch.zeros(40, 3).t()), dict(out=torch.zeros(3, 39)),
    dict(out=torch.zeros(3, 40, dtype=F16)), dict(out=torch.zeros(40, 3).t()), dict(out=torch.zeros(120)),
    dict(packed=lambda size: torch.zeros(size - 1, dtype=torch.uint8)), dict(packed=lambda size: torch.zeros(2 * size, dtype=torch.uint8)[::2]),
])
def test_vec_operands_that_do_not_fit_are_refused(lib_calls, packed_sizes, wtype, kw):
    refused(lib_calls, vec, wtype=wtype, **kw)


def test_vec_operands_that_fit(lib_calls, packed_sizes):
    wide = torch.zeros(3, 50)
    args = accepted(lib_calls, "b2q_mul_vec", vec, bias=torch.zeros(40), gate=torch.zeros(1, 40), resid=wide[:, 1:41], out=wide[:, 1:41])
    assert args[11] == args[13] == 200
    for kw in (dict(m=0, resid=torch.zeros(0, 40)), dict(m=1, out=torch.zeros(1, 40)), dict(x=torch.zeros(3, 512, dtype=BF16)),
               dict(packed=lambda size: torch.zeros(size + 9, dtype=torch.uint8))):
        lib_calls.clear()
        accepted(lib_calls, "b2q_mul_vec", vec, **kw)


# ------------------------------------------------------------------------------------------------ outputs of the plan
def plan_out(**kw):
    """The five outputs for 3 requests and 40 tokens."""
    o = dict(slots=torch.zeros(40, dtype=I64), positions=torch.zeros(40, dtype=I32), cu=torch.zeros(4, dtype=I32),
             kv_len=torch.zeros(3, dtype=I32), counts=torch.zeros(2, dtype=I32))
    o.update(kw)
    return tuple(o.values())


@pytest.mark.parametrize("kw", [
    dict(slots=torch.zeros(39, dtype=I64)), dict(slots=torch.zeros(40, dtype=I32)), dict(slots=torch.zeros(80, dtype=I64)[::2]),
    dict(positions=torch.zeros(39, dtype=I32)), dict(positions=torch.zeros(40, dtype=torch.int16)), dict(cu=torch.zeros(3, dtype=I32)),
    dict(cu=torch.zeros(8, dtype=I32)[::2]), dict(kv_len=torch.zeros(2, dtype=I32)), dict(counts=torch.zeros(1, dtype=I32)),
    dict(kv_len=torch.zeros(3, dtype=torch.int8)),
])
def test_plan_outputs_that_do_not_fit_are_refused(lib_calls, kw):
    refused(lib_calls, plan, out=plan_out(**kw))


def test_plan_outputs_that_fit(lib_calls):
    out = plan_out()
    args = accepted(lib_calls, "b2q_kv_cache_plan", plan, out=out)
    assert args[10:15] == tuple(t.data_ptr() for t in out)
    lib_calls.clear()
    accepted(lib_calls, "b2q_kv_cache_plan", plan, out=plan_out(slots=torch.zeros(50, dtype=I64)))  # room to spare


# --------------------------------------------------------------------------------- output and workspace of the attention
@pytest.mark.parametrize("kw", [
    dict(out=torch.zeros(6, 256)), dict(out=torch.zeros(6, 256, dtype=BF16)), dict(out=torch.zeros(5, 256, dtype=F16)),
    dict(out=torch.zeros(6, 128, dtype=F16)), dict(out=torch.zeros(256, 6, dtype=F16).t()),
    dict(ws=torch.zeros(4096, dtype=torch.uint8)[::2]),
])
def test_attention_operands_that_do_not_fit_are_refused(lib_calls, kw):
    refused(lib_calls, attention, **kw)


def test_attention_operands_that_fit(lib_calls):
    out, ws = torch.zeros(9, 280, dtype=F16)[:6, 8:264], torch.zeros(512, dtype=torch.uint8)
    args = accepted(lib_calls, "b2q_attention_paged", attention, out=out, ws=ws)
    assert args[23:27] == (out.data_ptr(), 560, ws.data_ptr(), 512)
    lib_calls.clear()
    assert accepted(lib_calls, "b2q_attention_paged", attention, ws=torch.zeros(64))[26] == 256


def test_outputs_may_have_rows_and_columns_to_spare(lib_calls, packed_sizes):
    """What lies past them is left alone."""
    accepted(lib_calls, "b2q_attention_paged", attention, out=torch.zeros(9, 264, dtype=F16))
    lib_calls.clear()
    accepted(lib_calls, "b2q_qkv_rope_cache", rope, out=torch.zeros(9, HQ * D_ + 8, dtype=F16))
    lib_calls.clear()
    accepted(lib_calls, "b2q_mul_vec", vec, out=torch.zeros(8, 44), resid=torch.zeros(4, 40))


# --------------------------------------------------------------------------------------------------------- devices
class On:
    """A tensor as far as its device goes."""

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


@pytest.mark.parametrize("devices", [(-1,), (0, -1), (0, 0, 1), (1, 0)])
def test_operands_on_the_host_or_on_several_devices_are_refused(devices):
    with pytest.raises(AssertionError):
        b2q._raw_stream(types.SimpleNamespace(cuda_stream=7), *(On(d) for d in devices))


def test_operands_on_one_device_are_taken():
    assert b2q._raw_stream(types.SimpleNamespace(cuda_stream=7), On(1), None, On(1)) == 7


@pytest.mark.parametrize("call,device_operands", [
    (plan, 4), (lambda **kw: plan(out=plan_out(), **kw), 9), (rope, 7), (lambda **kw: rope(norm=True, gamma_k=torch.ones(128), **kw), 8),
    (attention, 7), (lambda **kw: attention(ws=torch.zeros(64), **kw), 8), (lambda **kw: vec(bias=torch.zeros(40), **kw), 4),
])
def test_every_operand_is_looked_at(lib_calls, packed_sizes, monkeypatch, call, device_operands):
    looked = []
    monkeypatch.setattr(b2q, "_raw_stream", lambda stream, *t: looked.extend(x for x in t if x is not None) or 0)
    call()
    assert len(looked) == device_operands
