"""Paged cache on the CPU: refusals (Python and C ABI), the launch's split, and
the oracle's quantiser against torch's conversion."""
import ctypes as C

import numpy as np
import pytest
import torch

import bozo_amd
from bozo_amd import PagedKV, _lib as L, paged
from oracle import paged_ref as R

F8 = torch.float8_e4m3fn


def cache(dtype=F8, P=4, S=16, H=2, D=64):
    return PagedKV.empty(P, S, H, D, dtype, device="cpu")


TAB = torch.zeros(3, 2, dtype=torch.int32)
LEN = torch.ones(3, dtype=torch.int32)


def test_no_cpu_path():
    kv, x = cache(), torch.zeros(3, 1, 2, 64)
    for call in (lambda: bozo_amd.paged_append(kv, x, x, TAB, LEN), lambda: bozo_amd.paged_read(kv, TAB, LEN, 2),
                 lambda: bozo_amd.paged_decode(x[:, 0], kv, TAB, LEN, 8.0)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.mark.parametrize("change,error,match", [
    (dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.float64)), TypeError, "page dtype"),
    (dict(v=torch.zeros(4, 2, 16, 32).to(F8)), ValueError, "alike"),
    (dict(k=torch.zeros(2, 16, 64).to(F8)), ValueError, "alike"),
    (dict(k_exp=None), ValueError, "k_exp belongs"),
    (dict(v_exp=torch.zeros(4, 2, 16)), ValueError, "v_exp must be uint8"),
    (dict(v_exp=torch.zeros(4, 2, 15, dtype=torch.uint8)), ValueError, "v_exp must be uint8"),
    (dict(k=torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)), ValueError, "k_exp belongs"),
    (dict(k=torch.zeros(4, 2, 64, 16).to(F8).transpose(2, 3)), ValueError, "unit innermost"),
])
def test_cache_refusals(change, error, match):
    kv = cache()._replace(**change)
    with pytest.raises(error, match=match):
        paged._check_pages(kv, 3, TAB, lengths=LEN)


@pytest.mark.parametrize("table,lengths,match", [
    (TAB.long(), LEN, "table"), (TAB[:2], LEN, "table"), (TAB[0], LEN, "table"),
    (TAB, LEN.long(), "lengths"), (TAB, LEN[:2], "lengths"), (TAB, TAB, "lengths"),
])
def test_counter_refusals(table, lengths, match):
    with pytest.raises(ValueError, match=match):
        paged._check_pages(cache(), 3, table, lengths=lengths)


def test_operand_refusals():
    kv, x = cache(), torch.zeros(3, 1, 2, 64)
    with pytest.raises(ValueError, match="share one"):
        paged._check_append(kv, x, x[:, :, :1], TAB, LEN, None)
    with pytest.raises(ValueError, match="tokens of 1 heads"):
        paged._check_append(kv, x[:, :, :1], x[:, :, :1], TAB, LEN, None)
    with pytest.raises(ValueError, match="counts"):
        paged._check_append(kv, x, x, TAB, LEN, LEN[:1])
    with pytest.raises(TypeError, match="float64"):
        paged._check_append(kv, x.double(), x.double(), TAB, LEN, None)
    with pytest.raises(TypeError, match="do not go"):
        paged._check_append(cache(torch.float32), x.bfloat16(), x, TAB, LEN, None)
    with pytest.raises(ValueError, match="q must be"):
        paged._check_decode(x, kv, TAB, LEN, 0, 0)
    with pytest.raises(TypeError, match="q: unsupported"):
        paged._check_decode(x[:, 0].double(), kv, TAB, LEN, 0, 0)
    with pytest.raises(ValueError, match="multiple"):
        paged._check_decode(torch.zeros(3, 5, 64), kv, TAB, LEN, 0, 0)
    with pytest.raises(ValueError, match="window must"):
        bozo_amd.paged_decode(x[:, 0], kv, TAB, LEN, 8.0, window=0)
    with pytest.raises(TypeError, match="page dtype"):
        PagedKV.empty(2, 16, 2, 64, torch.float64, device="cpu")
    with pytest.raises(ValueError, match=">= 1"):
        PagedKV.empty(0, 16, 2, 64, device="cpu")


# ------------------------------------------------------------------ C ABI

_MEM = np.zeros(4096, np.uint8)


def buf(dt=L.BF16, strides=(4096, 64, 64, 1), ptr=None):
    return L.TensionBuf(C.c_void_p(_MEM.ctypes.data if ptr is None else ptr or None), dt, 0, (C.c_int64 * 4)(*strides))


def desc(**kw):
    none = L.TensionBuf()
    d = dict(k=buf(), v=buf(), k_exp=none, v_exp=none, table=_MEM.ctypes.data, table_stride=2, table_len=2, pages=4,
             page_size=16)
    d.update(kw)
    return L.TensionPaged(*(d[n] for n, _ in L.TensionPaged._fields_))


def decode(c=None, q=None, out=None, lengths=_MEM.ctypes.data, ws=_MEM.ctypes.data, N=3, H=2, Hk=2, D=64, W=0, most=0,
           scale=8.0, flags=1):
    ref = lambda x, d: C.byref(x if x is not None else d)  # noqa: E731
    return L.lib().tension_paged_decode(ref(c, desc()), ref(q, buf(strides=(128, 64, 1, 0))),
                                        ref(out, buf(strides=(128, 64, 1, 0))), lengths, ws, N, H, Hk, D, W, most, scale,
                                        flags, None)


@pytest.mark.parametrize("kw", [
    dict(N=-1), dict(H=3), dict(Hk=0), dict(D=0), dict(D=257), dict(W=-1), dict(W=1 << 40), dict(most=-1),
    dict(N=1 << 40), dict(scale=0.0), dict(scale=float("nan")), dict(flags=3), dict(lengths=None),
    dict(q=buf(strides=(128, 64, 2, 0))), dict(q=buf(L.F32, (128, 64, 1, 0))), dict(q=buf(9)),
    dict(c=desc(k=buf(strides=(4096, 64, 64, 2)))), dict(c=desc(k=buf(L.F64))), dict(c=desc(k=buf(ptr=0))),
    dict(c=desc(k=buf(L.E4M3))), dict(c=desc(k_exp=buf(L.U8))), dict(c=desc(k=buf(L.E4M3), k_exp=buf(L.BF16))),
    dict(c=desc(table=None)), dict(c=desc(pages=0)), dict(c=desc(pages=1 << 31)), dict(c=desc(page_size=0)),
    dict(c=desc(page_size=1 << 40)), dict(c=desc(table_len=-1)), dict(c=desc(table_len=1 << 31)),
    dict(c=desc(table_len=4096), N=1, ws=None),
], ids=str)
def test_abi_decode_refusals(kw):
    assert decode(**kw) == L.ERR_ARG and L.lib().tension_last_error()


def test_abi_float64_is_unsupported():
    assert decode(q=buf(L.F64, (128, 64, 1, 0)), out=buf(L.F64, (128, 64, 1, 0))) == L.ERR_UNSUPPORTED


@pytest.mark.parametrize("name", ["tension_paged_append", "tension_paged_read"])
def test_abi_rows_refusals(name):
    fn = getattr(L.lib(), name)
    good = dict(c=C.byref(desc()), k=C.byref(buf()), v=C.byref(buf()), start=_MEM.ctypes.data, counts=None, N=1, T=1,
                Hk=2, D=64, stream=None)
    for kw in (dict(c=None), dict(k=None), dict(v=None), dict(start=None), dict(N=-1), dict(T=-1), dict(Hk=-1),
               dict(D=0), dict(D=1 << 20), dict(T=1 << 31), dict(N=1 << 40), dict(Hk=1 << 40),
               dict(k=C.byref(buf(L.E4M3))), dict(c=C.byref(desc(pages=0))),
               dict(c=C.byref(desc(v=buf(strides=(4096, 64, 64, 3)))))):
        assert fn(*(good | kw).values()) == L.ERR_ARG, kw
    assert fn(*(good | dict(k=C.byref(buf(L.F64)))).values()) == L.ERR_UNSUPPORTED
    assert fn(*(good | dict(N=0, c=None, k=None, start=None)).values()) == L.OK  # nothing to do
    if name.endswith("append"):
        for dt in (L.F16, L.BF16):
            other = C.byref(desc(k=buf(L.F16 if dt == L.BF16 else L.BF16)))
            assert fn(*(good | dict(c=other, k=C.byref(buf(dt)))).values()) == L.ERR_ARG


def test_workspace_sizes():
    ws = L.lib().tension_paged_decode_workspace
    r = np.random.default_rng(0)
    pick = [0, 1, 2, 12, 16, 64, 100, 1000, 65536, (1 << 31) - 1, 1 << 31, 1 << 40, -1, (1 << 63) - 1]
    for _ in range(5000):
        a = [int(x) for x in r.choice(np.array(pick, dtype=object), 8)]
        assert ws(*a) >= -1
    assert ws(64, 12, 12, 64, 256, 0, 4096, 16) == 0 or ws(64, 12, 12, 64, 256, 0, 4096, 16) % 4 == 0
    assert ws(1, 12, 12, 64, 0, 32768, 4096, 16) > 0   # few rows, a long axis: split
    assert ws(128, 16, 16, 64, 0, 4096, 64, 64) == 0   # rows enough
    assert ws(1, 3, 2, 64, 0, 0, 16, 16) == -1


# ------------------------------------------------------------------ the oracle's quantiser

def test_quantiser_rounds_as_torch_converts():
    x = torch.randn(500, 48, generator=torch.Generator().manual_seed(0)) * torch.exp2(torch.randint(-30, 30, (500, 1)).float())
    val, byte = R.quantise(x.numpy())
    e = torch.from_numpy(byte.astype(np.float64)) - 127
    top = x.double().abs().amax(-1)
    assert bool((top <= 448 * torch.exp2(e)).all()) and bool((top > 448 * torch.exp2(e - 1)).all())
    y = (x.double() * torch.exp2(-e)[:, None]).float()  # exact: a power of two
    assert np.array_equal(y.to(F8).double().numpy() * np.exp2(e.numpy())[:, None], val)
