"""Seeded fuzz of the paged cache's C ABI, on a machine without a GPU: hostile
arguments, and valid descriptors with extreme sizes and strides that reach the
launch code.  Each call ends in an error with a message, or OK with nothing to
do (tests/test_abi_fuzz.py has the premise)."""
import ctypes as C
import random

import pytest

from tests.test_abi_fuzz import _BIG, _Gen, lib  # noqa: F401


def _paged(L, g, base=None):
    """A tension_paged; with ``base`` one that passes validation."""
    r, c = g.r, L.TensionPaged()
    if base is None:
        if r.random() < 0.1:
            return None
        for name in ("k", "v", "k_exp", "v_exp"):
            x = g.buf()
            if x:
                setattr(c, name, x.contents)
        c.table, c.table_stride, c.table_len, c.pages, c.page_size = g.ptr(), g.dim(), g.dim(), g.dim(), g.dim()
        return C.pointer(c)
    strides = [0, 1, 8, 64, 1000, 4096, 1 << 20, 1 << 24, 1 << 31, (1 << 40) + 8, 1 << 62, (1 << 63) - 1, -64, -(1 << 62)]
    kt = r.choice([L.BF16, L.F16, L.F32, L.E4M3])
    for side, t in (("k", kt), ("v", r.choice([kt, kt, L.BF16, L.E4M3]))):
        s = [r.choice(strides) for _ in range(3)]
        setattr(c, side, L.TensionBuf(C.c_void_p(base + r.choice([0, 0, 8, 1])), t, 0, (C.c_int64 * 4)(*s, 1)))
        if t == L.E4M3:
            s = [r.choice(strides) for _ in range(3)]
            setattr(c, side + "_exp", L.TensionBuf(C.c_void_p(base), L.U8, 0, (C.c_int64 * 4)(*s, 0)))
    c.table, c.table_stride = base, r.choice(strides)
    c.table_len = r.choice([0, 1, 2, 100, 1 << 20, (1 << 31) - 1])
    c.pages = r.choice([1, 7, 1 << 20, (1 << 31) - 1])
    c.page_size = r.choice([1, 7, 8, 16, 64, 128, 1 << 20, (1 << 30) - 1])
    return C.pointer(c)


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_random_arguments_fail_cleanly(lib, seed):  # noqa: F811
    g, h = _Gen(lib, seed), lib.lib()
    b, d, p = g.buf, g.dim, g.ptr
    calls = {
        "tension_paged_append": (lambda: (_paged(lib, g), b(), b(), p(), p(), d(), d(), d(), d(), None), slice(5, 8)),
        "tension_paged_read": (lambda: (_paged(lib, g), b(), b(), p(), p(), d(), d(), d(), d(), None), slice(5, 8)),
        "tension_paged_decode": (lambda: (_paged(lib, g), b(), b(), p(), p(), d(), d(), d(), d(), d(), d(), g.scale(),
                                          g.flags(), None), slice(5, 7)),
    }
    for name, (make, sizes) in calls.items():
        for i in range(2000):
            args = make()
            r = getattr(h, name)(*args)
            if r == lib.OK:
                assert 0 in args[sizes], f"{name} call {i}: OK without a GPU on sizes {args[sizes]}"
            else:
                assert r in (lib.ERR_ARG, lib.ERR_UNSUPPORTED, lib.ERR_LAUNCH), (name, i, r)
                assert h.tension_last_error(), (name, i)


def test_valid_descriptors_reach_launch_cleanly(lib):  # noqa: F811
    g, h = _Gen(lib, 7), lib.lib()
    r, base = g.r, (_BIG.ctypes.data + 255) // 256 * 256
    strides = [0, 1, 8, 64, 768, 1 << 20, 1 << 31, (1 << 40) + 8, 1 << 62]

    def dense(t, unit):
        s = [r.choice(strides) for _ in range(4)]
        s[unit] = 1
        return C.pointer(lib.TensionBuf(C.c_void_p(base + r.choice([0, 0, 2])), t, 0, (C.c_int64 * 4)(*s)))

    def rows():
        t = r.choice([lib.F32, lib.BF16, lib.F16])
        return (_paged(lib, g, base), dense(t, 3), dense(t, 3), base, r.choice([None, base]), r.choice([1, 64, 1 << 20]),
                r.choice([1, 5, 1000, 1 << 17]), r.choice([1, 3, 12]), r.choice([1, 20, 32, 64, 96, 128, 256, 300, 65535]), None)

    def decode():
        t, Hk = r.choice([lib.F32, lib.BF16, lib.F16]), r.choice([1, 2, 12])
        return (_paged(lib, g, base), dense(t, 2), dense(t, 2), base, base, r.choice([1, 3, 64, 1 << 16]),
                Hk * r.choice([1, 1, 2, 4, 17, 200000 // Hk]), Hk, r.choice([1, 20, 32, 64, 96, 128, 256]),
                r.choice([0, 0, 64, 1 << 29]), r.choice([0, 1, 1000, 1 << 20, 1 << 40]), r.choice([8.0, -1e-300, 1e300]),
                r.choice([0, 1, 2, 16, 17]), None)

    for name, make in (("tension_paged_append", rows), ("tension_paged_read", rows), ("tension_paged_decode", decode)):
        launched = 0
        for i in range(1500):
            res = getattr(h, name)(*make())
            assert res in (lib.ERR_ARG, lib.ERR_UNSUPPORTED, lib.ERR_LAUNCH), (name, i, res)
            assert h.tension_last_error(), (name, i)
            launched += res == lib.ERR_LAUNCH
        assert launched >= 200, f"{name}: only {launched} of 1500 calls passed validation"


def test_workspace_never_wraps(lib):  # noqa: F811
    g = _Gen(lib, 5)
    for _ in range(5000):
        a = [g.dim() for _ in range(8)]
        v = lib.lib().tension_paged_decode_workspace(*a)
        assert -1 <= v < 1 << 42
        assert min(a) >= 0 or v == -1
