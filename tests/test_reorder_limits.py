"""What a reorder call counts in 32 bits: the sizes up to which it is taken, on the host."""
import re

import numpy as np
import pytest

from tests.test_abi_fuzz import lib  # noqa: F401  (skips where a GPU is visible)
from tests.test_paged import desc

_MEM = np.zeros(4096, np.uint8)
PTR = _MEM.ctypes.data


def call(L, N=1, B=2, Hk=1, D=64, page_size=16, count=1):
    layers = (L.TensionPaged * count)(*[desc(page_size=page_size)] * count)
    r = L.lib().tension_paged_reorder(layers, count, PTR + 64, 4, PTR, PTR, 2, 1, N, B, Hk, D, None)
    return r, (L.lib().tension_last_error() or b"").decode()


@pytest.mark.parametrize("kw,match", [
    (dict(page_size=(1 << 22) + 1), "2\\^28 values"), (dict(Hk=1 << 12, page_size=(1 << 10) + 1), "2\\^28 values"),
    (dict(Hk=0xffff, D=0xffff), "2\\^28 values"), (dict(N=254201, B=1), "bad sizes"), (dict(N=3972, B=64), "bad sizes"),
    (dict(count=4097), "bad sizes"),
])
def test_refused(lib, kw, match):  # noqa: F811
    r, message = call(lib, **kw)
    assert r == lib.ERR_ARG
    assert re.search(match, message), message


@pytest.mark.parametrize("kw", [dict(page_size=1 << 22), dict(Hk=1 << 12, page_size=1 << 10), dict(N=254200, B=1), dict(N=3971, B=64),
                                dict(count=4096)])
def test_taken(lib, kw):  # noqa: F811
    """As far as the launch, which there is no device for."""
    r, message = call(lib, **kw)
    assert r == lib.ERR_LAUNCH, message
