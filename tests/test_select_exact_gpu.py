"""Scores of beam selection to 64 bits: what the definition settles exactly comes
out so, in one launch, over spans, and over many lists."""
import math

import numpy as np
import pytest
import torch

from bozo_amd import beam_select
from oracle import serving_ref as R

pytestmark = pytest.mark.gpu

# B, V, K: one launch, one and several spans of a vocabulary, many lists
SIZES = [(2, 1, 1), (2, 7, 2), (4, 2048, 4), (16, 2000, 32), (2, 2049, 2), (4, 20000, 16), (17, 300, 8), (64, 20000, 64), (40, 9000, 50)]


def select(x, s, K, ended=None, pad=0):
    out = beam_select(x, s, K, ended=ended, pad=pad)
    want = R.select(x.float().cpu().numpy(), s.cpu().numpy(), K, None if ended is None else ended.cpu().numpy(), pad)
    return [t.cpu().numpy() for t in out], want


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V,K", SIZES)
def test_one_live_token_has_log_probability_zero(B, V, K, dt):
    """A beam with one token above -inf, wherever it lies and whatever its logit: its score is the beam's."""
    x = torch.full((3, B, V), -math.inf, device="cuda", dtype=dt)
    for n in range(3):
        for b in range(B):
            x[n, b, (n * 977 + b * 8191) % V] = (b - 3) * 7.5 * (n + 1)
    s = torch.zeros(3, B, device="cuda")
    s[1] = -torch.arange(B, device="cuda") * 0.37
    s[2] = -1.0
    (out, tok, par), (want, wt, wp) = select(x, s, K)
    assert np.array_equal(out, want.astype(np.float32)) and np.array_equal(tok, wt) and np.array_equal(par, wp)
    assert np.array_equal(out[0, :min(B, K)], np.zeros(min(B, K), np.float32))


@pytest.mark.parametrize("ended_first", [True, False])
@pytest.mark.parametrize("B,V,K", SIZES)
def test_ended_and_forced_beams_tie(B, V, K, ended_first):
    """An ended beam and one whose next token is certain, of one score: the lower place first, with one kept too."""
    x = torch.full((1, B, V), -math.inf, device="cuda")
    x[:, :, V - 1] = 3.25
    ended = torch.zeros(1, B, dtype=torch.bool, device="cuda")
    ended[:, (0 if ended_first else 1)::2] = True
    s = torch.full((1, B), -1.0, device="cuda")
    for k in sorted({1, min(2, B * V), K}):
        (out, tok, par), (want, wt, wp) = select(x, s, k, ended, V // 2)
        assert np.array_equal(tok, wt) and np.array_equal(par, wp) and np.array_equal(out, want.astype(np.float32)), k
        assert par[0, 0] == 0 and tok[0, 0] == (V // 2 if ended_first else V - 1)


@pytest.mark.parametrize("B,V,K", [c for c in SIZES if c[1] > 1])
def test_scores_to_64_bits(B, V, K):
    """Log probabilities that are nothing but a small sum, and ordinary ones.

    A sum's exponentials are off by 2^-52 of their exponents (ln V of them on the whole, 14 at most), 2^-51 of their own
    and 2^-47 by their order, its logarithm by that and 2^-50 of itself, the oracle's likewise: 2^-45 covers both.  Then one rounding."""
    g = torch.Generator(device="cuda").manual_seed(V)
    near = -24 - 6 * torch.rand(2, B, V, generator=g, device="cuda")
    near[:, :, V // 3] = 0.0
    wide = torch.randn(2, B, V, generator=g, device="cuda") * 3
    for x in (near, wide):
        for score in (0.0, -2.5):
            s = torch.full((2, B), score, device="cuda")
            (out, tok, par), _ = select(x, s, K)
            full = {}
            y = x.double().cpu().numpy()
            c = score + y - y.max(-1, keepdims=True) - np.log(np.exp(y - y.max(-1, keepdims=True)).sum(-1, keepdims=True))
            for n in range(2):
                want = c[n, par[n], tok[n]]
                assert (np.abs(out[n] - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -45).all()
                assert (np.diff(want) <= 2.0 ** -45).all()
                assert want[-1] >= np.sort(c[n].ravel())[-K] - 2.0 ** -45


@pytest.mark.parametrize("B,V", [(2, 2000), (2, 20000), (64, 20000)])
def test_beams_that_are_close(B, V):
    """Gaps far below a float32's step of the sum of exponentials, far above its 64-bit error: the order is theirs."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = -22 - 4 * torch.rand(1, 1, V, generator=g, device="cuda").expand(1, B, V).contiguous()
    x[:, :, 5] = 0.0
    y = x[0, 0].double().cpu().numpy()
    own = -np.log(np.exp(y).sum())  # of beam 1, some 1e-6
    ended = torch.ones(1, B, dtype=torch.bool, device="cuda")
    ended[0, 1] = False
    for k in range(-30, 31):
        other = np.float32(own)
        for _ in range(abs(k)):
            other = np.nextafter(other, np.float32(-1 if k < 0 else 1))
        if abs(float(other) - own) < 2.0 ** -44:
            continue
        s = torch.full((1, B), -5.0, device="cuda")
        s[0, 0], s[0, 1] = float(other), 0.0
        (out, tok, par), _ = select(x, s, 2, ended, 9)
        assert par[0].tolist() == ([0, 1] if other > own else [1, 0]), (k, float(other), own)
        assert tok[0].tolist() == ([9, 5] if other > own else [5, 9])


@pytest.mark.parametrize("B,V,K", [(1, 2048, 4), (1, 2049, 4), (3, 2048, 32), (3, 2049, 32), (4, 20000, 16), (5, 300, 64), (64, 20000, 64),
                                   (17, 1000, 33), (1, 1 << 20, 64)])
def test_logits_that_scores_do_not_tell_apart(B, V, K):
    """Within a beam the order is the logits', also where a score rounds away what they differ by: on every path."""
    g = torch.Generator(device="cuda").manual_seed(V + B)
    x = 1e-17 * torch.randn(2, B, V, generator=g, device="cuda")  # against a logarithm of ln V
    s = torch.zeros(2, B, device="cuda")
    x[1], s[1] = x[1] * 1e9, -1e9
    x[1, 1:] = -math.inf
    x[1, :, V // 2:] = x[1, :, :V - V // 2].clone()  # and logits that are equal
    (out, tok, par), (want, wt, wp) = select(x, s, K)
    assert np.array_equal(tok, wt) and np.array_equal(par, wp)
    assert np.array_equal(np.sort(-x[0, 0].cpu().numpy())[:min(K, V)], -x[0, 0].cpu().numpy()[tok[0]][:min(K, V)])
    y = torch.randn(1, B, V, generator=g, device="cuda").bfloat16()  # one beam, whose score leaves steps of 2 or more
    s = torch.full((1, B), -math.inf, device="cuda")
    s[0, B // 2] = -1e16
    (out, tok, par), _ = select(y, s, min(K, V))
    want = np.lexsort((np.arange(V), -y[0, B // 2].double().cpu().numpy()))[:min(K, V)]
    assert (par == B // 2).all() and np.array_equal(tok[0], want)


def microseconds(x, s, K):
    """Of a call, the least of several runs of ten."""
    times = []
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            beam_select(x, s, K)
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 100)
    return min(times[1:])


@pytest.mark.parametrize("B,V,K", [(16, 200, 32), (16, 130, 32), (8, 100, 16), (1, 250, 32), (1, 128, 32), (1, 129, 17), (2, 250, 32), (3, 9, 20),
                                   (16, 17, 32), (5, 255, 31)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_short_rows(B, V, K, dt):
    """Vocabularies that fill few lanes: right, and no slower by orders than ones that fill all."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(3, B, V, generator=g, device="cuda") * 2).to(dt)
    s = -torch.rand(3, B, generator=g, device="cuda")
    ended = torch.rand(3, B, generator=g, device="cuda") < 0.3
    for e in (None, ended):
        (out, tok, par), (want, wt, wp) = select(x, s, K, e, V - 1)
        assert np.array_equal(tok, wt) and np.array_equal(par, wp)
    full = torch.randn(3, B, 2048, generator=g, device="cuda").to(dt)
    assert microseconds(x, s, K) <= 25 * microseconds(full, s, K)


@pytest.mark.parametrize("B,V,K", [(1, 2048, 4), (1, 2048, 1), (2, 2000, 32), (4, 500, 8), (4, 2048, 32), (16, 2048, 32), (16, 128, 32), (7, 777, 5),
                                   (16, 2049, 32), (3, 8192, 64), (64, 20000, 64)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_many_equal_scores(B, V, K, dt):
    """Rows of one value, or of three; beams at their end, beams that run out of tokens: right, and no slower by orders."""
    g = torch.Generator(device="cuda").manual_seed(V + B)
    zeros = torch.zeros(2, B, V, device="cuda", dtype=dt)
    few = torch.randint(0, 3, (2, 1, V), generator=g, device="cuda").to(dt).expand(2, B, V).contiguous()
    few[:, :, ::5] *= -0.0
    scores = torch.zeros(2, B, device="cuda")
    scores[1] = -0.25 * (torch.arange(B, device="cuda") % 3)
    ended = torch.rand(2, B, generator=g, device="cuda") < 0.3
    out_of = few.clone()
    out_of[:, 0, 3:] = -math.inf
    out_of[0, B // 2, 1:] = -math.inf
    for x in (zeros, few, out_of):
        for e in (None, ended):
            (out, tok, par), (want, wt, wp) = select(x, scores, K, e, V // 2)
            assert np.array_equal(tok, wt) and np.array_equal(par, wp)
    usual = torch.randn(2, B, V, generator=g, device="cuda").to(dt)
    assert max(microseconds(zeros, scores, K), microseconds(few, scores, K)) <= 25 * microseconds(usual, scores, K)
