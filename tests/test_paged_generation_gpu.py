"""Sequences of different lengths over paged caches (bozo_amd/paged_generation.py)
against the full forward over each sequence by itself, what the reference runs
for every token (model.py:617-652).

float32 models: 1e-5 relative, as the ring caches are held to.  Quantised
pages: against float32 pages that hold the same quantised values."""
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_read
from bozo_amd import model as M
from bozo_amd import paged_generation as G
from bozo_amd.generation import generate_cached
from tests._util import rel_l2

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def make_model(seed, dev, **kw):
    torch.manual_seed(seed)
    cfg = dict(vocab_size=80, dim=128, num_layers=4, num_heads=4, window=6, max_seq_len=48, dropout=0.0, global_every=2,
               use_rope=True, use_triton=True)
    m = M.TensionLM(M.TensionConfig(**{**cfg, **kw}))
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.05 * torch.randn_like(p))
    return m.to(dev).eval()


def tokens(seed, n, vocab=80):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed))


def err(a, b):
    return rel_l2(a.float().cpu().numpy(), b.float().cpu().numpy())


@pytest.mark.parametrize("use_rope,use_triton,heads", [(True, True, 4), (True, False, 2), (False, True, 4)])
@pytest.mark.parametrize("page_size", [4, 16, 64])
def test_steps_match_full_forward(dev, use_rope, use_triton, heads, page_size):
    """Sequences that start, grow, take whole turns and end at different
    times, in orders that change, over pages that others held before."""
    m = make_model(3, dev, use_rope=use_rope, use_triton=use_triton, num_heads=heads)
    c = G.TensionPagedCache(m, 3, 3 * -(-48 // page_size), page_size=page_size)
    text = {}

    def full(s):
        return m(text[s][None].to(dev))[0, -1]

    def start(seed, lengths):
        prompts = [tokens(seed + i, n) for i, n in enumerate(lengths)]
        seqs, logits = c.prefill(prompts)
        for s, p, row in zip(seqs, prompts, logits):
            text[s] = p
            assert err(row, full(s)) < 1e-5
        return seqs

    def step(seqs, seed):
        new = tokens(seed, len(seqs))
        logits = c.step(seqs, new)
        for i, s in enumerate(seqs):
            text[s] = torch.cat([text[s], new[i:i + 1]])
            assert err(logits[i], full(s)) < 1e-5, (s, len(text[s]))

    with torch.no_grad():
        a, b = start(10, [9, 1])
        for t in range(8):
            step([b, a] if t % 2 else [a, b], 100 + t)
        (d,) = start(20, [30])
        for t in range(5):
            step([d, a, b], 200 + t)
        more = tokens(300, 13)
        text[a] = torch.cat([text[a], more])
        assert err(c.extend(a, more), full(a)) < 1e-5
        text[b] = torch.cat([text[b], more[:1]])
        assert err(c.extend(b, more[:1]), full(b)) < 1e-5
        step([a, b, d], 301)
        c.release(a)
        (e,) = start(40, [17])
        assert e == a
        for t in range(12):
            step([e, d], 400 + t)
        assert len(text[d]) == 48
        with pytest.raises(ValueError, match="max_seq_len"):
            c.step([e, d], tokens(1, 2))
        step([e, b], 500)


def test_steps_under_autocast(dev):
    """The model's autocast flow (float32 keys, bf16 values in the local
    layers, bf16 in the global ones): 2e-2 relative, the bound of the ring
    caches' bf16 step."""
    m = make_model(4, dev, num_heads=2, window=64, max_seq_len=320, vocab_size=512)
    c = G.TensionPagedCache(m, 3, 3 * 5)
    prompts = [tokens(30 + n, n, 512) for n in (250, 70, 3)]
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        seqs, _ = c.prefill(prompts)
        for t in range(6):
            new = tokens(50 + t, 3, 512)
            got = c.step(seqs, new)
            for i in range(3):
                prompts[i] = torch.cat([prompts[i], new[i:i + 1]])
                assert err(got[i], m(prompts[i][None].to(dev))[0, -1]) < 2e-2
    assert c.layers[0].k.dtype == torch.float32 and c.layers[0].v.dtype == torch.bfloat16
    assert c.layers[1].k.dtype == torch.bfloat16


def test_quantised_pages(dev, monkeypatch):
    """e4m3 pages give what float32 pages with the same quantised values give."""
    m = make_model(5, dev, num_heads=2)
    prompts, turn = [tokens(60 + n, n) for n in (20, 7)], tokens(70, 9)

    def rounded(x):
        """[N, T, H, D] through an e4m3 cache and back."""
        N, T, H, D = x.shape
        kv = PagedKV.empty(N, T, H, D, F8, device=x.device)
        table = torch.arange(N, dtype=torch.int32, device=x.device)[:, None]
        zero = torch.zeros(N, dtype=torch.int32, device=x.device)
        paged_append(kv, x, x, table, zero)
        return paged_read(kv, table, zero, T, x.dtype)[0]

    def run(dtype):
        c = G.TensionPagedCache(m, 2, 2 * 12, page_size=4, dtype=dtype)
        seqs, _ = c.prefill(prompts)
        out = [c.step(seqs, tokens(80 + t, 2)) for t in range(9)]
        out.append(c.extend(seqs[0], turn)[None])
        out += [c.step(seqs[::-1], tokens(90 + t, 2)) for t in range(3)]
        assert c.layers[0].k.dtype == (dtype or torch.float32)
        return torch.cat(out)

    a = run(F8)
    monkeypatch.setattr(G, "paged_append", lambda kv, k, v, *rest: paged_append(kv, rounded(k), rounded(v), *rest))
    b = run(None)
    assert err(a, b) < 1e-5
    monkeypatch.undo()
    assert err(a, run(None)) > 1e-4  # the quantised values were used


def test_generate_batch(dev):
    """Prompts of different lengths together, each as ``generate_cached``
    continues it by itself (greedy: one token holds the whole nucleus)."""
    m = make_model(6, dev)
    prompts = [tokens(n, n).tolist() for n in (20, 3, 41)]
    out = G.generate_batch(m, prompts, max_new=12, top_p=1e-9, page_size=16)
    for p, o in zip(prompts, out):
        assert o == generate_cached(m, p, max_new=min(12, 48 - len(p)), top_p=1e-9)
    assert [len(o) for o in out] == [32, 15, 48]
    assert G.generate_batch(m, [], 5) == [] and G.generate_batch(m, [[1, 2]], 0) == [[1, 2]]
    with pytest.raises(ValueError, match="max_seq_len"):
        G.generate_batch(m, [[1] * 49], 5)
    q = G.generate_batch(m, prompts, max_new=4, dtype=F8)
    assert [len(o) for o in q] == [24, 7, 45]
