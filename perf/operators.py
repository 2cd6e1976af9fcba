"""The paged-cache operators on the work a serving program gives them: cases that can be timed and checked.

A case is one of three kinds:

* ``store``   new tokens written into the pages (``paged_append``): one token a sequence in a decode step, or
  whole prompts.  Quantised pages are read back with ``paged_read``, so that the outputs are the values the codes
  stand for; pages of a 16- or 32-bit type are returned themselves;
* ``read``    cached tokens read back dense (``paged_read``): what a prompt that continues on cached tokens takes;
* ``decode``  one new token a sequence over its cached tokens (``paged_decode``).

``pages`` names the cache's element type (``mixed``: float32 keys with bf16 values, the model's own flow under
autocast), ``flow`` the type of the tokens, the queries or the dense rows.

With ``own`` false, ``run`` computes the operators in elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}


def _types(name):
    """Element types of keys and values."""
    return ("f32", "bf16") if name == "mixed" else (name, name)


def listed():
    return [
        # One decode step's new tokens of the 117M model's width, 64 sequences, into a quantised cache.
        dict(name="store_step_e4m3", kind="store", flow="bf16", pages="e4m3", N=64, T=1, Hk=12, D=64, S=16, L=900,
             ragged=True, fused=False),
        # Prompts of different lengths (up to the model's 1024 tokens) as the prefill hands them over.
        dict(name="store_prompts_e4m3", kind="store", flow="bf16", pages="e4m3", N=8, T=1024, Hk=12, D=64, S=64, L=0,
             ragged=True, fused=False),
        # A large prefill at the 350M width into bf16 pages; keys and values are views of one fused projection.
        dict(name="store_prompts_bf16", kind="store", flow="bf16", pages="bf16", N=32, T=1000, Hk=16, D=64, S=16, L=0,
             ragged=False, fused=True),
        # The last 256 tokens of 16 sequences, for local layers of a prompt that continues: window 256.
        dict(name="read_window_e4m3", kind="read", flow="bf16", pages="e4m3", N=16, T=256, Hk=16, D=64, S=16, L=1024,
             ragged=True),
        # Whole conversations for the global layers of a continued prompt, quantised pages, odd length.
        dict(name="read_long_e4m3", kind="read", flow="bf16", pages="e4m3", N=4, T=16381, Hk=12, D=64, S=64, L=16381,
             ragged=False),
        # The smallest decode: one sequence of the 117M model, every earlier token (a global layer).
        dict(name="decode_one_bf16", kind="decode", flow="bf16", pages="bf16", N=1, H=12, Hk=12, D=64, S=16, L=777,
             W=0, ragged=False, own_key=True, norm="mass"),
        # A local layer of the 350M preset (H16, W256): 64 sequences of different lengths.
        dict(name="decode_window_bf16", kind="decode", flow="bf16", pages="bf16", N=64, H=16, Hk=16, D=64, S=16,
             L=1024, W=256, ragged=True, own_key=False, norm="mass"),
        # A local layer of the 117M model under autocast (float32 keys, bf16 values), valid-count normalised.
        dict(name="decode_window_mixed", kind="decode", flow="f32", pages="mixed", N=48, H=12, Hk=12, D=64, S=16,
             L=1000, W=64, ragged=True, own_key=False, norm="count"),
        # A global layer over 2048 tokens, quantised cache, sequences of different lengths.
        dict(name="decode_global_e4m3", kind="decode", flow="bf16", pages="e4m3", N=64, H=12, Hk=12, D=64, S=64,
             L=2048, W=0, ragged=True, own_key=True, norm="mass"),
        # Two long conversations, four query heads to a key head, head dim 128: few rows, a long axis.
        dict(name="decode_long_shared_e4m3", kind="decode", flow="bf16", pages="e4m3", N=2, H=16, Hk=4, D=128, S=64,
             L=65500, W=0, ragged=False, own_key=True, norm="mass"),
        # The model without autocast: everything float32.
        dict(name="decode_global_f32", kind="decode", flow="f32", pages="f32", N=16, H=12, Hk=12, D=64, S=32, L=2000,
             W=0, ragged=True, own_key=True, norm="mass"),
        # A full batch over long bf16 caches: the largest stream.
        dict(name="decode_batch_bf16", kind="decode", flow="bf16", pages="bf16", N=128, H=16, Hk=16, D=64, S=64,
             L=4096, W=0, ragged=True, own_key=True, norm="mass"),
    ]


# ------------------------------------------------------------------ sizes of a case

def _spread(n, top, ragged):
    """n lengths up to ``top``: all alike, or evenly from a quarter of it."""
    if not ragged or n == 1:
        return [top] * n
    return [max(1, top - (top * 3 // 4) * i // (n - 1)) for i in range(n)]


def _range(case, length):
    """Keys [lo, hi) that the newest of ``length`` tokens attends to."""
    hi = length if case["own_key"] else length - 1
    return (max(0, length - 1 - case["W"]) if case["W"] else 0), hi


def _row_bytes(types, D):
    return sum(D * _BYTES[t] + (1 if t == "e4m3" else 0) for t in types)


def work(case):
    D, N = case["D"], case["N"]
    cached = _row_bytes(_types(case["pages"]), D)
    if case["kind"] == "decode":
        keys = sum(max(0, hi - lo) for lo, hi in (_range(case, n) for n in _spread(N, case["L"], case["ragged"])))
        return {"bytes": keys * case["Hk"] * cached + 2 * N * case["H"] * D * _BYTES[case["flow"]],
                "flops": 4.0 * keys * case["H"] * D}
    dense = _row_bytes(_types(case["flow"]), D)
    if case["kind"] == "read":  # rows of positions that hold no token are written as zeros
        rows = sum(_spread(N, case["T"], case["ragged"])) * case["Hk"]
        return {"bytes": rows * cached + N * case["T"] * case["Hk"] * dense, "flops": 2.0 * rows * D}
    rows = (N if case["T"] == 1 else sum(_spread(N, case["T"], case["ragged"]))) * case["Hk"]
    back = N * case["T"] * case["Hk"] * dense if case["pages"] == "e4m3" else 0  # read back dense
    return {"bytes": rows * (dense + cached) + back, "flops": 6.0 * rows * D}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = {k: max(work(c)["bytes"] for c in listed() if c["kind"] == k) for k in ("store", "read", "decode")}
    while True:
        kind = rng.choices(("store", "read", "decode"), (0.25, 0.2, 0.55))[0]
        D, S = rng.choice((32, 64, 64, 64, 128)), rng.choice((16, 16, 32, 64, 128))
        heads = rng.choice((4, 8, 12, 16))
        if kind == "decode":
            pages, flow = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("e4m3", "bf16"), ("e4m3", "bf16"),
                                      ("e4m3", "f16"), ("e4m3", "f32"), ("f16", "f16"), ("f32", "f32"),
                                      ("mixed", "f32")))
            shared = rng.choice((1, 1, 1, 2, 4))
            case = dict(kind=kind, flow=flow, pages=pages, N=_log_int(rng, 1, 128), H=heads, Hk=heads // shared, D=D,
                        S=S, L=_log_int(rng, 1, 32768), W=rng.choice((0, 0, 0, 8, 64, 100, 256)),
                        ragged=rng.random() < 0.7, own_key=rng.random() < 0.6, norm=rng.choice(("mass", "mass", "count", "raw")))
            if not case["own_key"] and case["L"] < 8:  # sequences of one token would attend to nothing at all
                continue
        elif kind == "store":
            flow = rng.choice(("bf16", "bf16", "f16", "f32", "mixed"))
            pages = "e4m3" if rng.random() < 0.7 else flow
            T = rng.choice((1, _log_int(rng, 2, 2048)))
            case = dict(kind=kind, flow=flow, pages=pages, N=_log_int(rng, 1, 128), T=T, Hk=heads, D=D, S=S,
                        L=_log_int(rng, 1, 2048) if rng.random() < 0.5 else 0, ragged=rng.random() < 0.6,
                        fused=flow != "mixed" and rng.random() < 0.3)
        else:
            case = dict(kind=kind, flow=rng.choice(("bf16", "bf16", "f16", "f32")), pages=rng.choice(("e4m3", "e4m3", "bf16")),
                        N=_log_int(rng, 1, 32), T=_log_int(rng, 8, 8192), Hk=heads, D=D, S=S, L=0,
                        ragged=rng.random() < 0.5)
            if case["pages"] != "e4m3":
                case["flow"] = "bf16"
            case["L"] = case["T"] + _log_int(rng, 1, 2048) - 1
        if work(case)["bytes"] <= limit[kind]:
            return case


# ------------------------------------------------------------------ the quantised type

def _quantise(x):
    """Codes (as bytes) and exponent bytes of rows x [..., D]: the smallest power of two that brings the row's
    largest value within 448, codes rounded to nearest even."""
    x = x.float()
    top = x.abs().amax(-1).contiguous().view(torch.int32)
    e = ((top >> 23) - 8 + ((top & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    codes = (x * torch.exp2((127 - e).float())[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), e.to(torch.uint8)


def _values(codes, exps):
    """float32 values of codes [..., D] with exponent bytes [...]; other types as they are."""
    if exps is None:
        return codes.float()
    return codes.view(torch.float8_e4m3fn).float() * torch.exp2(exps.float() - 127.0)[..., None]


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _pool(g, P, Hk, S, D, kind):
    """Pages of one of keys / values that hold tokens everywhere (those no sequence owns are another's)."""
    if kind != "e4m3":
        return torch.randn(P, Hk, S, D, generator=g, device="cuda", dtype=_DT[kind]), None
    codes, exps = _quantise(torch.randn(P, Hk, S, D, generator=g, device="cuda", dtype=torch.bfloat16))
    return codes.view(torch.float8_e4m3fn), exps


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed))
    N, Hk, D, S, kind = case["N"], case["Hk"], case["D"], case["S"], case["kind"]
    # tokens in the cache of each sequence, the new ones included; the order of the lengths comes from the seed
    order = torch.randperm(N, generator=host)
    if kind == "decode":
        lengths = torch.tensor(_spread(N, case["L"], case["ragged"]))[order]
        counts, start = None, None
    else:
        counts = torch.tensor(_spread(N, case["T"], case["ragged"] and case["T"] > 1))[order]
        before = torch.tensor(_spread(N, case["L"], case["ragged"]))[order] if kind == "store" else case["L"] - counts
        start, lengths = before, before + counts
    used = (lengths + S - 1) // S
    P = int(used.sum()) + 1
    ids = torch.randperm(P, generator=host).to(torch.int32)
    slot = torch.arange(int(used.max()))[None, :]
    table = torch.where(slot < used[:, None], ids[(torch.cumsum(used, 0) - used)[:, None].add(slot).clamp(max=P - 1)],
                        torch.tensor(-1, dtype=torch.int32))
    s = {"case": case, "table": table.cuda(), "lengths": lengths.to(torch.int32).cuda()}
    kt, vt = _types(case["pages"])
    (k, ke), (v, ve) = _pool(g, P, Hk, S, D, kt), _pool(g, P, Hk, S, D, vt)
    s["kv"] = (k, v, ke, ve)
    if kind == "decode":
        s["q"] = _randn(g, N, case["H"], D, dtype=_DT[case["flow"]])
        return s
    s["start"] = start.to(torch.int32).cuda()
    s["counts"] = counts.to(torch.int32).cuda()
    if kind == "store":
        ft, T = _types(case["flow"]), case["T"]
        if case["fused"]:
            s["k_new"], s["v_new"] = _randn(g, N, T, Hk, 2 * D, dtype=_DT[ft[0]]).split(D, dim=-1)
        else:
            s["k_new"], s["v_new"] = _randn(g, N, T, Hk, D, dtype=_DT[ft[0]]), _randn(g, N, T, Hk, D, dtype=_DT[ft[1]])
    return s


# ------------------------------------------------------------------ the plain forms

def _places(table, pos, S):
    """Page and row of positions pos [N, n] (clamped into the table)."""
    p = pos.clamp(min=0, max=table.shape[1] * S - 1).long()
    return table.long().gather(1, p // S).clamp(min=0), p % S


def _plain_append(pages, exps, new, table, start, counts):
    pos = start[:, None] + torch.arange(new.shape[1], device=new.device)
    live = torch.arange(new.shape[1], device=new.device) < counts[:, None]
    page, row = _places(table, pos, pages.shape[2])
    page, row, x = page[live], row[live], new[live]
    if exps is None:
        pages[page, :, row] = x.to(pages.dtype)
    else:
        codes, e = _quantise(x)
        pages.view(torch.uint8)[page, :, row] = codes
        exps[page, :, row] = e


def _plain_read(pages, exps, table, start, T, counts, dtype):
    pos = start[:, None] + torch.arange(T, device=table.device)
    live = torch.arange(T, device=table.device) < counts[:, None]
    page, row = _places(table, pos, pages.shape[2])
    raw = pages if exps is None else pages.view(torch.uint8)
    x = _values(raw[page, :, row], None if exps is None else exps[page, :, row])
    return torch.where(live[..., None, None], x, x.new_zeros(())).to(dtype)


def _plain_decode(q, kv, table, lengths, scale, W, own_key, norm, L):
    k, v, ke, ve = kv
    N, H, D = q.shape
    Hk = k.shape[1]
    hi = lengths - (0 if own_key else 1)
    lo = (lengths - 1 - W).clamp(min=0) if W else torch.zeros_like(lengths)
    pos = lo[:, None] + torch.arange(min(L, W + 1) if W else L, device=q.device)
    live = pos < hi[:, None]
    page, row = _places(table, pos, k.shape[2])

    def rows(pages, exps):  # [N, Hk, n, D] in 32 bits
        raw = pages if exps is None else pages.view(torch.uint8)
        return _values(raw[page, :, row], None if exps is None else exps[page, :, row]).transpose(1, 2)

    x = torch.matmul(rows(k, ke), q.float().view(N, Hk, H // Hk, D).transpose(2, 3).contiguous()) / scale  # [N, Hk, n, G]
    tau = torch.where(live[:, None, :, None], 1.0 / (1.0 + torch.exp(-x)), x.new_zeros(()))
    out = torch.matmul(tau.transpose(2, 3), rows(v, ve))  # [N, Hk, G, D]
    if norm == "mass":
        out = out / tau.sum(2).clamp(min=1e-6)[..., None]
    elif norm == "count":
        out = out / (hi - lo).clamp(min=1).float()[:, None, None, None]
    return out.reshape(N, H, D).to(q.dtype)


# ------------------------------------------------------------------ one pass

def run(s):
    case, table, scale = s["case"], s["table"], math.sqrt(s["case"]["D"])
    if own:
        import bozo_amd
        kv = bozo_amd.PagedKV(*s["kv"])
    else:
        k, v, ke, ve = s["kv"]
    kind = case["kind"]
    if kind == "decode":
        if own:
            return bozo_amd.paged_decode(s["q"], kv, table, s["lengths"], scale, window=case["W"] or None,
                                         include_self=case["own_key"], normalize=case["norm"], max_len=case["L"])
        return _plain_decode(s["q"], s["kv"], table, s["lengths"], scale, case["W"], case["own_key"], case["norm"], case["L"])
    start, counts, T = s["start"], s["counts"], case["T"]
    if kind == "store":
        if own:
            bozo_amd.paged_append(kv, s["k_new"], s["v_new"], table, start, counts)
        else:
            _plain_append(k, ke, s["k_new"], table, start, counts)
            _plain_append(v, ve, s["v_new"], table, start, counts)
        if case["pages"] != "e4m3":
            return s["kv"][0], s["kv"][1]
    kt, vt = (_DT[t] for t in _types(case["flow"]))
    if own:
        return bozo_amd.paged_read(kv, table, start, T, (kt, vt), counts)
    return _plain_read(k, ke, table, start, T, counts, kt), _plain_read(v, ve, table, start, T, counts, vt)


# ------------------------------------------------------------------ the definition in 64 bits

def _rounded64(x):
    """float64 rows as the e4m3 cache holds them: exponent from the row's largest value, four significant bits
    (fewer below 2^-6 of the scaled value), ties to even."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, torch.where(m <= 0.875, e - 9, e - 8), torch.full_like(e, -126)).clamp(min=-126).double()
    y = x * torch.exp2(-e)
    step = torch.exp2((torch.frexp(y)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def _held64(pages, exps):
    """float64 values of the rows that pages hold."""
    if exps is None:
        return pages.double()
    b = pages.view(torch.uint8).long()
    f, m = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(f > 0, (8 + m) * torch.exp2(f.double() - 10), m * 2.0 ** -9)
    return torch.where(b >= 128, -mag, mag) * torch.exp2(exps.double() - 127)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    N, D, S, kind = case["N"], case["D"], case["S"], case["kind"]
    table, lengths = s["table"].cpu().tolist(), s["lengths"].cpu().tolist()
    k, v, ke, ve = s["kv"]

    def tokens(pages, exps, n, lo, hi):
        """[hi - lo, Hk, D] in 64 bits: the tokens lo .. hi - 1 of sequence n."""
        ids = torch.tensor(table[n][lo // S:(hi + S - 1) // S], device=pages.device)
        raw = pages if exps is None else pages.view(torch.uint8)
        x = _held64(raw[ids], None if exps is None else exps[ids])
        return x.transpose(1, 2).flatten(0, 1)[lo % S:lo % S + hi - lo]

    if kind == "decode":
        out = torch.zeros(N, case["H"], D, dtype=torch.float64, device=k.device)
        for n in range(N):
            lo, hi = _range(case, lengths[n])
            if hi <= lo:
                continue
            G = case["H"] // case["Hk"]
            K, V = tokens(k, ke, n, lo, hi).transpose(0, 1), tokens(v, ve, n, lo, hi).transpose(0, 1)  # [Hk, n, D]
            tau = torch.sigmoid((s["q"][n].double().view(-1, G, 1, D) * K[:, None]).sum(-1) / math.sqrt(D))  # [Hk, G, n]
            o = (tau[..., None] * V[:, None]).sum(2)
            if case["norm"] == "mass":
                o = o / tau.sum(-1, keepdim=True).clamp(min=1e-6)
            elif case["norm"] == "count":
                o = o / (hi - lo)
            out[n] = o.reshape(-1, D)
        return out
    counts, start, T = s["counts"].cpu().tolist(), s["start"].cpu().tolist(), case["T"]
    res = []
    for pages, exps, new in ((k, ke, s.get("k_new")), (v, ve, s.get("v_new"))):
        if kind == "store" and exps is None:  # the pages themselves, the new tokens in their places
            held = pages.clone()
            for n in range(N):
                pos = torch.arange(start[n], start[n] + counts[n], device=pages.device)
                held[torch.tensor(table[n], device=pages.device)[pos // S], :, pos % S] = new[n, :counts[n]]
            res.append(held.double())
            continue
        out = torch.zeros(N, T, case["Hk"], D, dtype=torch.float64, device=pages.device)
        for n in range(N):
            out[n, :counts[n]] = _rounded64(new[n, :counts[n]].double()) if kind == "store" else \
                tokens(pages, exps, n, start[n], start[n] + counts[n])
        res.append(out)
    return tuple(res)
