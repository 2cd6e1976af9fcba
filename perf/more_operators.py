"""Operators of paged generation with 4-bit caches and beams, on the work a serving program gives them.

A case is one of five kinds:

* ``store``    new tokens written into 4-bit pages (``paged_append`` by table and start, or ``paged_store`` by slots) and
  read back (``paged_read``), so that the outputs are the values the codes stand for;
* ``decode``   one new token a sequence over its cached tokens in 4-bit pages (``paged_decode``);
* ``plan``     pages taken for the tokens of a step or of whole prompts and their slots (``paged_plan``), and given back
  again: a drafted step that is cut back, or sequences that come and end;
* ``select``   the best continuations of a group's beams over the vocabulary (``beam_select``);
* ``reorder``  the beams' tables after a selection, and the copies of pages that two beams go on from
  (``paged_reorder``).

4-bit rows hold e2m1 codes, two to a byte (the first in the low half), and an exponent byte for every 32 values: the
smallest power of two that brings the 32's largest value within 6.

With ``own`` false, ``run`` computes the operators in elementary torch operations in 32 bits (``select``'s scores in 64,
where two candidates may lie next to each other).
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_GROUP = 32  # values that share an exponent


def listed():
    return [
        # One decode step's new tokens of the 117M model's width, 64 sequences, slots from the step's plan.
        dict(name="store_step", kind="store", flow="bf16", N=64, T=1, Hk=12, D=64, S=16, L=900, ragged=True, fused=False,
             slots=True),
        # Prompts of different lengths at the 350M width; keys and values are views of one fused projection.
        dict(name="store_prompts", kind="store", flow="bf16", N=16, T=1000, Hk=16, D=64, S=64, L=0, ragged=True,
             fused=True, slots=False),
        # The smallest decode: one sequence of the 117M model, every earlier token (a global layer).
        dict(name="decode_one", kind="decode", flow="bf16", N=1, H=12, Hk=12, D=64, S=16, L=777, W=0, ragged=False,
             own_key=True, norm="mass"),
        # A local layer of the 350M preset (H16, W256): 64 sequences of different lengths.
        dict(name="decode_window", kind="decode", flow="bf16", N=64, H=16, Hk=16, D=64, S=16, L=1024, W=256, ragged=True,
             own_key=False, norm="mass"),
        # Two long conversations, four query heads to a key head, head dim 128: few rows, a long axis.
        dict(name="decode_long_shared", kind="decode", flow="bf16", N=2, H=16, Hk=4, D=128, S=64, L=65500, W=0,
             ragged=False, own_key=True, norm="mass"),
        # A full batch over long caches: the largest stream.
        dict(name="decode_batch", kind="decode", flow="bf16", N=128, H=16, Hk=16, D=64, S=64, L=4096, W=0, ragged=True,
             own_key=True, norm="mass"),
        # Room for one token of each of 64 sequences, and the step taken back.
        dict(name="plan_step", kind="plan", N=64, T=1, S=16, L=1000, W=0, ragged=True),
        # 256 prompts of up to 1024 tokens come (16-token pages, a slot for every token), and end.
        dict(name="plan_prompts", kind="plan", N=256, T=1024, S=16, L=0, W=0, ragged=True),
        # One group of four beams over the reference's default vocabulary.
        dict(name="select_one", kind="select", flow="f32", N=1, B=4, V=2048, K=4, first=False, ended=False),
        # 64 groups of eight beams over the 117M model's vocabulary, twice the beams kept, some beams at their end.
        dict(name="select_batch", kind="select", flow="bf16", N=64, B=8, V=32768, K=16, first=False, ended=True),
        # One group of four beams on the 117M model's twelve layers, bf16 pages.
        dict(name="reorder_one", kind="reorder", pages="bf16", N=1, B=4, layers=12, Hk=12, D=64, S=16, L=509),
        # 32 groups of eight beams, 4-bit pages of 64 tokens.
        dict(name="reorder_batch", kind="reorder", pages="e2m1", N=32, B=8, layers=12, Hk=16, D=64, S=64, L=301),
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


def _row_bytes(D):
    """Codes and exponents of one row."""
    return D // 2 + -(-D // _GROUP)


def work(case):
    kind, N = case["kind"], case["N"]
    if kind == "decode":
        keys = sum(max(0, hi - lo) for lo, hi in (_range(case, n) for n in _spread(N, case["L"], case["ragged"])))
        return {"bytes": 2 * keys * case["Hk"] * _row_bytes(case["D"]) + 2 * N * case["H"] * case["D"] * _BYTES[case["flow"]],
                "flops": 4.0 * keys * case["H"] * case["D"]}
    if kind == "store":
        rows = 2 * case["Hk"] * sum(_counts(case))
        dense = case["D"] * _BYTES[case["flow"]]
        return {"bytes": rows * (dense + 2 * _row_bytes(case["D"])) + 2 * N * case["T"] * case["Hk"] * dense,
                "flops": 6.0 * rows * case["D"]}
    if kind == "plan":  # entries taken and given back (table, free page), counters, slots
        entries = sum(-(-(a + c) // case["S"]) - -(-a // case["S"]) for a, c in zip(_before(case), _counts(case)))
        return {"bytes": 16 * entries + 16 * N + 8 * N * case["T"], "flops": 4.0 * N * case["T"]}
    if kind == "select":
        return {"bytes": N * case["B"] * (case["V"] * _BYTES[case["flow"]] + 5) + 20 * N * case["K"],
                "flops": 4.0 * N * case["B"] * case["V"]}
    S, row = case["S"], case["D"] * 2 if case["pages"] == "bf16" else _row_bytes(case["D"])
    copies = sum(case["B"] - len(set(p)) for p in _parents(case, 0).tolist())  # pages that a second beam goes on from
    return {"bytes": 4 * case["layers"] * case["Hk"] * copies * (case["L"] % S) * row +
            8 * N * case["B"] * -(-case["L"] // S), "flops": 0.0}


def _counts(case):
    return _spread(case["N"], case["T"], case["ragged"] and case["T"] > 1)


def _before(case):
    return _spread(case["N"], case["L"], case["ragged"]) if case["L"] else [0] * case["N"]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = {k: max(work(c)["bytes"] for c in listed() if c["kind"] == k)
             for k in ("store", "decode", "plan", "select", "reorder")}
    while True:
        kind = rng.choices(("store", "decode", "plan", "select", "reorder"), (0.2, 0.35, 0.15, 0.15, 0.15))[0]
        D, S = rng.choice((32, 64, 64, 64, 96, 128)), rng.choice((16, 16, 32, 64, 128))
        heads, share = rng.choice((1, 3, 4, 5, 8, 12, 16)), rng.choice((1, 1, 1, 2, 4, 5))
        flow = rng.choice(("bf16", "bf16", "f16", "f32"))
        if kind == "decode":
            case = dict(kind=kind, flow=flow, N=_log_int(rng, 1, 128), H=heads * share, Hk=heads, D=D, S=S,
                        L=_log_int(rng, 1, 65536), W=rng.choice((0, 0, 0, 8, 64, 100, 256)), ragged=rng.random() < 0.7, own_key=rng.random() < 0.6, norm=rng.choice(("mass", "mass", "count", "raw")))
            if not case["own_key"] and case["L"] < 8:  # sequences of one token would attend to nothing at all
                continue
        elif kind == "store":
            case = dict(kind=kind, flow=flow, N=_log_int(rng, 1, 128), T=rng.choice((1, _log_int(rng, 2, 2048))), Hk=heads,
                        D=D, S=S, L=rng.choice((0, _log_int(rng, 1, 2048))), ragged=rng.random() < 0.6,
                        fused=rng.random() < 0.3, slots=rng.random() < 0.5)
        elif kind == "plan":
            case = dict(kind=kind, N=_log_int(rng, 1, 1024), T=rng.choice((1, 1, _log_int(rng, 2, 4096))), S=S,
                        L=rng.choice((0, _log_int(rng, 1, 8192))), W=rng.choice((0, 0, 64, 256)), ragged=rng.random() < 0.7)
        elif kind == "select":
            B = rng.choice((1, 2, 3, 4, 4, 5, 8, 16))
            V = _log_int(rng, 64, 65536)
            case = dict(kind=kind, flow=flow, N=_log_int(rng, 1, 64), B=B, V=V, K=rng.choice((B, B, min(2 * B, V))),
                        first=rng.random() < 0.2, ended=rng.random() < 0.4)
        else:
            case = dict(kind=kind, pages=rng.choice(("bf16", "e2m1")), N=_log_int(rng, 1, 32), B=rng.choice((2, 3, 4, 5, 8)),
                        layers=rng.choice((1, 4, 12, 24)), Hk=heads, D=D, S=S, L=_log_int(rng, 1, 1024))
        if work(case)["bytes"] <= limit[kind]:
            return case


# ------------------------------------------------------------------ the 4-bit type

def _quantise(x):
    """Codes, two to a byte, and exponent bytes of rows x [..., D], D a multiple of 32."""
    x = x.float().unflatten(-1, (-1, _GROUP))
    top = x.abs().amax(-1).view(torch.int32)
    e = ((top >> 23) - 2 + ((top & 0x7FFFFF) > 0x400000).int()).clamp(min=1)
    y = x * torch.exp2((127 - e).float())[..., None]
    a = y.abs()
    # eight magnitudes 0 0.5 1 1.5 2 3 4 6: steps of a half below 2, of one below 4, of two above; ties to even
    code = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    code = (code + torch.where(torch.signbit(y), 8.0, 0.0)).to(torch.uint8).flatten(-2)
    return code[..., ::2] | code[..., 1::2] << 4, e.to(torch.uint8)


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values(codes, exps):
    """float32 values of code bytes [..., D / 2] with exponent bytes [..., D / 32]."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[both.int()].unflatten(-1, (-1, _GROUP)) * torch.exp2(exps.float() - 127.0)[..., None]
    return x.flatten(-2)


# ------------------------------------------------------------------ inputs

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _pool(g, P, Hk, S, D):
    """Pages that hold tokens everywhere (those no sequence owns are another's)."""
    return _quantise(torch.randn(P, Hk, S, D, generator=g, device="cuda", dtype=torch.bfloat16))


def _parents(case, seed):
    """Which beam each beam of a group goes on from: the better ones more often."""
    N, B = case["N"], case["B"]
    host = torch.Generator().manual_seed(1000 + int(seed))
    return torch.randint(0, B, (N, B, 2), generator=host).amin(-1)


def _table(used, ids, width=None, first=None):
    """Entries [N, width] int32: ``used[n]`` pages of a sequence from entry ``first[n]`` on, -1 elsewhere."""
    slot = torch.arange(width or int(used.max()))[None, :] - (0 if first is None else first[:, None])
    at = (torch.cumsum(used, 0) - used)[:, None] + slot
    inside = (slot >= 0) & (slot < used[:, None])
    return torch.where(inside, ids[at.clamp(0, len(ids) - 1)], torch.tensor(-1, dtype=torch.int32))


def prepare(case, seed):
    made = {"store": _prepare_store, "decode": _prepare_decode, "plan": _prepare_plan, "select": _prepare_select,
            "reorder": _prepare_reorder}[case["kind"]]
    return made(case, torch.Generator(device="cuda").manual_seed(int(seed)), torch.Generator().manual_seed(int(seed)), seed)


def _prepare_decode(case, g, host, seed):
    N, S = case["N"], case["S"]
    lengths = torch.tensor(_spread(N, case["L"], case["ragged"]))[torch.randperm(N, generator=host)]
    used = (lengths + S - 1) // S
    P = int(used.sum()) + 1
    table = _table(used, torch.randperm(P, generator=host).to(torch.int32))
    return {"case": case, "table": table.cuda(), "lengths": lengths.to(torch.int32).cuda(),
            "k": _pool(g, P, case["Hk"], S, case["D"]), "v": _pool(g, P, case["Hk"], S, case["D"]),
            "q": _randn(g, N, case["H"], case["D"], dtype=_DT[case["flow"]])}


def _prepare_store(case, g, host, seed):
    N, T, Hk, D, S = (case[n] for n in ("N", "T", "Hk", "D", "S"))
    order = torch.randperm(N, generator=host)
    counts, start = torch.tensor(_counts(case))[order], torch.tensor(_before(case))[order]
    used = (start + counts + S - 1) // S
    P = int(used.sum()) + 1
    table = _table(used, torch.randperm(P, generator=host).to(torch.int32))
    dt = _DT[case["flow"]]
    if case["fused"]:
        k_new, v_new = _randn(g, N, T, Hk, 2 * D, dtype=dt).split(D, dim=-1)
    else:
        k_new, v_new = _randn(g, N, T, Hk, D, dtype=dt), _randn(g, N, T, Hk, D, dtype=dt)
    # every 32 values their own size, as channels of a projection have
    size = torch.exp2(torch.randint(-3, 4, (N, T, Hk, D // _GROUP), generator=g, device="cuda").float())
    size = size.to(dt).repeat_interleave(_GROUP, -1)
    k_new.mul_(size)
    v_new.mul_(size)
    pos = start[:, None] + torch.arange(T)
    slots = table.long().gather(1, (pos // S).clamp(max=table.shape[1] - 1)) * S + pos % S
    slots = torch.where(torch.arange(T) < counts[:, None], slots, -1)
    return {"case": case, "table": table.cuda(), "start": start.to(torch.int32).cuda(),
            "counts": counts.to(torch.int32).cuda(), "slots": slots.cuda(), "k": _pool(g, P, Hk, S, D),
            "v": _pool(g, P, Hk, S, D), "k_new": k_new, "v_new": v_new}


def _prepare_plan(case, g, host, seed):
    N, T, S, W = (case[n] for n in ("N", "T", "S", "W"))
    order = torch.randperm(N, generator=host)
    counts, before = torch.tensor(_counts(case))[order], torch.tensor(_before(case))[order]
    first = (before - W).clamp(min=0) // S if W else torch.zeros_like(before)
    used = (before + S - 1) // S - first
    end = (before + counts + S - 1) // S
    P = int(used.sum() + (end - first).sum()) + 8
    ids = torch.randperm(P, generator=host).to(torch.int32)
    held = int(used.sum())
    free = torch.full((P,), -1, dtype=torch.int32)
    free[:P - held] = ids[held:]
    return {"case": case, "table": _table(used, ids, int(end.max()) + 1, first).cuda(), "free": free.cuda(),
            "top": torch.tensor([P - held], dtype=torch.int32).cuda(), "lengths": before.to(torch.int32).cuda(),
            "counts": counts.to(torch.int32).cuda(), "after": (before + counts).to(torch.int32).cuda(),
            "back": -counts.to(torch.int32).cuda()}


def _prepare_select(case, g, host, seed):
    N, B, V = case["N"], case["B"], case["V"]
    # a language model's logits: a few likely tokens above many unlikely ones
    logits = _randn(g, N, B, V) * 2.0 + 6.0 * (torch.rand(N, B, V, generator=g, device="cuda") < 8.0 / V)
    scores = -_randn(g, N, B).abs() * 3 - 20.0
    if case["first"]:  # a group starts from one beam
        scores[:, 1:] = -math.inf
    ended = torch.rand(N, B, generator=g, device="cuda") < 0.3 if case["ended"] else None
    return {"case": case, "logits": logits.to(_DT[case["flow"]]), "scores": scores, "ended": ended}


def _prepare_reorder(case, g, host, seed):
    N, B, S, layers, Hk, D, L = (case[n] for n in ("N", "B", "S", "layers", "Hk", "D", "L"))
    full, width = L // S, L // S + 2
    # full pages are a group's, the page being filled is a beam's own
    P = N * (full + B)
    ids = torch.randperm(P, generator=host).to(torch.int32).view(N, full + B)
    table = torch.full((N, B, width), -1, dtype=torch.int32)
    table[:, :, :full] = ids[:, None, :full]
    table[:, :, full] = ids[:, full:]
    if case["pages"] == "bf16":
        k = torch.randn(layers, P, Hk, S, D, generator=g, device="cuda", dtype=torch.bfloat16)
        v = torch.randn(layers, P, Hk, S, D, generator=g, device="cuda", dtype=torch.bfloat16)
        tensors = [k, v]
    else:
        (k, ke), (v, ve) = _pool(g, layers * P, Hk, S, D), _pool(g, layers * P, Hk, S, D)
        tensors = [x.unflatten(0, (layers, P)) for x in (k, v, ke, ve)]
    return {"case": case, "table": table.view(N * B, width).cuda(), "parents": _parents(case, seed).cuda(),
            "lengths": torch.full((N,), L, dtype=torch.int32).cuda(), "tensors": tensors}


# ------------------------------------------------------------------ the plain forms

def _places(table, pos, S):
    """Page and row of positions pos [N, n] (clamped into the table)."""
    p = pos.clamp(min=0, max=table.shape[1] * S - 1).long()
    return table.long().gather(1, p // S).clamp(min=0), p % S


def _plain_store(pages, new, table, start, counts):
    codes, exps = pages
    pos = start[:, None] + torch.arange(new.shape[1], device=new.device)
    live = torch.arange(new.shape[1], device=new.device) < counts[:, None]
    page, row = _places(table, pos, codes.shape[2])
    page, row = page[live], row[live]
    codes[page, :, row], exps[page, :, row] = _quantise(new[live])


def _plain_store_slots(pages, new, slots):
    codes, exps = pages
    live = slots >= 0
    page, row = slots[live] // codes.shape[2], slots[live] % codes.shape[2]
    codes[page, :, row], exps[page, :, row] = _quantise(new[live])


def _plain_read(pages, table, start, T, counts, dtype):
    codes, exps = pages
    pos = start[:, None] + torch.arange(T, device=table.device)
    live = torch.arange(T, device=table.device) < counts[:, None]
    page, row = _places(table, pos, codes.shape[2])
    x = _values(codes[page, :, row], exps[page, :, row])
    return torch.where(live[..., None, None], x, x.new_zeros(())).to(dtype)


def _plain_decode(s, scale):
    case, q, table, lengths = s["case"], s["q"], s["table"], s["lengths"]
    N, H, D = q.shape
    Hk, W, L = case["Hk"], case["W"], case["L"]
    hi = lengths - (0 if case["own_key"] else 1)
    lo = (lengths - 1 - W).clamp(min=0) if W else torch.zeros_like(lengths)
    pos = lo[:, None] + torch.arange(min(L, W + 1) if W else L, device=q.device)
    live = pos < hi[:, None]
    page, row = _places(table, pos, case["S"])

    def rows(pages):  # [N, Hk, n, D] in 32 bits
        return _values(pages[0][page, :, row], pages[1][page, :, row]).transpose(1, 2)

    x = torch.matmul(rows(s["k"]), q.float().view(N, Hk, H // Hk, D).transpose(2, 3).contiguous()) / scale  # [N, Hk, n, G]
    tau = torch.where(live[:, None, :, None], 1.0 / (1.0 + torch.exp(-x)), x.new_zeros(()))
    out = torch.matmul(tau.transpose(2, 3), rows(s["v"]))  # [N, Hk, G, D]
    if case["norm"] == "mass":
        out = out / tau.sum(2).clamp(min=1e-6)[..., None]
    elif case["norm"] == "count":
        out = out / (hi - lo).clamp(min=1).float()[:, None, None, None]
    return out.reshape(N, H, D).to(q.dtype)


def _plain_plan(free, top, table, lengths, counts, S, W, T):
    """Pages past the new length (or that no later token reads) pushed on the stack ``free`` of ``top`` pages, pages for
    the new tokens popped, in the order of the sequences and of their entries; then the tokens' slots."""
    P, width = len(free), table.shape[1]
    e = torch.arange(width, device=table.device)
    length = lengths[:, None].clamp(0, width * S)
    end = (length + counts[:, None]).clamp(0, width * S)
    hi, has = (end + S - 1) // S, (table >= 0) & (table < P)
    before = (torch.minimum(length, end) - W).clamp(min=0) // S if W else torch.zeros_like(length)
    first = (end - W).clamp(min=0) // S if W else torch.zeros_like(length)
    run = torch.where(e < before, has, True).flip(1).cumprod(1).flip(1).bool()  # no hole from here to the window
    give = has & ((e >= hi) & (e < (length + S - 1) // S) | (e < before) & run)
    take = ~has & (e >= torch.maximum(first, length // S)) & (e < hi) & (end > length)
    given, taken = give.sum(), take.sum()
    room = top + given
    fits = taken <= room
    back = (room - 1).long() - (torch.cumsum(give.flatten(), 0) - 1)  # the first given lies on top
    old = table.clone()
    into = torch.where(give.flatten() & fits, back, P)
    free.copy_(torch.cat((free, free.new_zeros(1))).scatter(0, into, old.flatten())[:P])
    at = (room - 1).long() - (torch.cumsum(take.flatten(), 0) - 1)
    new = torch.where(take, free[at.clamp(0, P - 1)].view_as(table), torch.where(give, -1, table))
    table.copy_(torch.where(fits, new, table))
    top.copy_(torch.where(fits, room - taken, top))
    t = torch.arange(T, device=table.device)
    pos = lengths[:, None].long() + t
    inside = (t < counts[:, None]) & (pos >= 0) & (pos < width * S)
    page = table.long().gather(1, (pos // S).clamp(0, width - 1))
    slots = torch.where(inside & (page >= 0) & (page < P), page * S + pos % S, -1)
    return slots, torch.where(fits, 0, taken - room).to(torch.int32).view(1)


def _plain_select(logits, scores, ended, K):
    N, B, V = logits.shape
    x = logits.double()
    m = x.amax(-1, keepdim=True)
    c = scores.double()[..., None] + (x - m - torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    if ended is not None:  # a beam at its end goes on as it is, with token 0
        alone = torch.full_like(c, -math.inf)
        alone[..., 0] = scores.double()
        c = torch.where(ended[..., None], alone, c)
    best, at = torch.sort(c.view(N, B * V), dim=-1, descending=True, stable=True)
    return best[:, :K].float(), at[:, :K] % V, at[:, :K] // V


def _plain_reorder(s):
    case, table, parents, lengths = s["case"], s["table"], s["parents"], s["lengths"]
    N, B, S = case["N"], case["B"], case["S"]
    old = table.view(N, B, -1)
    i = torch.arange(B, device=table.device)
    same = parents[:, :, None] == parents[:, None, :]
    second = (same & (i[None, :] < i[:, None])).any(-1)            # an earlier beam goes on from the same one
    dead = ~(parents[:, :, None] == i).any(1)                      # nobody goes on from it
    spare = torch.argsort((~dead).int(), dim=-1, stable=True)      # the dead, in order
    own_page = torch.where(second, spare.gather(1, (torch.cumsum(second.int(), 1) - 1).clamp(min=0)), parents)
    full = (lengths // S)[:, None, None]
    wide = lambda x: x[..., None].expand_as(old)  # noqa: E731
    e = torch.arange(old.shape[2], device=table.device)
    new = torch.where(e < full, old.gather(1, wide(parents)), old.gather(1, wide(own_page)))
    at = full.clamp(max=old.shape[2] - 1).long().expand(N, B, 1)
    src, dst = old.gather(1, wide(parents)).gather(2, at)[..., 0], new.gather(2, at)[..., 0]
    src, dst = src[second].long(), dst[second].long()
    rows = case["L"] % S
    for t in s["tensors"]:  # [layers, P, Hk, S, row]
        t[:, dst, :, :rows] = t[:, src, :, :rows]
    return new.view(N * B, -1)


# ------------------------------------------------------------------ one pass

def run(s):
    return {"store": _run_store, "decode": _run_decode, "plan": _run_plan, "select": _run_select,
            "reorder": _run_reorder}[s["case"]["kind"]](s)


def _kv(s):
    import bozo_amd
    f4 = torch.float4_e2m1fn_x2
    return bozo_amd.PagedKV(s["k"][0].view(f4), s["v"][0].view(f4), s["k"][1], s["v"][1])


def _run_decode(s):
    case, scale = s["case"], math.sqrt(s["case"]["D"])
    if own:
        import bozo_amd
        return bozo_amd.paged_decode(s["q"], _kv(s), s["table"], s["lengths"], scale, window=case["W"] or None,
                                     include_self=case["own_key"], normalize=case["norm"], max_len=case["L"])
    return _plain_decode(s, scale)


def _run_store(s):
    case, table, start, counts = s["case"], s["table"], s["start"], s["counts"]
    T, dt = case["T"], _DT[case["flow"]]
    if own:
        import bozo_amd
        kv = _kv(s)
        if case["slots"]:
            bozo_amd.paged_store(kv, s["k_new"], s["v_new"], s["slots"])
        else:
            bozo_amd.paged_append(kv, s["k_new"], s["v_new"], table, start, counts)
        return bozo_amd.paged_read(kv, table, start, T, dt, counts)
    if case["slots"]:
        _plain_store_slots(s["k"], s["k_new"], s["slots"])
        _plain_store_slots(s["v"], s["v_new"], s["slots"])
    else:
        _plain_store(s["k"], s["k_new"], table, start, counts)
        _plain_store(s["v"], s["v_new"], table, start, counts)
    return _plain_read(s["k"], table, start, T, counts, dt), _plain_read(s["v"], table, start, T, counts, dt)


def _run_plan(s):
    case, table, lengths, counts = s["case"], s["table"], s["lengths"], s["counts"]
    S, W, T = case["S"], case["W"], case["T"]
    if own:
        import bozo_amd
        pool = bozo_amd.PagePool(s["free"], s["top"])
        slots, missing = bozo_amd.paged_plan(pool, table, lengths, counts, S, T, window=W or None)
        _, none = bozo_amd.paged_plan(pool, table, s["after"], s["back"], S, 0, window=W or None)
    else:
        slots, missing = _plain_plan(s["free"], s["top"], table, lengths, counts, S, W, T)
        _, none = _plain_plan(s["free"], s["top"], table, s["after"], s["back"], S, W, 0)
    return slots, missing, none, table, s["free"], s["top"]


def _run_select(s):
    if own:
        import bozo_amd
        return bozo_amd.beam_select(s["logits"], s["scores"], s["case"]["K"], ended=s["ended"], pad=0)
    return _plain_select(s["logits"], s["scores"], s["ended"], s["case"]["K"])


def _run_reorder(s):
    if own:
        import bozo_amd
        tensors = s["tensors"]
        if s["case"]["pages"] == "e2m1":
            tensors = [t.view(torch.float4_e2m1fn_x2) for t in tensors[:2]] + tensors[2:]
        layers = [bozo_amd.PagedKV(*(t[i] for t in tensors)) for i in range(s["case"]["layers"])]
        table = bozo_amd.paged_reorder(layers, s["table"], s["lengths"], s["parents"])
    else:
        table = _plain_reorder(s)
    return (table, *s["tensors"])


# ------------------------------------------------------------------ the definition in 64 bits

def _rounded64(x):
    """float64 rows as the 4-bit cache holds them: the nearest of the sixteen values of each 32's scale, the even code
    of two as near."""
    x = x.unflatten(-1, (-1, _GROUP))
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 6 = 0.75 * 2^3
    e = torch.where(top > 0, torch.where(m <= 0.75, e - 3, e - 2), torch.full_like(e, -126)).clamp(min=-126).double()
    y = x * torch.exp2(-e)
    held = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    off = (y.abs()[..., None] - held).abs()
    off[..., 1::2] += 2.0 ** -40  # no input lies that near to a tie without being one: an odd code loses it
    return (held[off.argmin(-1)] * torch.sign(y) * torch.exp2(e)).flatten(-2)


def _held64(codes, exps):
    """float64 values of rows as pages hold them: sign, two exponent bits, one bit after the point."""
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.int16, device=codes.device)
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    e, m = (c % 8 // 2).double(), (c % 2).double()
    x = torch.where(e > 0, (1 + m / 2) * torch.exp2(e - 1), m / 2) * torch.where(c >= 8, -1.0, 1.0)
    return x * torch.exp2(exps.double() - 127).repeat_interleave(_GROUP, -1)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("plan", "reorder"):  # whole numbers, and bytes that are copied
        return None
    s = prepare(case, seed)
    if kind == "select":
        N, B, V, K = (case[n] for n in ("N", "B", "V", "K"))
        x, scores = s["logits"].double(), s["scores"].double()
        c = scores[..., None] + x - torch.logsumexp(x, -1, keepdim=True)
        if s["ended"] is not None:
            c[s["ended"]] = -math.inf
            c[..., 0] = torch.where(s["ended"], scores, c[..., 0])
        return torch.topk(c.view(N, B * V), K).values, None, None
    N, D, S = case["N"], case["D"], case["S"]
    if kind == "store":
        counts, res = s["counts"].cpu().tolist(), []
        for new in (s["k_new"], s["v_new"]):
            out = torch.zeros(new.shape, dtype=torch.float64, device=new.device)
            for n in range(N):
                out[n, :counts[n]] = _rounded64(new[n, :counts[n]].double())
            res.append(out)
        return tuple(res)
    table, lengths = s["table"].cpu().tolist(), s["lengths"].cpu().tolist()

    def tokens(pages, n, lo, hi):
        """[Hk, hi - lo, D] in 64 bits: the tokens lo .. hi - 1 of sequence n."""
        ids = torch.tensor(table[n][lo // S:(hi + S - 1) // S], device="cuda")
        x = _held64(pages[0][ids], pages[1][ids])
        return x.transpose(1, 2).flatten(0, 1)[lo % S:lo % S + hi - lo].transpose(0, 1)

    out = torch.zeros(N, case["H"], D, dtype=torch.float64, device="cuda")
    for n in range(N):
        lo, hi = _range(case, lengths[n])
        if hi <= lo:
            continue
        G = case["H"] // case["Hk"]
        K, V = tokens(s["k"], n, lo, hi), tokens(s["v"], n, lo, hi)
        tau = torch.sigmoid((s["q"][n].double().view(-1, G, 1, D) * K[:, None]).sum(-1) / math.sqrt(D))  # [Hk, G, n]
        o = (tau[..., None] * V[:, None]).sum(2)
        if case["norm"] == "mass":
            o = o / tau.sum(-1, keepdim=True).clamp(min=1e-6)
        elif case["norm"] == "count":
            o = o / (hi - lo)
        out[n] = o.reshape(-1, D)
    return out
