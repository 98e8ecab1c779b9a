"""The operators of serving from an 8-bit cache with drafted tokens, as cases that can be timed and checked.

    store    rotary, quantisation and the write of a step's keys and values into 8-bit pages, and the
             written pages read back
    read     pages of whole sequences read back into the activations' type
    attend   attention of a step's tokens over 8-bit pages: one token a sequence, a few drafted ones,
             or a prompt's portion
    verify   drafted tokens held against the target's probabilities, from given random numbers

An 8-bit vector is ``head_dim`` codes (e4m3 or int8) and one float32 scale: with ``a`` the largest
magnitude (2^-100 at least), scale = a / L and code = round(x * (L / a)), L = 448 or 127.  A vector
that holds an infinity or a NaN is codes of zero and a scale of NaN.

``run`` computes the operators either in elementary torch operations, in 32 bits and the random
draws' sums in 64, or (``own``) by the framework's kernels.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 64
LIMIT = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DEVICE = "cuda"


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def _store(fmt, dtype, heads, kv, dim, batch, new, past, splits=0, window=0, rotary=0, style=0):
    return {"op": "store", "fmt": fmt, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "batch": batch,
            "new_low": new[0], "new_high": new[1], "past_low": past[0], "past_high": past[1],
            "splits": splits, "window": window, "rotary": rotary or dim, "style": style}


def _read(fmt, dtype, kv, dim, batch, length):
    return {"op": "read", "fmt": fmt, "dtype": dtype, "kv": kv, "dim": dim, "batch": batch,
            "low": length[0], "high": length[1]}


def _attend(fmt, dtype, heads, kv, dim, batch, new, past, window=0):
    return {"op": "attend", "fmt": fmt, "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "batch": batch,
            "new_low": new[0], "new_high": new[1], "past_low": past[0], "past_high": past[1], "window": window}


def _verify(vocab, batch, drafts, temperature, draft_logits):
    return {"op": "verify", "vocab": vocab, "batch": batch, "low": drafts[0], "high": drafts[1],
            "temperature": temperature, "draft_logits": draft_logits}


def listed():
    named = {
        # a decoding step of the 7B shape at batch 8 writes its tokens: latency is all
        "store-one-8": _store("e4m3", "bfloat16", 28, 4, 128, 8, (1, 1), (1900, 2047), splits=4),
        # three unequal prompts of the 0.5B shape come in whole
        "store-prompts": _store("int8", "bfloat16", 14, 2, 64, 3, (517, 2801), (0, 0)),
        # a long document's cached prefix for the next portion's attention (7B shape)
        "read-long": _read("e4m3", "bfloat16", 4, 128, 4, (15001, 31999)),
        # the 32-bit engine looks at what it has cached
        "read-32bit": _read("int8", "float32", 2, 64, 5, (1, 700)),
        # the headline: eight sequences of the 7B shape at about 2,000 tokens, one token each
        "one-8": _attend("e4m3", "bfloat16", 28, 4, 128, 8, (1, 1), (1801, 2047)),
        # a small model serves many unequal requests
        "one-64-ragged": _attend("int8", "bfloat16", 14, 2, 64, 64, (1, 1), (0, 4095)),
        # a full batch of the 7B shape at 2,000 to 8,000 tokens: the cache's bandwidth
        "one-64-long": _attend("e4m3", "bfloat16", 28, 4, 128, 64, (1, 1), (2047, 8100)),
        # sixteen sequences, each with its last token and four drafted ones
        "drafts-16": _attend("e4m3", "bfloat16", 28, 4, 128, 16, (5, 5), (1501, 3001)),
        # a prompt's portion of 512 tokens after 8,000 cached ones (14B shape)
        "portion-512": _attend("int8", "bfloat16", 40, 8, 128, 1, (512, 512), (8001, 8001)),
        # the 32-bit engine, used to check a model: short and ragged
        "few-32bit": _attend("e4m3", "float32", 14, 2, 64, 4, (1, 3), (60, 611)),
        # one user, a draft model ahead by four tokens
        "verify-1": _verify(151936, 1, (4, 4), 0.8, True),
        # a full batch with drafts looked up in the prompts: no probabilities, ragged
        "verify-64-lookup": _verify(152064, 64, (0, 7), 1.0, False),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


_SHAPES = [(28, 4, 128), (14, 2, 64), (40, 8, 128), (16, 4, 128), (16, 16, 64), (6, 1, 128), (12, 4, 96), (4, 1, 32)]
_MOST = {"store": 4e8, "read": 2e9, "attend": 1.5e9, "verify": 3.5e8}


def draw(rng):
    """Any of the four, over the listed ranges: batches of 1 to 64, contexts of 0 to 32,000, portions
    of up to 512 tokens, vocabularies of 1,000 to 152,064."""
    while True:
        op = rng.choice(["store", "read", "attend", "attend", "attend", "verify"])
        fmt = rng.choice(["e4m3", "int8"])
        dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
        heads, kv, dim = rng.choice(_SHAPES)
        batch = _log_uniform(rng, 1, 64)
        if op == "store":
            if rng.random() < 0.5:
                high = _log_uniform(rng, 1, 16)
                past = _log_uniform(rng, 1, 8000)
            else:
                high, past = _log_uniform(rng, 17, 4000), rng.choice([0, _log_uniform(rng, 1, 2000)])
            low = max(1, int(high * rng.choice([1.0, 0.5, 0.1])))
            window = rng.choice([0, 0, _log_uniform(rng, 16, 1000)])
            rotary, style = rng.choice([(dim, 0), (dim, 0), (dim // 2, 0), (dim, 1)])
            # (in float32 a code that a last bit's difference turns is more than the type's precision)
            case = _store(fmt, "bfloat16", heads, kv, dim, batch, (low, high), (past // 2, past), rng.choice([0, 2, 5]),
                          window, rotary, style)
        elif op == "read":
            high = _log_uniform(rng, 1, 32000)
            case = _read(fmt, dtype, kv, dim, batch, (max(1, int(high * rng.choice([1.0, 0.3, 0.0]))), high))
        elif op == "attend":
            high = rng.choice([1, 1, rng.randint(2, 9), _log_uniform(rng, 10, 512)])
            low = max(1, int(high * rng.choice([1.0, 0.5])))
            past = _log_uniform(rng, 1, 32000 if dtype == "bfloat16" else 2000)
            window = rng.choice([0, 0, 0, _log_uniform(rng, 16, 4000)])
            case = _attend(fmt, dtype, heads, kv, dim, batch, (low, high),
                           (int(past * rng.choice([1.0, 0.5, 0.0])), past), window)
        else:
            high = rng.randint(1, 8)
            case = _verify(rng.choice([152064, 151936, 32000, _log_uniform(rng, 1000, 150000)]), batch,
                           (rng.randint(0, high), high), rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]), rng.random() < 0.6)
        # 32-bit products run on the FP32 pipe: a tenth of the work costs as much
        if _cost(case) <= _MOST[op] * (0.1 if op == "attend" and dtype == "float32" else 1.0):
            return case


def _spread(low, high, n):
    """``n`` lengths from ``low`` to ``high``, the longest first."""
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, cached positions before them) of every sequence."""
    new = _spread(case["new_low"], case["new_high"], case["batch"])
    past = _spread(case["past_low"], case["past_high"], case["batch"])[::-1]
    return new, past


def _seen(window, new, past):
    """Keys that some of a sequence's ``new`` queries see."""
    return min(past + new, window + new - 1) if window else past + new


def work(case):
    op = case["op"]
    if op == "verify":
        n = sum(_spread(case["low"], case["high"], case["batch"]))
        rows = n + case["batch"] + (n if case["draft_logits"] else 0)
        return {"bytes": 4.0 * rows * case["vocab"], "flops": 4.0 * rows * case["vocab"]}
    size = 2 if case["dtype"] == "bfloat16" else 4
    kv, dim = case["kv"], case["dim"]
    vector = dim + 4                                       # codes and a scale
    if op == "read":
        n = sum(_spread(case["low"], case["high"], case["batch"]))
        return {"bytes": 2.0 * kv * n * (vector + dim * size), "flops": 2.0 * kv * n * dim}
    new, past = _lengths(case)
    tokens = sum(new)
    if op == "store":
        width = (case["heads"] + 2 * kv) * dim
        ring = _ring(case)                                     # the written pages' positions
        back = sum(min(n + p, ring) if ring else n + p - p // PAGE * PAGE for n, p in zip(new, past))
        return {"bytes": tokens * width * (4.0 * max(1, case["splits"]) + size) + 2.0 * tokens * kv * vector
                + 2.0 * back * kv * (vector + dim * size), "flops": 6.0 * tokens * width}
    w = case["window"]
    keys = sum(_seen(w, n, p) for n, p in zip(new, past))
    pairs = 0
    for n, p in zip(new, past):
        if w:
            pairs += sum(min(p + i + 1, w) for i in range(n))
        else:
            pairs += n * p + n * (n + 1) // 2
    return {"bytes": 2.0 * kv * keys * vector + 2.0 * tokens * case["heads"] * dim * size,
            "flops": 4.0 * pairs * case["heads"] * dim}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _torch_type(case):
    return torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32


def _quantise(x, fmt):
    """Codes and scales of vectors along the last dimension."""
    limit = LIMIT[fmt]
    a = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    a = torch.where(bad, torch.ones_like(a), a).clamp_min(2.0 ** -100)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x) * (limit / a).unsqueeze(-1)
    code = code.clamp(-limit, limit)
    code = code.to(torch.float8_e4m3fn) if fmt == "e4m3" else code.round().to(torch.int8)
    return code, torch.where(bad, torch.full_like(a, float("nan")), a / limit)


def _pool(case, n_pages, gen):
    """A cache that has been in use: every page holds vectors of somebody."""
    shape = (n_pages, case["kv"], PAGE, case["dim"])
    offset = torch.randn(case["kv"], 1, case["dim"], generator=gen, device=DEVICE)
    k, ks = _quantise(torch.randn(shape, generator=gen, device=DEVICE) + 0.7 * offset, case["fmt"])
    v, vs = _quantise(torch.randn(shape, generator=gen, device=DEVICE) * 0.6, case["fmt"])
    return k, v, ks, vs


def _ring(case):
    """Positions a ring keeps: the window and what a step may add (0: linear)."""
    w = case.get("window", 0)
    return 0 if not w else -(-(w + case["new_high"] - 1) // PAGE) * PAGE


def _pages(ends, ring):
    return [-(-(min(e, ring) if ring else e) // PAGE) for e in ends]


def _table(ends, ring, gen, spare=3):
    """(page table [rows, width], pages in the pool): pages in any order, -1 where a row has none."""
    need = _pages(ends, ring)
    width = max(1, max(need))
    total = sum(need) + spare
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32).cpu()
    table = torch.full((len(ends), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(DEVICE), total


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    op = case["op"]
    s = {"case": case, "op": op}
    if op == "verify":
        _prepare_verify(case, gen, s)
        return s
    s["status"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    if op == "read":
        ends = _spread(case["low"], case["high"], case["batch"])
        s["table"], n_pages = _table(ends, 0, gen)
        s["pages"] = _pool(case, n_pages, gen)
        s["end"], s["ring"] = _ints(ends), 0
        return s
    new, past = _lengths(case)
    ends = [n + p for n, p in zip(new, past)]
    ring = _ring(case)
    s["ring"], s["end"] = ring, _ints(ends)
    s["cu"] = _ints([0] + np.cumsum(new).tolist())
    s["longest"], s["max_end"] = max(new), max(ends)
    s["positions"] = _ints([p + i for n, p in zip(new, past) for i in range(n)])
    s["token_row"] = _ints([b for b, n in enumerate(new) for _ in range(n)])
    s["table"], n_pages = _table(ends, ring, gen)
    s["pages"] = _pool(case, n_pages, gen)
    tokens, heads, kv, dim = sum(new), case["heads"], case["kv"], case["dim"]
    if op == "attend":
        q = torch.randn(tokens, heads, dim, generator=gen, device=DEVICE) * 1.5
        s["q"] = q.to(_torch_type(case))
        s["scale"] = dim ** -0.5
        return s
    # store: what the projection of q, k and v left, in K splits where a step has few tokens
    width = (heads + 2 * kv) * dim
    n = case["splits"]
    x = torch.randn((n, tokens, width) if n else (tokens, width), generator=gen, device=DEVICE)
    s["qkv"] = x * (1.0 / math.sqrt(max(1, n)))
    s["bias"] = torch.randn(width, generator=gen, device=DEVICE) * 0.5 if n else None
    half = torch.arange(case["rotary"] // 2, dtype=torch.float64)
    s["inv_freq"] = (1e6 ** (-2.0 * half / case["rotary"])).to(DEVICE)
    # the pages that the step writes, for reading them back: all of a ring's, else from the first
    # written one on
    first = [0 if ring else p // PAGE for p in past]
    need = _pages(ends, ring)
    wide = max(1, max(e - f for e, f in zip(need, first)))
    back = torch.full((len(new), wide), -1, dtype=torch.int32)
    table = s["table"].cpu()
    for b, (f, e) in enumerate(zip(first, need)):
        back[b, :e - f] = table[b, f:e]
    s["back"] = back.to(DEVICE)
    s["back_end"] = _ints([e - f * PAGE for e, f in zip(ends, first)])
    return s


def _prepare_verify(case, gen, s):
    vocab = case["vocab"]
    counts = _spread(case["low"], case["high"], case["batch"])
    n, rows = sum(counts), case["batch"]
    s["cu"] = _ints([0] + np.cumsum(counts).tolist())
    s["counts"] = counts
    # a language model's logits: a wide body and a few tokens far above it
    logits = torch.randn(n + rows, vocab, generator=gen, device=DEVICE) * 2.0
    peaks = torch.randint(0, vocab, (n + rows, 24), generator=gen, device=DEVICE)
    logits.scatter_(1, peaks, 8.0 + 3.0 * torch.randn(n + rows, 24, generator=gen, device=DEVICE))
    s["logits"] = logits
    place = _places(counts)
    target = logits[torch.tensor(place["draft"], dtype=torch.long, device=DEVICE)]
    draft = target + 0.8 * torch.randn(n, vocab, generator=gen, device=DEVICE)
    t = case["temperature"]
    if n == 0:
        s["drafts"] = torch.zeros(0, dtype=torch.int32, device=DEVICE)
    elif t < 1e-6:
        s["drafts"] = draft.argmax(-1).to(torch.int32)
    else:
        noise = torch.rand(n, vocab, generator=gen, device=DEVICE).clamp_min(1e-9).log().neg().log().neg()
        s["drafts"] = (draft / t + noise).argmax(-1).to(torch.int32)
    s["draft_logits"] = draft if case["draft_logits"] else None
    s["accept_u"] = torch.rand(n, generator=gen, device=DEVICE)
    s["draw_u"] = torch.rand(rows, generator=gen, device=DEVICE)


def _places(counts):
    """Rows of the logits: each sequence has a place for every draft and one more."""
    draft, first, at = [], [], 0
    for n in counts:
        first.append(at)
        draft.extend(range(at, at + n))
        at += n + 1
    return {"draft": draft, "first": first}


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"store": _own_store, "read": _own_read, "attend": _own_attend, "verify": _own_verify}[state["op"]](state)
    return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend, "verify": _plain_verify}[state["op"]](state)


def _own_store(s):
    from minfer_b200.kernels import api as K
    c, table = s["case"], s["table"]
    tokens, dt = s["positions"].shape[0], _torch_type(c)
    q = torch.empty((tokens, c["heads"], c["dim"]), dtype=dt, device=DEVICE)
    k = torch.empty((tokens, c["kv"], c["dim"]), dtype=dt, device=DEVICE)
    v = torch.empty_like(k)
    pages = K.Q8Pages(*s["pages"])
    K.rope_kvstore_q8(s["qkv"], s["positions"], s["token_row"], s["end"], s["inv_freq"], q, k, v, pages, table,
                      table.shape[1], s["ring"], c["heads"], c["kv"], c["dim"], c["rotary"], c["style"], s["status"],
                      n_partials=c["splits"], bias=s["bias"])
    back = s["back"]
    k_back = torch.empty((back.numel(), c["kv"], PAGE, c["dim"]), dtype=dt, device=DEVICE)
    v_back = torch.empty_like(k_back)
    K.read_pages_q8(pages, back, back.shape[1], s["ring"], s["back_end"], k_back, v_back, s["status"])
    return q, k, v, k_back, v_back


def _own_read(s):
    from minfer_b200.kernels import api as K
    c, table = s["case"], s["table"]
    k = torch.empty((table.numel(), c["kv"], PAGE, c["dim"]), dtype=_torch_type(c), device=DEVICE)
    v = torch.empty_like(k)
    K.read_pages_q8(K.Q8Pages(*s["pages"]), table, table.shape[1], 0, s["end"], k, v, s["status"])
    return k, v


def _own_attend(s):
    from minfer_b200.kernels import api as K
    c, table = s["case"], s["table"]
    out = torch.empty_like(s["q"])
    K.attention_paged_q8(s["q"], K.Q8Pages(*s["pages"]), s["cu"], s["end"], table, table.shape[1], s["ring"], out,
                         s["longest"], s["max_end"], c["heads"], c["kv"], c["dim"], c["window"], s["scale"], s["status"])
    return out


def _own_verify(s):
    from minfer_b200.kernels import api as K
    rows = s["draw_u"].shape[0]
    accepted = torch.empty(rows, dtype=torch.int32, device=DEVICE)
    tokens = torch.empty(rows, dtype=torch.int32, device=DEVICE)
    K.verify_drafts(s["logits"], s["drafts"], s["cu"], s["draft_logits"], s["accept_u"], s["draw_u"],
                    s["case"]["temperature"], accepted, tokens)
    return accepted, tokens


# ---- the plain forms -----------------------------------------------------------------------------
def _held(end, width, ring):
    """The position that every place of a row's pages holds ([rows, width * 64]; -1: none)."""
    place = torch.arange(width * PAGE, device=DEVICE).unsqueeze(0)
    last = (end.long() - 1).unsqueeze(1)
    if ring:
        pos = last - torch.remainder(last - place, ring)
        return torch.where((place < ring) & (last >= 0), pos, -1)
    return torch.where(place <= last, place, -1)


def _values(codes, scales, table, held):
    """float32 vectors of a table's pages, zeros where a place holds no position."""
    index = table.clamp_min(0).long().reshape(-1)
    x = codes[index].float() * scales[index].unsqueeze(-1)
    there = held.reshape(table.numel(), 1, PAGE, 1) >= 0
    return torch.where(there, x, torch.zeros_like(x))


def _plain_read(s):
    dt = _torch_type(s["case"])
    held = _held(s["end"], s["table"].shape[1], 0)
    k, v, ks, vs = s["pages"]
    return _values(k, ks, s["table"], held).to(dt), _values(v, vs, s["table"], held).to(dt)


def _plain_store(s):
    c = s["case"]
    heads, kv, dim, r, ring = c["heads"], c["kv"], c["dim"], c["rotary"], s["ring"]
    dt = _torch_type(c)
    x = s["qkv"].sum(0) if c["splits"] else s["qkv"]
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.view(-1, heads + 2 * kv, dim)
    angle = s["positions"].double().unsqueeze(1) * s["inv_freq"]
    cos, sin = angle.cos().float().unsqueeze(1), angle.sin().float().unsqueeze(1)
    y = x[:, :heads + kv].clone()
    if c["style"] == 0:
        lo, hi = x[:, :heads + kv, :r // 2], x[:, :heads + kv, r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = lo * cos - hi * sin, lo * sin + hi * cos
    else:
        lo, hi = x[:, :heads + kv, 0:r:2], x[:, :heads + kv, 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = lo * cos - hi * sin, lo * sin + hi * cos
    q, k, v = y[:, :heads], y[:, heads:], x[:, heads + kv:]
    # into the pages: a ring keeps a sequence's last positions only
    pos, row = s["positions"].long(), s["token_row"].long()
    place = pos % ring if ring else pos
    page = s["table"][row, place // PAGE].long()
    if ring:
        keep = (pos >= s["end"][row] - ring).nonzero().squeeze(1)
        page, place = page[keep], place[keep]
    else:
        keep = slice(None)
    pk, pv, pks, pvs = s["pages"]
    for src, codes, scales in ((k, pk, pks), (v, pv, pvs)):
        code, scale = _quantise(src[keep], c["fmt"])
        codes.view(torch.uint8)[page, :, place % PAGE] = code.view(torch.uint8)
        scales[page, :, place % PAGE] = scale
    held = _held(s["back_end"], s["back"].shape[1], ring)
    return (q.to(dt), k.to(dt), v.to(dt), _values(pk, pks, s["back"], held).to(dt),
            _values(pv, pvs, s["back"], held).to(dt))


def _plain_attend(s):
    c, table = s["case"], s["table"]
    heads, kv, dim, rows, width = c["heads"], c["kv"], c["dim"], table.shape[0], table.shape[1]
    held = _held(s["end"], width, s["ring"])

    def keys(codes, scales):
        x = _values(codes, scales, table, held).view(rows, width, kv, PAGE, dim)
        return x.transpose(1, 2).reshape(rows, kv, width * PAGE, dim)

    k, v = keys(s["pages"][0], s["pages"][2]), keys(s["pages"][1], s["pages"][3])
    # queries padded to the longest row
    row, cu, most = s["token_row"].long(), s["cu"].long(), s["longest"]
    at = torch.arange(row.shape[0], device=DEVICE) - cu[row]
    q = torch.zeros(rows, most, heads, dim, device=DEVICE)
    q[row, at] = s["q"].float()
    where = torch.full((rows, most), -1, dtype=torch.long, device=DEVICE)
    where[row, at] = s["positions"].long()
    q = q.view(rows, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(rows, kv, -1, dim)
    score = (q @ k.transpose(2, 3)).view(rows, kv, heads // kv, most, width * PAGE) * s["scale"]
    seen = (held.unsqueeze(1) >= 0) & (held.unsqueeze(1) <= where.unsqueeze(2))
    if c["window"]:
        seen &= held.unsqueeze(1) > where.unsqueeze(2) - c["window"]
    score = score.masked_fill(~seen.view(rows, 1, 1, most, -1), float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp()
    total = p.sum(-1, keepdim=True)
    o = (p.view(rows, kv, -1, width * PAGE) @ v).view(rows, kv, heads // kv, most, dim)
    o = torch.where(total > 0, o / total.clamp_min(1e-30), torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(rows, most, heads, dim)
    return o[row, at].to(s["q"].dtype)


def _plain_verify(s):
    t = s["case"]["temperature"]
    cu, logits, drafts = s["cu"].long(), s["logits"], s["drafts"].long()
    rows, n, vocab = s["draw_u"].shape[0], drafts.shape[0], logits.shape[1]
    count = cu[1:] - cu[:-1]
    row = torch.repeat_interleave(torch.arange(rows, device=DEVICE), count, output_size=n)
    place = torch.arange(n, device=DEVICE) + row                # a place more for every row before
    # the first maximum: the lowest index of those that are the largest
    index = torch.arange(vocab, device=DEVICE)
    if t < 1e-6:
        top = logits.amax(-1, keepdim=True)
        best = torch.where(logits == top, index, vocab).amin(-1)
        ok = best[place] == drafts
    else:
        p = ((logits.double() - logits.double().amax(-1, keepdim=True)) / t).exp()
        p = p / p.sum(-1, keepdim=True)
        here = p[place, drafts]
        if s["draft_logits"] is not None:
            d = s["draft_logits"].double()
            d = ((d - d.amax(-1, keepdim=True)) / t).exp() if n else d
            d = d / d.sum(-1, keepdim=True)
            ok = s["accept_u"].double() * d.gather(1, drafts.unsqueeze(1)).squeeze(1) < here
        else:
            ok = s["accept_u"].double() < here
    # accepted: the drafts before the first that is not
    at = torch.arange(n, device=DEVICE) - cu[row]
    accepted = count.clone()
    accepted.scatter_reduce_(0, row, torch.where(ok, count[row], at), "amin")
    stop = cu[:-1] + torch.arange(rows, device=DEVICE) + accepted
    if t < 1e-6:
        return accepted.to(torch.int32), best[stop].to(torch.int32)
    left = p[stop]
    cut = accepted < count
    if n:
        which = (cu[:-1] + accepted).clamp_max(n - 1)            # the rejected draft, where there is one
        if s["draft_logits"] is not None:
            less = (left - d[which]).clamp_min(0)
        else:
            less = left.scatter(1, drafts[which].unsqueeze(1), 0.0)
        cut = (cut & (less.sum(-1) > 0)).unsqueeze(1)
        left = torch.where(cut, less, left)
    run_sum = left.cumsum(-1)
    token = (run_sum <= s["draw_u"].double().unsqueeze(1) * run_sum[:, -1:]).sum(-1)
    last = torch.where(left > 0, index, 0).amax(-1)
    return accepted.to(torch.int32), torch.minimum(token, last).to(torch.int32)


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ------------------------------------------------------------------------------------------------
def _exact_vector(x, fmt):
    """What a 64-bit vector reads back as."""
    a = x.abs().max(-1, keepdim=True).values.clamp_min(2.0 ** -100)
    u = x / a * LIMIT[fmt]
    if fmt == "int8":
        return torch.round(u) * a / LIMIT[fmt]
    # e4m3: eight steps between two powers of two, the smallest step 2^-9
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(u / step) * step * a / LIMIT[fmt]


def _sequence(pages, scales, table, end, ring):
    """Position -> (place in the row's pages), and the row's vectors in 64 bits by place."""
    pages_of = table[table >= 0].long()
    x = pages[pages_of].double() * scales[pages_of].double().unsqueeze(-1)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])          # [kv, places, dim]


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "read": _exact_read, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](s)


def _exact_read(s):
    k, v, ks, vs = s["pages"]
    out = []
    ends, table = s["end"].tolist(), s["table"]
    for codes, scales in ((k, ks), (v, vs)):
        full = torch.zeros(table.shape[0], table.shape[1], codes.shape[1], PAGE, codes.shape[3], dtype=torch.float64, device=DEVICE)
        for b, end in enumerate(ends):
            n = -(-end // PAGE)
            x = codes[table[b, :n].long()].double() * scales[table[b, :n].long()].double().unsqueeze(-1)
            full[b, :n] = x
            if end % PAGE:
                full[b, n - 1, :, end % PAGE:] = 0
        out.append(full.view(-1, *full.shape[2:]))
    return tuple(out)


def _exact_store(s):
    c, ring = s["case"], s["ring"]
    heads, kv, dim, r = c["heads"], c["kv"], c["dim"], c["rotary"]
    x = s["qkv"].double()
    x = x.sum(0) if c["splits"] else x
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.view(x.shape[0], heads + 2 * kv, dim)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE), s["positions"].double()[:, None] * s["inv_freq"][None])
    y = x.clone()
    first = (torch.arange(r // 2, device=DEVICE) * (1 if c["style"] == 0 else 2))
    second = first + (r // 2 if c["style"] == 0 else 1)
    z = torch.complex(x[:, :heads + kv][..., first], x[:, :heads + kv][..., second]) * turn[:, None]
    y[:, :heads + kv, first], y[:, :heads + kv, second] = z.real, z.imag
    k, v = y[:, heads:heads + kv], y[:, heads + kv:]
    out = [y[:, :heads], k, v]
    cu, ends, back_ends = s["cu"].tolist(), s["end"].tolist(), s["back_end"].tolist()
    pk, pv, pks, pvs = s["pages"]
    for src, codes, scales in ((k, pk, pks), (v, pv, pvs)):
        full = torch.zeros(len(ends), s["back"].shape[1], PAGE, kv, dim, dtype=torch.float64, device=DEVICE)
        for b, end in enumerate(ends):
            table = s["back"][b]
            old = _sequence(codes, scales, table, end, ring)                   # what was there before
            flat = full[b].view(-1, kv, dim)
            base = end - back_ends[b]                                          # position of place 0 (linear)
            n, start = cu[b + 1] - cu[b], end - (cu[b + 1] - cu[b])
            for lo, hi, vectors in ((max(0, end - ring) if ring else base, start, None), (start, end, src[cu[b]:cu[b + 1]])):
                pos = torch.arange(max(lo, end - ring) if ring else lo, hi, device=DEVICE)
                if pos.numel() == 0:
                    continue
                place = pos % ring if ring else pos - base
                if vectors is None:
                    flat[place] = old.transpose(0, 1)[place]
                else:
                    flat[place] = _exact_vector(vectors[pos - start], c["fmt"])
        out.append(full.transpose(2, 3).reshape(-1, kv, PAGE, dim))
    return tuple(out)


def _exact_attend(s):
    c, ring = s["case"], s["ring"]
    w = work(c)
    if w["flops"] > 4e11:
        return None
    heads, kv = c["heads"], c["kv"]
    pk, pv, pks, pvs = s["pages"]
    cu, ends = s["cu"].tolist(), s["end"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b, end in enumerate(ends):
        k = _sequence(pk, pks, s["table"][b], end, ring)
        v = _sequence(pv, pvs, s["table"][b], end, ring)
        start = end - (cu[b + 1] - cu[b])
        lo = max(0, start - c["window"] + 1) if c["window"] else 0
        pos = torch.arange(lo, end, device=DEVICE)
        place = pos % ring if ring else pos
        k, v = k[:, place], v[:, place]
        q = s["q"][cu[b]:cu[b + 1]].double()
        at = torch.arange(start, end, device=DEVICE)[:, None]
        hidden = pos[None] > at
        if c["window"]:
            hidden |= pos[None] <= at - c["window"]
        for h in range(heads):
            score = torch.einsum("td,kd->tk", q[:, h], k[h * kv // heads]) * s["scale"]
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[cu[b]:cu[b + 1], h] = torch.einsum("tk,kd->td", p, v[h * kv // heads])
    return out


def _exact_verify(s):
    t = s["case"]["temperature"]
    cu, drafts = s["cu"].tolist(), s["drafts"].tolist()
    u, r = s["accept_u"].double().tolist(), s["draw_u"].double().tolist()
    accepted, tokens = [], []
    for b in range(len(r)):
        n, first = cu[b + 1] - cu[b], cu[b] + b
        got, token = n, None
        for j in range(n + 1):
            logits = s["logits"][first + j].double()
            if t < 1e-6:
                best = int((logits == logits.max()).nonzero()[0])
                if j == n or best != drafts[cu[b] + j]:
                    got, token = j, best
                    break
                continue
            p = torch.softmax(logits / t, -1)
            if j < n:
                x = drafts[cu[b] + j]
                if s["draft_logits"] is not None:
                    q = torch.softmax(s["draft_logits"][cu[b] + j].double() / t, -1)
                else:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                if u[cu[b] + j] * float(q[x]) < float(p[x]):
                    continue
                less = torch.relu(p - q) if s["draft_logits"] is not None else p * (1.0 - q)
                p = less if float(less.sum()) > 0 else p
            got = j
            sums = torch.cumsum(p, 0)
            above = (sums > r[b] * sums[-1]).nonzero()
            token = int(above[0]) if above.numel() else int((p > 0).nonzero()[-1])
            break
        accepted.append(got)
        tokens.append(token)
    return _ints(accepted), _ints(tokens)
