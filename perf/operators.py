"""Operators over a key / value cache held in 4 bits, as cases that can be timed and compared.

The cache is a pool of 16-token pages.  ``data`` (uint8 [pages][kv heads][18 * D]) holds for a page and kv head

    K codes  [16 tokens][D / 2 bytes]    element d in byte d // 2, low half for even d; code = q + 8, q in -7 .. 7
    V codes  [16 tokens][D / 2 bytes]
    maxima   [16 tokens][K, V][D / 32]   bf16

and element d of a token's row stands for ``q * maximum[(d // 4) % (D / 32)] / 7``: 32 elements share a maximum, quads of
them dealt out in turn.  ``mass`` (fp32 [pages][kv heads][16]) is the attention weight that a cached token has drawn so far.
``table`` (int32 [slots][pages of a sequence]) maps a sequence's pages, -1 where none is mapped.

Four kinds of pass, each through calls that a serving program makes:

attend   rows of many sequences over the cache: softmax(scale * q k^T) v, optional sliding window and sigmoid output gate;
         a row that sees no key gives zeros
weigh    attention of the last rows of a prompt, which sets the mass of every token of the sequence to the weight that it
         drew (summed over rows and the query heads of a kv head), then of one later row over the same tokens, which adds to it
write    rows of a prompt chunk (or one token) are quantised into the pages, then the whole sequence is read back as bf16,
         which is what attention over a following prompt chunk works on
evict    per kv head the tokens with the most mass are selected (with the first `sink` and the last `recent` ones; ties go
         to the earlier token), moved to fresh pages with their mass, and read back as bf16
"""
import math

import torch

own = False

_PAGE = 16


# ------------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------------
def _attend(rows, length, hkv, group, d, window=0, gate=False, empty=0):
    return {"op": "attend", "rows": rows, "length": length, "hkv": hkv, "group": group, "d": d, "window": window, "gate": gate, "empty": empty}


def _weigh(seqs, length, window_rows, hkv, group, d):
    return {"op": "weigh", "rows": seqs, "length": length, "observed": window_rows, "hkv": hkv, "group": group, "d": d}


def _write(new, length, hkv, d):
    return {"op": "write", "rows": 1, "new": new, "length": length, "hkv": hkv, "group": 1, "d": d}


def _evict(seqs, length, keep, recent, sink, hkv, d):
    return {"op": "evict", "rows": seqs, "length": length, "keep": keep, "recent": recent, "sink": sink, "hkv": hkv, "group": 1, "d": d}


def listed():
    return [
        # one user, a short question: nothing but latency (40 query / 8 kv heads x 128, the dense 27B geometry)
        {"name": "attend_one_short", **_attend(1, 107, 8, 5, 128)},
        # one user with a very long document
        {"name": "attend_one_131072", **_attend(1, 131072, 8, 5, 128)},
        # eight users at a few thousand tokens, every length another one: the ordinary serving step
        {"name": "attend_eight_ragged", **_attend(8, 4999, 8, 5, 128)},
        # gated attention of the hybrid 27B (24 query / 4 kv heads x 256), sixteen users
        {"name": "attend_gated_256", **_attend(16, 8191, 4, 6, 256, gate=True)},
        # small heads without sharing, sliding window, rows of a padded batch that see nothing
        {"name": "attend_window_64", **_attend(24, 6000, 16, 1, 64, window=1024, empty=3)},
        # thirty-two users at 32k tokens: more than a gigabyte of cache in one step
        {"name": "attend_batch_32768", **_attend(32, 32768, 8, 5, 128)},
        # after a prompt of ordinary length: which tokens did its last rows look at, then the first generated token
        {"name": "weigh_prompt_2001", **_weigh(1, 2001, 16, 8, 5, 128)},
        # the same for four long prompts
        {"name": "weigh_four_16384", **_weigh(4, 16384, 32, 8, 5, 128)},
        # one generated token of a short conversation
        {"name": "write_one_row", **_write(1, 1003, 8, 128)},
        # a prompt chunk behind a long history
        {"name": "write_chunk_4096", **_write(4096, 36001, 8, 128)},
        # one conversation cut to half its cache
        {"name": "evict_one_2000", **_evict(1, 2000, 1024, 64, 4, 8, 128)},
        # eight long conversations cut to an eighth
        {"name": "evict_eight_32768", **_evict(8, 32768, 4096, 256, 4, 8, 128)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "weigh", "write", "evict"])
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    if op == "attend":
        rows = _log(rng, 1, 64)
        length = _log(rng, 1, min(131072, 400000 // rows, (1 << 32) // (hkv * group * d * rows)))
        window = _log(rng, 1, length) if rng.random() < 0.25 else 0
        return _attend(rows, length, hkv, group, d, window, rng.random() < 0.4, rng.choice([0, 0, rows // 3]))
    if op == "weigh":
        seqs = _log(rng, 1, 8)
        length = _log(rng, 2, 65536 // seqs)
        return _weigh(seqs, length, min(length // 2, _log(rng, 1, max(1, min(32, 163840 // (hkv * group * d))))), hkv, group, d)
    if op == "write":
        new = _log(rng, 1, 4096)
        return _write(new, new + _log(rng, 1, 32000), hkv, d)
    seqs = _log(rng, 1, 8)
    length = _log(rng, 2, 100000 // seqs)
    keep = _log(rng, 1, length)
    recent = rng.randint(0, keep)
    return _evict(seqs, length, keep, recent, rng.randint(0, min(4, keep - recent)), hkv, d)


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """A length for every row, the same for every seed: the first one is the case's, the others lie between a half of it and
    all of it."""
    n, s = case["length"], case["rows"]
    if s == 1:
        return [n]
    r = torch.rand(s, generator=torch.Generator().manual_seed(n))
    out = [max(1, int(n * (0.5 + 0.5 * float(x)))) for x in r]
    out[0] = n
    return out


def _fill(data, g, d):
    """Random cached rows in every page: normal values, a few channels of K four times as large, as trained keys have them."""
    pages, hkv, _ = data.shape
    gain = torch.ones(d, device="cuda")
    gain[torch.randperm(d, generator=g, device="cuda")[: max(1, d // 32)]] = 4.0
    step = max(1, (1 << 28) // (hkv * _PAGE * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        part = data[a:b]
        for which in (0, 1):
            x = torch.randn(b - a, hkv, _PAGE, d, generator=g, device="cuda")
            codes, amax = _quantise((x * gain if which == 0 else x).bfloat16())
            part[:, :, which * 8 * d: (which + 1) * 8 * d] = codes.flatten(2)
            part[:, :, 16 * d:].view(torch.bfloat16).unflatten(-1, (_PAGE, 2, d // 32))[:, :, :, which] = amax


def prepare(case, seed):
    op, d, hkv, group = case["op"], case["d"], case["hkv"], case["group"]
    host = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens = _lengths(case)
    seqs = len(lens)
    most = max(lens)
    per_seq = [(n + _PAGE - 1) // _PAGE for n in lens]
    kept_pages = (case["keep"] + _PAGE - 1) // _PAGE if op == "evict" else 0
    pages = sum(per_seq) + seqs * kept_pages + 3
    order = torch.randperm(pages, generator=host).to(torch.int32)
    slots = torch.randperm(seqs + 1, generator=host)[:seqs].tolist()          # rows do not come in the order of the slots
    width = max(per_seq) + 2
    table = torch.full((seqs + 1, width), -1, dtype=torch.int32)
    at = 0
    for s, n in zip(slots, per_seq):
        table[s, :n] = order[at: at + n]
        at += n
    st = {"op": op, "d": d, "hkv": hkv, "group": group, "length": most, "lengths": i32(lens), "slots": i32(slots), "table": table.cuda(),
          "data": torch.zeros(pages, hkv, 18 * d, dtype=torch.uint8, device="cuda"), "scale": 1.0 / math.sqrt(d)}
    _fill(st["data"], g, d)
    hq = hkv * group
    rows = lambda n, w: torch.randn(n, w, generator=g, device="cuda")  # noqa: E731
    if op == "attend":
        pos = [n - 1 for n in lens]
        for i in range(case["empty"]):
            pos[-1 - i] = -1                                                   # padding rows of the batch
        st |= {"q": (1.5 * rows(seqs, hq * d)).bfloat16(), "pos": i32(pos), "window": case["window"],
               "gate": rows(seqs, hq * d).bfloat16() if case["gate"] else None, "out": torch.empty(seqs, hq * d, dtype=torch.bfloat16, device="cuda")}
    elif op == "weigh":
        w = case["observed"]                                                    # the last w tokens' rows of every prompt
        st |= {"q": (1.5 * rows(seqs * w, hq * d)).bfloat16(), "pos": i32((torch.tensor(lens)[:, None] - w + torch.arange(w)).flatten().tolist()),
               "row_slots": st["slots"].repeat_interleave(w), "observed": w,
               "q1": (1.5 * rows(seqs, hq * d)).bfloat16(), "pos1": i32([n - 1 for n in lens]),
               "mass": torch.rand(pages, hkv, _PAGE, generator=g, device="cuda"),
               "out": torch.empty(seqs * w, hq * d, dtype=torch.bfloat16, device="cuda"), "out1": torch.empty(seqs, hq * d, dtype=torch.bfloat16, device="cuda")}
    elif op == "write":
        n = case["new"]
        st |= {"k": rows(n, hkv * d).bfloat16(), "v": rows(n, hkv * d).bfloat16(), "pos": torch.arange(most - n, most, dtype=torch.int32, device="cuda"),
               "row_slots": st["slots"].expand(n).contiguous()}
    else:
        # weights fall off steeply and many tokens were never looked at: whole runs of equal (zero) mass
        m = torch.exp(2.5 * torch.randn(pages, hkv, _PAGE, generator=g, device="cuda"))
        st |= {"mass": m * (torch.rand(pages, hkv, _PAGE, generator=g, device="cuda") < 0.7), "keep": case["keep"], "recent": case["recent"], "sink": case["sink"],
               "fresh": order[at: at + seqs * kept_pages].reshape(seqs, kept_pages).cuda()}
    if op in ("write", "evict"):
        n = case["keep"] if op == "evict" else most
        st["dense_k"] = torch.zeros(seqs, n, hkv * d, dtype=torch.bfloat16, device="cuda")
        st["dense_v"] = torch.zeros_like(st["dense_k"])
    return st


# ------------------------------------------------------------------------------------------------------------------------
# plain form
# ------------------------------------------------------------------------------------------------------------------------
def _quantise(x):
    """bf16 [..., D] -> (bytes of two codes [..., D / 2], maxima bf16 [..., D / 32]).  7 x / max has at most 11 bits over 8: the
    quotient of 32 bits rounds as the exact one does."""
    d = x.shape[-1]
    ng = d // 32
    quads = x.float().unflatten(-1, (8, ng, 4))
    amax = quads.abs().amax(dim=(-3, -1))
    div = torch.where(amax > 0, amax, torch.ones_like(amax))[..., None, :, None]
    codes = (torch.round(quads * 7 / div) + 8).to(torch.uint8).flatten(-3)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), amax.bfloat16()


def _values(part, d):
    """Pages [..., 18 * D] -> K, V as fp32 [..., 16, D]."""
    codes = part[..., : 16 * d].unflatten(-1, (2, _PAGE, d // 2))
    amax = part[..., 16 * d:].contiguous().view(torch.bfloat16).unflatten(-1, (_PAGE, 2, d // 32)).transpose(-3, -2).float()
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float() - 8
    x = (q.unflatten(-1, (8, d // 32, 4)) * amax[..., None, :, None] / 7).flatten(-3)
    return x.select(-3, 0), x.select(-3, 1)


def _cached(st, slots, length):
    """K, V of the sequences in ``slots``, fp32 [sequences][kv heads][length][D]."""
    n = (length + _PAGE - 1) // _PAGE
    part = st["data"][st["table"][slots.long(), :n].clamp_min(0).long()].transpose(1, 2)
    k, v = _values(part, st["d"])
    return k.flatten(2, 3)[:, :, :length], v.flatten(2, 3)[:, :, :length]


def _softmax(st, k, q, pos, window):
    """Weights [sequences][kv heads][rows * group][length] of ``rows`` query rows a sequence."""
    s, hkv, length, d = k.shape
    w = q.shape[0] // s
    qq = q.float().reshape(s, w, hkv, st["group"], d).transpose(1, 2).flatten(2, 3)
    sc = (qq @ k.transpose(2, 3)) * st["scale"]
    p = pos.reshape(s, 1, w, 1, 1).long()
    t = torch.arange(length, device="cuda")
    seen = (t <= p) & (t > p - window) if window else t <= p
    sc = sc.unflatten(2, (w, st["group"])).masked_fill(~seen, -math.inf)
    top = sc.amax(dim=-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    return (e / torch.where(total > 0, total, torch.ones_like(total))).flatten(2, 3)


def _rows(st, weights, v):
    """weights @ v, back in the order of the rows: [rows][query heads * D] fp32."""
    s, hkv, wg, _ = weights.shape
    o = (weights @ v).unflatten(2, (wg // st["group"], st["group"]))
    return o.transpose(1, 2).reshape(s * (wg // st["group"]), hkv * st["group"] * st["d"])


def _plain_attend(st):
    k, v = _cached(st, st["slots"], st["length"])
    o = _rows(st, _softmax(st, k, st["q"], st["pos"], st["window"]), v)
    if st["gate"] is not None:
        o = o / (1 + torch.exp(-st["gate"].float()))
    return o.bfloat16()


def _plain_weigh(st):
    length = st["length"]
    k, v = _cached(st, st["slots"], length)
    w0 = _softmax(st, k, st["q"], st["pos"], 0)
    w1 = _softmax(st, k, st["q1"], st["pos1"], 0)
    t = torch.arange(length, device="cuda")
    page = st["table"][st["slots"].long()][:, t // _PAGE].long()               # [sequences][length]
    page, slot, mass = page.clamp_min(0), t % _PAGE, st["mass"]
    live = t < st["lengths"][:, None]
    seq, tok = live.nonzero(as_tuple=True)
    mass[page[seq, tok], :, slot[tok]] = w0.sum(2)[seq, :, tok]
    mass[page[seq, tok], :, slot[tok]] += w1.sum(2)[seq, :, tok]
    return _rows(st, w0, v).bfloat16(), _rows(st, w1, v).bfloat16()


def _plain_write(st):
    d, data, ng = st["d"], st["data"], st["d"] // 32
    n = st["k"].shape[0]
    page = st["table"][st["row_slots"].long(), (st["pos"] // _PAGE).long()].long()
    slot = (st["pos"] % _PAGE).long()
    codes = data[..., : 16 * d].unflatten(-1, (2, _PAGE, d // 2))
    amax = data[..., 16 * d:].view(torch.bfloat16).unflatten(-1, (_PAGE, 2, ng))
    kq, ka = _quantise(st["k"].reshape(n, st["hkv"], d))
    vq, va = _quantise(st["v"].reshape(n, st["hkv"], d))
    codes[page, :, 0, slot], codes[page, :, 1, slot] = kq, vq
    amax[page, :, slot, 0], amax[page, :, slot, 1] = ka, va
    k, v = _cached(st, st["slots"], st["length"])
    return k.transpose(1, 2).flatten(2).bfloat16(), v.transpose(1, 2).flatten(2).bfloat16()


def _plain_evict(st):
    length, keep = st["length"], st["keep"]
    t = torch.arange(length, device="cuda")
    n = st["lengths"][:, None].long()
    page = st["table"][st["slots"].long()][:, t // _PAGE].clamp_min(0).long()  # [sequences][length]
    slot = (t % _PAGE).expand_as(page)
    mass = st["mass"][page, :, slot].transpose(1, 2)                           # [sequences][kv heads][length]
    must = ((t < st["sink"]) | (t >= n - st["recent"])) & (t < n)
    rank = torch.where((t < n)[:, None], mass, torch.full_like(mass, -1)).masked_fill(must[:, None], math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.where(best < n[:, None], best, torch.full_like(best, length)).sort(dim=-1).values
    some = best < length                                                       # fewer tokens than `keep`: all of them stay
    idx = torch.where(some, best, torch.full_like(best, -1)).to(torch.int32)
    src = best.clamp_max(length - 1)
    head = torch.arange(st["hkv"], device="cuda")[:, None]
    seq = torch.arange(src.shape[0], device="cuda")[:, None, None]
    sp, ss = page[seq, src], src % _PAGE                                       # where each kept token lies
    to = torch.arange(keep, device="cuda")
    dp, ds = st["fresh"][:, to // _PAGE].long()[:, None].expand_as(sp), (to % _PAGE).expand_as(sp)
    d, data = st["d"], st["data"]
    codes = data[..., : 16 * d].unflatten(-1, (2, _PAGE, d // 2))
    amax = data[..., 16 * d:].view(torch.bfloat16).unflatten(-1, (_PAGE, 2, d // 32))
    hh = head.expand_as(sp)
    pick = lambda x: x[some]  # noqa: E731
    a, b, c = pick(dp), pick(hh), pick(ds)
    for_codes = codes[pick(sp), b, :, pick(ss)]
    for_amax = amax[pick(sp), b, pick(ss)]
    for_mass = st["mass"][pick(sp), b, pick(ss)]
    codes[a, b, :, c], amax[a, b, c], st["mass"][a, b, c] = for_codes, for_amax, for_mass
    part = data[st["fresh"].long()].transpose(1, 2)
    k, v = (x.flatten(2, 3)[:, :, :keep].transpose(1, 2).flatten(2).bfloat16() for x in _values(part, d))
    full = (torch.arange(keep, device="cuda") < n)[..., None]                  # rows past the kept tokens are not written
    st["dense_k"].copy_(torch.where(full, k, st["dense_k"]))
    st["dense_v"].copy_(torch.where(full, v, st["dense_v"]))
    return idx, st["mass"], st["dense_k"], st["dense_v"]


# ------------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------------
def _own(st):
    from grimoire_b200.ops import kv4
    from grimoire_b200.ops.core import AttnGeom

    op, table = st["op"], st["table"]
    kv = kv4.Kv4Layer(st["data"], st.get("mass"))
    if op in ("attend", "weigh"):
        geom = AttnGeom(st["hkv"] * st["group"], st["hkv"], st["d"], st["d"], st["scale"], window=st.get("window", 0))
    if op == "attend":
        kv4.kv4_attn(st["q"], st["slots"], st["pos"], table, kv, geom, st["out"], st["length"], gate=st["gate"])
        return st["out"]
    if op == "weigh":
        kv4.kv4_attn(st["q"], st["row_slots"], st["pos"], table, kv, geom, st["out"], st["length"], block=st["observed"], observe="set")
        kv4.kv4_attn(st["q1"], st["slots"], st["pos1"], table, kv, geom, st["out1"], st["length"], observe="add")
        return st["out"], st["out1"]
    if op == "write":
        kv4.kv4_append(kv, st["k"], st["v"], st["pos"], st["row_slots"], table)
        kv4.kv4_gather(kv, table, st["slots"], st["lengths"], st["dense_k"], st["dense_v"])
        return st["dense_k"], st["dense_v"]
    idx = kv4.kv4_select(kv, st["slots"], st["lengths"], table, st["keep"], st["recent"], st["sink"])
    kv4.kv4_compact(kv, st["slots"], idx, table, st["fresh"])
    kv4.kv4_gather(kv, st["fresh"], None, st["lengths"], st["dense_k"], st["dense_v"])
    return idx, st["mass"], st["dense_k"], st["dense_v"]


def run(state):
    op = state["op"]
    if own:
        r = _own(state)
    else:
        r = {"attend": _plain_attend, "weigh": _plain_weigh, "write": _plain_write, "evict": _plain_evict}[op](state)
    if op == "attend":
        return {"out": r}
    if op == "weigh":
        return {"out": r[0], "out1": r[1], "mass": state["mass"]}
    if op == "write":
        return {"k": r[0], "v": r[1]}
    return {"kept": r[0], "mass": r[1], "k": r[2], "v": r[3]}


def work(case):
    """What one pass cannot do without (a ragged batch's mean length is three quarters of its longest)."""
    op, d, hkv, group, s = case["op"], case["d"], case["hkv"], case["group"], case["rows"]
    token = hkv * 18 * d / 16                                                  # bytes of a cached token
    n = case["length"] * (1.0 if s == 1 else 0.75 + 0.25 / s)
    hq = hkv * group
    if op == "attend":
        live = s - case["empty"]
        seen = min(n, case["window"]) if case["window"] else n
        return {"bytes": live * seen * token + s * hq * d * (6 if case["gate"] else 4), "flops": 4.0 * live * seen * hq * d}
    if op == "weigh":
        w = case["observed"]
        return {"bytes": s * n * (2 * token + 4 * 3 * hkv) + s * (w + 1) * hq * d * 4, "flops": 4.0 * s * n * (w + 1) * hq * d}
    if op == "write":
        return {"bytes": case["new"] * (4 * hkv * d + token) + n * (token + 4 * hkv * d), "flops": 4.0 * n * hkv * d}
    kept = min(case["keep"], n)
    return {"bytes": s * (n * 4 * hkv + 4 * hkv * case["keep"] + kept * (2 * (token + 4 * hkv) + token + 4 * hkv * d)), "flops": 2.0 * s * n * hkv}


# ------------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------------------------------
def _element(st, page, head, which, slot):
    """Rows of the cache from the definition: [tokens][D] in 64 bits.  page, slot: [tokens]."""
    d, ng = st["d"], st["d"] // 32
    e = torch.arange(d, device="cuda")
    byte = st["data"][page[:, None], head, which * 8 * d + slot[:, None] * (d // 2) + e // 2].to(torch.int32)
    code = torch.where(e % 2 == 0, byte % 16, byte // 16)
    place = 16 * d + 2 * ((slot[:, None] * 2 + which) * ng + (e // 4) % ng)
    low, high = (st["data"][page[:, None], head, place + i].to(torch.int32) for i in (0, 1))
    top = ((high * 256 + low) * 65536).view(torch.float32).double()            # the bits of a bf16 are the upper ones of 32
    return (code - 8).double() * top / 7


def _exact_rows(st, slot, head, q, pos, window):
    """(outputs, weights) in 64 bits of the rows ``q`` [rows][group][D] of one sequence and kv head."""
    n = int(pos.max()) + 1
    t = torch.arange(n, device="cuda")
    page = st["table"][slot, t // _PAGE].long()
    k, v = _element(st, page, head, 0, t % _PAGE), _element(st, page, head, 1, t % _PAGE)
    s = torch.einsum("rgd,td->rgt", q.double(), k) * st["scale"]
    hidden = t > pos[:, None]
    if window:
        hidden = hidden | (t <= pos[:, None] - window)
    w = torch.softmax(s.masked_fill(hidden[:, None], -math.inf), dim=-1)
    return torch.einsum("rgt,td->rgd", w, v), w


def exact(case, seed):
    st = prepare(case, seed)
    op, d, hkv, group = st["op"], st["d"], st["hkv"], st["group"]
    slots, lens = st["slots"].tolist(), st["lengths"].tolist()
    if op in ("attend", "weigh"):
        def over(q, pos, w, mass, add):
            out = torch.zeros(q.shape[0], hkv, group, d, dtype=torch.float64, device="cuda")
            for i, slot in enumerate(slots):
                p = pos[i * w: (i + 1) * w].long()
                if int(p.max()) < 0:
                    continue
                for h in range(hkv):
                    rows = q[i * w: (i + 1) * w].reshape(w, hkv, group, d)[:, h]
                    out[i * w: (i + 1) * w, h], weights = _exact_rows(st, slot, h, rows, p, st.get("window", 0))
                    if mass is not None:
                        t = torch.arange(weights.shape[-1], device="cuda")
                        at = (st["table"][slot, t // _PAGE].long(), h, t % _PAGE)
                        mass[at] = weights.sum((0, 1)) + (mass[at] if add else 0)
            return out.reshape(q.shape[0], -1)

        if op == "attend":
            o = over(st["q"], st["pos"], 1, None, False)
            return {"out": o if st["gate"] is None else o * torch.sigmoid(st["gate"].double())}
        mass = st["mass"].double()
        o = over(st["q"], st["pos"], st["observed"], mass, False)
        return {"out": o, "out1": over(st["q1"], st["pos1"], 1, mass, True), "mass": mass}
    if op == "write":
        n, new = st["length"], st["k"].shape[0]
        t = torch.arange(n - new, device="cuda")
        page = st["table"][slots[0], t // _PAGE].long()
        got = []
        for which, x in ((0, st["k"]), (1, st["v"])):
            old = torch.stack([_element(st, page, h, which, t % _PAGE) for h in range(hkv)], dim=1)
            x = x.double().reshape(new, hkv, d)
            kind = (torch.arange(d, device="cuda") // 4) % (d // 32)
            fresh = torch.zeros_like(x)
            for j in range(d // 32):
                part = x[..., kind == j]
                top = part.abs().max(dim=-1, keepdim=True).values
                fresh[..., kind == j] = torch.where(top > 0, torch.round(7 * part / top) * top / 7, 0 * part)
            got.append(torch.cat((old, fresh)).reshape(1, n, hkv * d))
        return {"k": got[0], "v": got[1]}
    kept, mass = torch.full((len(slots), hkv, st["keep"]), -1, dtype=torch.int32), st["mass"].double()
    k, v = st["dense_k"].double(), st["dense_v"].double()
    host = st["mass"].cpu()
    for i, (slot, n) in enumerate(zip(slots, lens)):
        pages = st["table"][slot, : (n + _PAGE - 1) // _PAGE].long()
        for h in range(hkv):
            m = host[pages.cpu(), h].reshape(-1)[:n].double().numpy()
            lo, hi = min(st["sink"], n), max(n - st["recent"], min(st["sink"], n))
            order = sorted(range(lo, hi), key=lambda j: (-m[j], j))[: max(0, st["keep"] - lo - (n - hi))]
            idx = torch.tensor(sorted(list(range(lo)) + order + list(range(hi, n)))[: st["keep"]])
            kept[i, h, : len(idx)] = idx.to(torch.int32)
            idx = idx.cuda()
            at, to = (pages[idx // _PAGE], idx % _PAGE), torch.arange(len(idx), device="cuda")
            k[i, : len(idx), h * d: (h + 1) * d] = _element(st, at[0], h, 0, at[1])
            v[i, : len(idx), h * d: (h + 1) * d] = _element(st, at[0], h, 1, at[1])
            mass[st["fresh"][i, to // _PAGE].long(), h, to % _PAGE] = st["mass"][at[0], h, at[1]].double()
    return {"kept": kept, "mass": mass, "k": k, "v": v}
