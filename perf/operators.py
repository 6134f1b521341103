"""Operators of many completions of one prompt, and of long contexts: the cache in 8 bits, the attention of single
tokens over it, and the attention of sequences that share a prefix.

``"op": "store"``   keys and values of a step's tokens go into the cache's pages as e4m3 codes with one power of two a
                    row (a token's head): the least 2^e with max |x| <= 448 * 2^e over the row's finite values.  With
                    ``"rounded"`` the rounded rows come back as bfloat16 too, for the prompt's own attention.
``"op": "decode"``  one new token per sequence attends over the 8-bit cache: grouped heads, softcap, a sliding window or
                    a chunk, first tokens that stay in sight, a sink per head; rows of a window lie in a ring of pages.
``"op": "shared"``  one new token per sequence; the sequences of a group share their first pages, in a bfloat16 cache
                    or in the 8-bit one.

A cache page holds 64 rows of every kv head.  Pages are taken in no order; rows behind a sequence's end hold what an
earlier sequence left there (in the 8-bit cache any byte).  Queries, keys and values are normal, a few channels of the
keys some times larger, as projections give them.
"""
import math

import torch

own = False

PAGE = 64
TOP = 448.0                 # the largest e4m3 value


# ---------------------------------------------------------------------------------------------- the cases

def _store(name, lens, before, nkv, group, hd, rounded, window=0, keep=0):
    return {"name": name, "op": "store", "batch": len(lens), "new": " ".join(map(str, lens)), "before": " ".join(map(str, before)),
            "nkv": nkv, "group": group, "hd": hd, "rounded": rounded, "window": window, "keep": keep}


def _decode(name, batch, tokens, nkv, group, hd, ragged=False, cap=0.0, mask="window", window=0, keep=0, sinks=False):
    return {"name": name, "op": "decode", "batch": batch, "tokens": tokens, "nkv": nkv, "group": group, "hd": hd, "ragged": ragged,
            "cap": cap, "mask": mask, "window": window, "keep": keep, "sinks": sinks}


def _shared(name, bits, groups, members, prefix, rest, nkv, group, hd, cap=0.0, sinks=False):
    return {"name": name, "op": "shared", "bits": bits, "groups": groups, "members": members, "prefix": prefix, "rest": rest,
            "nkv": nkv, "group": group, "hd": hd, "cap": cap, "sinks": sinks}


def listed():
    return [
        # a decode step of eight sequences (Gemma-2 2B heads): one row a sequence and head, launches count
        _store("store decode b8", [1] * 8, [2048] * 8, 4, 2, 256, False),
        # a document's keys and values, with the rounded rows for its own attention
        _store("store prompt 2048", [2048], [0], 4, 2, 256, True),
        # three unequal prompts of heads of 128 into a window's ring: only the last rows stay
        _store("store prompts in a ring", [9001, 333, 5000], [0, 0, 0], 16, 2, 128, True, window=4096),
        # one conversation: the smallest decode step
        _decode("decode8 b1 x 700", 1, 701, 4, 2, 256, cap=50.0),
        # the headline workload's attention: eight sequences behind 2,048-token prompts
        _decode("decode8 b8 x 2048", 8, 2049, 4, 2, 256, cap=50.0),
        # a full server: 64 sequences of unequal lengths, a sliding layer of Gemma-2 9B
        _decode("decode8 b64 ragged window", 64, 8192, 8, 2, 256, ragged=True, cap=50.0, window=4096),
        # heads of 64 in groups of four, kept first tokens beside a window, sinks
        _decode("decode8 b16 heads of 64", 16, 3001, 2, 4, 64, ragged=True, window=1024, keep=16, sinks=True),
        # one very long context of grouped heads: bound by the cache's bytes
        _decode("decode8 b1 x 131072", 1, 131072, 8, 4, 128),
        # four answers to a question about a page of text
        _shared("shared b4 prefix 1024", 16, 1, 4, 1024, 60, 4, 2, 256, cap=50.0),
        # 64 completions of a long prompt, Gemma-2 2B heads
        _shared("shared b64 prefix 7168", 16, 1, 64, 7168, 300, 4, 2, 256, cap=50.0),
        # three prompts with 5 completions each, sinks
        _shared("shared 3 x 5 prefix 3000", 8, 3, 5, 2985, 200, 6, 3, 128, sinks=True),
        # 32 completions behind a book's chapter, the cache in 8 bits
        _shared("shared 8 bits b32 prefix 32768", 8, 1, 32, 32768, 500, 8, 4, 128),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "shared", "shared"])
    hd = rng.choice([64, 128, 256])
    nkv, group = rng.choice([1, 2, 3, 4, 5, 8, 16]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    if op == "store":
        window = rng.choice([0, 0, 100, 512, 4096])
        keep = rng.choice([0, 4, 70]) if window else 0
        if rng.random() < 0.5:
            batch = _log(rng, 1, 256)
            case = _store("", [1] * batch, [_log(rng, 1, 8000) for _ in range(batch)], nkv, group, hd, False, window, keep)
        else:
            batch = _log(rng, 1, 8)
            most = max(2, min(12000, 16_000_000 // (nkv * hd * batch)))
            case = _store("", [_log(rng, 1, most) for _ in range(batch)], [0] * batch, nkv, group, hd, True, window, keep)
    elif op == "decode":
        window = rng.choice([0, 0, 0, 33, 1024, 4096])
        batch = _log(rng, 1, 128)
        most = max(2, int(min(131072, 6.0e7 / (nkv * hd * batch), 3.0e9 / (nkv * group * hd * batch))))
        case = _decode("", batch, _log(rng, 1, most), nkv, group, hd, ragged=bool(rng.random() < 0.6),
                       cap=rng.choice([0.0, 0.0, 30.0, 50.0]), mask=rng.choice(["window", "window", "chunk"]) if window else "window",
                       window=window, keep=rng.choice([0, 0, 5, 64]) if window else 0, sinks=bool(rng.random() < 0.3))
    else:
        groups, members = rng.choice([1, 1, 1, 2, 3, 5]), _log(rng, 2, 64)
        most = max(65, int(min(40000, 3.0e7 / (nkv * hd * groups), 2.0e9 / (nkv * group * hd * groups * members))))
        case = _shared("", rng.choice([8, 16]), groups, members, _log(rng, 65, most), _log(rng, 1, 400), nkv, group, hd,
                       cap=rng.choice([0.0, 0.0, 50.0]), sinks=bool(rng.random() < 0.2))
    del case["name"]
    return case


def _lengths(n, batch, ragged):
    """Tokens of every sequence: all equal, or from the longest down over the logarithm of the range."""
    if not ragged:
        return [n] * batch
    return [n] + [max(1, int(n ** ((i * 0.6180339887498949) % 1.0 * 0.7 + 0.3))) for i in range(1, batch)]


def _members(case):
    """Per sequence of a "shared" case: (group, tokens shared, tokens in all)."""
    out = []
    for g in range(case["groups"]):
        p = max(PAGE, case["prefix"] - 131 * g)
        for m in range(case["members"]):
            out.append((g, p, p + 1 + (case["rest"] * (7 * m + 3 * g + 1)) % (case["rest"] + 1)))
    return out


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _row_of(pos, ring, keep):
    """The cache row of a position: its own, or behind the kept pages a ring of rows."""
    kept = _pages(keep) * PAGE
    if not ring:
        return pos
    return torch.where(pos >= kept, kept + (pos - kept) % ring, pos)


def _seen(pos, mask, window, keep):
    """How many positions the token at `pos` sees: (the first of the near ones, how many kept ones before it)."""
    if not window:
        return 0, 0
    lo = pos - pos % window if mask == "chunk" else max(0, pos - window + 1)
    return lo, min(keep, lo)


# ---------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _keys(gen, *shape):
    """Rows as a key projection gives them: a few channels are larger."""
    x = torch.randn(*shape, generator=gen, device="cuda")
    wide = 1.0 + 7.0 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.03).float()
    return x * wide


def _codes(x):
    """(e4m3 codes as bytes, biased exponents) of bfloat16 rows [..., hd]."""
    x = x.float()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)                                  # top = m 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(top > 0, e, -126).clamp(min=-126)
    y = torch.where(fine, x * torch.exp2(-e.float())[..., None], float("nan"))
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _cache(gen, n_pages, nkv, hd, bits):
    """Random pages [n_pages, nkv, 64, hd] of keys and values: bfloat16, or codes and exponents."""
    out = {}
    for name in ("k", "v"):
        rows = (_keys if name == "k" else lambda g, *s: torch.randn(*s, generator=g, device="cuda"))(gen, n_pages, nkv, PAGE, hd)
        rows = rows.to(torch.bfloat16)
        if bits == 8:
            out[name], out[name + "_exp"] = _codes(rows)
        else:
            out[name] = rows
    return out


def _take(gen, counts, width):
    """A page table [sequences, width] of pages in no order, -1 behind a sequence's pages; and how many pages there are."""
    total = sum(counts)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    return table, total


def _dirty(state, gen, counts, rows):
    """What lies behind a sequence's last row in its last page: in 8 bits any byte, NaN among them."""
    if "k_exp" not in state:
        return
    for i, (n, r) in enumerate(zip(counts, rows)):
        if r % PAGE and n:
            p = int(state["table_host"][i][n - 1])
            for name in ("k", "v"):
                left = state[name][p, :, r % PAGE:]
                left.copy_(torch.randint(0, 256, tuple(left.shape), generator=gen, device="cuda", dtype=torch.uint8))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = _gen(seed)
    nkv, hd, nq = case["nkv"], case["hd"], case["nkv"] * case["group"]
    s = {"case": case}
    if case["op"] == "store":
        new, before = ([int(t) for t in case[k].split()] for k in ("new", "before"))
        after = [a + b for a, b in zip(new, before)]
        ring = _pages(case["window"]) * PAGE if case["window"] else 0
        kept = _pages(case["keep"]) * PAGE if ring else 0
        counts = [_pages(min(n, kept + ring) if ring else n) for n in after]
        s["table"], total = _take(gen, counts, max(counts))
        s["qkv"] = torch.cat([_keys(gen, sum(new), (nq + nkv) * hd), torch.randn(sum(new), nkv * hd, generator=gen, device="cuda")], 1).to(torch.bfloat16)
        for name in ("k", "v"):
            s[name] = torch.zeros(total, nkv, PAGE, hd, dtype=torch.uint8, device="cuda")
            s[name + "_exp"] = torch.zeros(total, nkv, PAGE, dtype=torch.uint8, device="cuda")
        s["ring"], s["lens"] = ring, after
        s["positions"] = _ints([p for a, b in zip(new, before) for p in range(b, b + a)])
        s["seq_of"] = _ints([i for i, a in enumerate(new) for _ in range(a)])
        s["slots"], s["len_after"] = _ints(list(range(len(new)))), _ints(after)
        starts = [0]
        for a in new:
            starts.append(starts[-1] + a)
        s["starts"], s["new"] = _ints(starts), new
    else:
        if case["op"] == "decode":
            lens = _lengths(case["tokens"], case["batch"], case["ragged"])
            ring = _pages(case["window"]) * PAGE if case["window"] else 0
            kept = _pages(case["keep"]) * PAGE if ring else 0
            rows = [min(n, kept + ring) if ring else n for n in lens]
            counts = [_pages(r) for r in rows]
            table, total = _take(gen, counts, max(counts))
            bits = 8
            whole = [r if not ring or n <= kept + ring else 0 for n, r in zip(lens, rows)]     # (a full ring has no rest)
        else:
            who = _members(case)
            lens, ring, bits = [n for _, _, n in who], 0, case["bits"]
            lead = [next(j for j, w in enumerate(who) if w[0] == g) for g, _, _ in who]
            pages = [p // PAGE for _, p, _ in who]
            counts = [_pages(n) for n in lens]
            own_pages = [c if lead[i] == i else c - pages[i] for i, c in enumerate(counts)]
            table, total = _take(gen, own_pages, max(counts))
            for i, c in enumerate(counts):
                if lead[i] != i:
                    table[i, pages[i]:c] = table[i, :c - pages[i]].clone()
                    table[i, :pages[i]] = table[lead[i], :pages[i]]
            s["lead"], s["pages"], s["most"] = _ints(lead), _ints(pages), max(pages)
            s["lead_host"], s["pages_host"] = lead, pages
            whole = lens
        s.update(_cache(gen, total, nkv, hd, bits))
        s["table_host"] = table.tolist()
        _dirty(s, gen, counts, whole)
        # slots in no order: sequence i's pages are row slot[i] of the table
        order = torch.randperm(len(lens), generator=gen, device="cuda")
        s["table"] = torch.empty_like(table)
        s["table"][order] = table
        s["slots"] = order.to(torch.int32)
        s["ring"], s["lens"], s["len_after"] = ring, lens, _ints(lens)
        s["q"] = (2.0 * torch.randn(len(lens), nq * hd, generator=gen, device="cuda")).to(torch.bfloat16)
        s["sinks"] = torch.randn(nq, generator=gen, device="cuda") if case["sinks"] else None
    s["rows"] = s["table"] if case["op"] == "store" else torch.tensor(s["table_host"], dtype=torch.int64, device="cuda")
    if own:
        from airframe_b200.cache import KVView
        from airframe_b200.engine import StepBatch
        from airframe_b200.parts import KVNeed
        f8 = torch.float8_e4m3fn
        window, keep = case.get("window", 0), case.get("keep", 0)
        eight = "k_exp" in s
        s["kv"] = KVView(s["k"].view(f8) if eight else s["k"], s["v"].view(f8) if eight else s["v"], s["table"], s["ring"],
                         KVNeed(nkv, hd, window or None, keep_first=keep, eight_bits=eight), keep if s["ring"] else 0,
                         k_exp=s.get("k_exp"), v_exp=s.get("v_exp"))
        B = len(s["lens"])
        if case["op"] == "store":
            T = s["positions"].numel()
            s["batch"] = StepBatch(is_prefill=case["rounded"], n_tokens=T, n_seqs=B, max_len=max(s["new"]), seq_lens=s["new"], tokens=s["positions"],
                                   positions=s["positions"], seq_of_token=s["seq_of"], slots=s["slots"], len_after=s["len_after"],
                                   seq_starts=s["starts"], want_rows=None, max_len_after=max(s["lens"]))
        else:
            rows = _ints(list(range(B + 1)))
            s["batch"] = StepBatch(is_prefill=False, n_tokens=B, n_seqs=B, max_len=1, seq_lens=[1] * B, tokens=rows[:B], positions=s["len_after"] - 1,
                                   seq_of_token=rows[:B], slots=s["slots"], len_after=s["len_after"], seq_starts=rows, want_rows=rows[:B],
                                   n_want=B, max_len_after=max(s["lens"]))
    return s


# ---------------------------------------------------------------------------------------------- a pass

def _scale(case):
    return case["hd"] ** -0.5


def run(s):
    case = s["case"]
    if case["op"] == "store":
        return _store_own(s) if own else _store_plain(s)
    if not own:
        return _attend_plain(s)
    from airframe_b200 import kernels
    nkv, hd = case["nkv"], case["hd"]
    nq = nkv * case["group"]
    out = torch.empty(len(s["lens"]), nq * hd, dtype=torch.bfloat16, device="cuda")
    s["batch"].aux.clear()              # (a pass of its own: what layers share in a step is made again)
    if case["op"] == "decode":
        kernels.attn_decode(out, s["q"], s["kv"], s["batch"], nq, nkv, hd, _scale(case), case["cap"], case["window"], mask=case["mask"], sinks=s["sinks"])
    else:
        kernels.attn_decode_shared(out, s["q"], s["kv"], s["batch"], nq, nkv, hd, _scale(case), case["cap"], s["lead"], s["pages"], s["most"], sinks=s["sinks"])
    return out


def _kept(s):
    """What a store leaves: codes as the e4m3 values they are, and the rows' biased exponents."""
    f8 = torch.float8_e4m3fn
    return {"k": s["k"].view(f8), "v": s["v"].view(f8), "k_exp": s["k_exp"], "v_exp": s["v_exp"]}


def _store_own(s):
    from airframe_b200 import kernels
    case = s["case"]
    nkv, hd = case["nkv"], case["hd"]
    out = _kept(s)
    if case["rounded"]:
        out["rounded"] = torch.empty(s["qkv"].shape[0], 2 * nkv * hd, dtype=torch.bfloat16, device="cuda")
    kernels.store_kv8(s["qkv"], s["batch"], nkv * case["group"], nkv, hd, s["kv"], rounded=out.get("rounded"))
    return out


def _stored(s):
    """(rows of the step that are stored, their pages, their rows in the page)."""
    pos, seq = s["positions"].long(), s["seq_of"].long()
    ring, keep = s["ring"], s["case"]["keep"]
    on = torch.ones_like(pos, dtype=torch.bool)
    if ring:                          # of the tokens of a step that share a ring row only the last is stored
        on = (pos < _pages(keep) * PAGE) | (pos + ring >= s["len_after"].long()[seq])
    rows = torch.nonzero(on)[:, 0]
    row = _row_of(pos[rows], ring, keep)
    return rows, s["rows"].long()[seq[rows], row // PAGE], row % PAGE


def _store_plain(s):
    case = s["case"]
    nkv, hd = case["nkv"], case["hd"]
    nq, T = nkv * case["group"], s["qkv"].shape[0]
    rows, page, at = _stored(s)
    kv = s["qkv"][:, nq * hd:].reshape(T, 2, nkv, hd)
    codes, exps = _codes(kv)
    out = _kept(s)
    for i, name in enumerate(("k", "v")):
        s[name][page, :, at] = codes[rows, i]
        s[name + "_exp"][page, :, at] = exps[rows, i]
    if case["rounded"]:
        values = codes.view(torch.float8_e4m3fn).float() * torch.exp2(exps.float() - 127.0)[..., None]
        out["rounded"] = values.to(torch.bfloat16).reshape(T, 2 * nkv * hd)
    return out


def _visible(s, i):
    """(pages, rows in them) of the positions that sequence i's new token sees."""
    case, pos = s["case"], s["lens"][i] - 1
    lo, kept = _seen(pos, case.get("mask"), case.get("window", 0), case.get("keep", 0))
    at = torch.arange(lo, pos + 1, device="cuda")
    if kept:
        at = torch.cat([torch.arange(kept, device="cuda"), at])
    row = _row_of(at, s["ring"], case.get("keep", 0))
    return s["rows"][i].long()[row // PAGE], row % PAGE


def _attend_plain(s):
    case = s["case"]
    nkv, group, hd, cap = case["nkv"], case["group"], case["hd"], case["cap"]
    out = torch.empty(len(s["lens"]), nkv * group * hd, dtype=torch.bfloat16, device="cuda")
    for i in range(len(s["lens"])):
        page, row = _visible(s, i)
        kv = []
        for name in ("k", "v"):
            rows = s[name][page, :, row]                                         # [n, nkv, hd]
            if name + "_exp" in s:
                rows = rows.view(torch.float8_e4m3fn).float() * torch.exp2(s[name + "_exp"][page, :, row].float() - 127.0)[..., None]
            kv.append(rows.float().transpose(0, 1))                              # [nkv, n, hd]
        q = s["q"][i].float().view(nkv, group, hd)
        z = (q @ kv[0].transpose(1, 2)) * _scale(case)
        if cap:
            z = cap * torch.tanh(z / cap)
        top = z.amax(-1, keepdim=True)
        sink = None
        if s["sinks"] is not None:
            sink = s["sinks"].view(nkv, group, 1)
            top = torch.maximum(top, sink)
        p = torch.exp(z - top)
        total = p.sum(-1, keepdim=True)
        if sink is not None:
            total = total + torch.exp(sink - top)
        out[i] = ((p @ kv[1]) / total).reshape(-1).to(torch.bfloat16)
    return out


# ---------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    nkv, hd, nq = case["nkv"], case["hd"], case["nkv"] * case["group"]
    if case["op"] == "store":
        new, before = ([int(t) for t in case[k].split()] for k in ("new", "before"))
        T, stored = sum(new), 0
        for a, b in zip(new, before):
            stored += a
            if case["window"]:
                ring, kept = _pages(case["window"]) * PAGE, _pages(case["keep"]) * PAGE
                gone = max(0, min(a + b - ring, a + b) - max(b, kept))           # positions whose ring row a later token takes
                stored -= min(gone, a)
        read = T if case["rounded"] else stored
        return {"bytes": read * nkv * hd * 4 + stored * nkv * (hd + 1) * 2 + (T * nkv * hd * 4 if case["rounded"] else 0), "flops": read * nkv * hd * 6}
    row = 2 * nkv * (hd + 1) if case.get("bits", 8) == 8 else 4 * nkv * hd
    if case["op"] == "decode":
        lens = _lengths(case["tokens"], case["batch"], case["ragged"])
        keys = sum(n - lo + kept for n in lens for lo, kept in [_seen(n - 1, case["mask"], case["window"], case["keep"])])
        return {"bytes": keys * row + len(lens) * nq * hd * 4, "flops": 4 * keys * nq * hd}
    who = _members(case)
    read = sum(n - p // PAGE * PAGE for _, p, n in who) + sum({g: p // PAGE * PAGE for g, p, _ in who}.values())
    return {"bytes": read * row + len(who) * nq * hd * 4, "flops": 4 * sum(n for _, _, n in who) * nq * hd}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits

def _to_e4m3(y):
    """The nearest e4m3 value (ties to the even one) of numbers up to 448, by arithmetic in 64 bits."""
    size = y.abs()
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3.0)          # 2^-9 below the least normal, 2^-6
    step = torch.where(size >= step * 16.0, step * 2.0, torch.where((size < step * 8.0) & (step > 2.0 ** -9), step / 2.0, step))
    return torch.round(y / step) * step


def _quantised64(x):
    x = x.double()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / TOP))
    e = torch.where(top > TOP * torch.exp2(e), e + 1, torch.where(top <= TOP * torch.exp2(e - 1), e - 1, e)).clamp(min=-126.0)
    y = _to_e4m3(torch.where(fine, x, 0.0) * torch.exp2(-e)[..., None])
    return torch.where(fine, y, float("nan")), e


def exact(case, seed):
    s = prepare(case, seed)
    nkv, hd, nq = case["nkv"], case["hd"], case["nkv"] * case["group"]
    if case["op"] == "store":
        T = s["qkv"].shape[0]
        y, e = _quantised64(s["qkv"][:, nq * hd:].reshape(T, 2, nkv, hd))
        table, before = s["table"].tolist(), [int(t) for t in case["before"].split()]
        kept, ring = _pages(case["keep"]) * PAGE, s["ring"]
        out = {"k": torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda"), "v": torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda"),
               "k_exp": torch.zeros_like(s["k_exp"]), "v_exp": torch.zeros_like(s["v_exp"])}
        src, page, at, t = [], [], [], 0
        for i, n in enumerate(s["new"]):
            last = {}
            for p in range(before[i], before[i] + n):                      # (a later token takes an earlier one's ring row)
                last[kept + (p - kept) % ring if ring and p >= kept else p] = t
                t += 1
            for r, j in last.items():
                src.append(j)
                page.append(table[i][r // PAGE])
                at.append(r % PAGE)
        src, page, at = (torch.tensor(x, device="cuda") for x in (src, page, at))
        for j, name in enumerate(("k", "v")):
            out[name][page, :, at] = y[src, j]
            out[name + "_exp"][page, :, at] = (e[src, j] + 127).to(torch.uint8)
        if case["rounded"]:
            out["rounded"] = (y * torch.exp2(e)[..., None]).reshape(T, 2 * nkv * hd)
        return out
    values = {}
    for name in ("k", "v"):
        if name + "_exp" in s:
            c = s[name].to(torch.int32)
            field, frac = (c >> 3) & 15, (c & 7).double()
            size = torch.where(field > 0, (8.0 + frac) * torch.exp2(field.double() - 10.0), frac * 2.0 ** -9)
            size = torch.where((c & 127) == 127, float("nan"), size)
            values[name] = torch.where(c > 127, -size, size) * torch.exp2(s[name + "_exp"].double() - 127.0)[..., None]
        else:
            values[name] = s[name].double()
    out, table = [], s["table_host"]
    for i, n in enumerate(s["lens"]):
        pos = n - 1
        w, keep, ring = case.get("window", 0), case.get("keep", 0), s["ring"]
        seen = [p for p in range(n) if not w or p < keep or (p // w == pos // w if case["mask"] == "chunk" else p > pos - w)]
        kept = _pages(keep) * PAGE
        rows = [kept + (p - kept) % ring if ring and p >= kept else p for p in seen]
        page = torch.tensor([table[i][r // PAGE] for r in rows], device="cuda")
        at = torch.tensor([r % PAGE for r in rows], device="cuda")
        k, v = (values[name][page, :, at] for name in ("k", "v"))             # [n, nkv, hd]
        q = s["q"][i].double().view(nkv, case["group"], hd)
        z = torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(hd)
        if case["cap"]:
            z = case["cap"] * torch.tanh(z / case["cap"])
        if s["sinks"] is not None:
            z = torch.cat([z, s["sinks"].double().view(nkv, case["group"], 1)], -1)
        p = torch.softmax(z, -1)
        out.append(torch.einsum("hgn,nhd->hgd", p[..., :len(seen)], v).reshape(-1))
    return torch.stack(out)
