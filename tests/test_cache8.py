"""The 8-bit cache: storing keys and values as e4m3 codes with a power of two a row, and the attention of single tokens
over them, against plain implementations in 64 bits."""
import math
from types import SimpleNamespace

import pytest
import torch

PAGE = 64
DEV = "cuda:0"
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def K():
    from airframe_b200 import kernels
    return kernels


# ---------------------------------------------------------------------------------------------- the format, in 64 bits

def e4m3_table():
    """The 256 code values, from the format's definition."""
    v = []
    for c in range(256):
        f, m = (c >> 3) & 15, c & 7
        x = math.nan if c & 127 == 127 else (8 + m) * 2.0 ** (f - 10) if f else m * 2.0 ** -9
        v.append(-x if c > 127 else x)
    return torch.tensor(v, dtype=torch.float64)


def quantise(x):
    """(codes uint8, biased exponents uint8) of rows x [..., hd] by search among the codes: the nearest, ties to the even code."""
    x = x.double()
    fine = torch.isfinite(x)
    top = torch.where(fine, x.abs(), 0.0).amax(-1)
    e = torch.full_like(top, -126.0)
    for _ in range(400):                                          # the least e with top <= 448 * 2^e
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    y = torch.where(fine, x, 0.0) * torch.exp2(-e)[..., None]
    grid = e4m3_table()[:127]                                     # 0 .. 448, ascending
    hi = torch.searchsorted(grid, y.abs()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y.abs(), y.abs() - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(torch.signbit(x), code + 128, code)
    code = torch.where(fine, code, 127)
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, exps):
    return e4m3_table()[codes.long()] * torch.exp2(exps.double() - 127.0)[..., None]


def test_format_against_torch():
    """The plain format agrees with torch's own conversion (on the CPU)."""
    assert torch.equal(e4m3_table()[:127].float(), torch.arange(127, dtype=torch.uint8).view(F8).float())
    x = torch.randn(64, 128).to(torch.bfloat16)
    codes, exps = quantise(x)
    y = x.float() * torch.exp2(127.0 - exps.float())[..., None]
    assert torch.equal(codes, y.to(F8).view(torch.uint8))
    assert float(y.abs().max()) <= 448.0 and float(y.abs().amax(-1).min()) > 224.0


def pages_for(n):
    return (n + PAGE - 1) // PAGE


def cache_row(pos, ring, keep):
    kept = pages_for(keep) * PAGE
    return kept + (pos - kept) % ring if ring and pos >= kept else pos


class View:
    """A layer's view of an 8-bit cache of its own: pages in no order, slots in no order, bytes of any value behind the ends."""

    def __init__(self, lens, nkv, hd, ring=0, keep=0, spare=2, extra_pages=0):
        kept = pages_for(keep) * PAGE if ring else 0
        counts = [pages_for(min(n, kept + ring) if ring else n) for n in lens]
        n_slots = len(lens) + spare
        self.order = torch.randperm(n_slots)[: len(lens)].tolist()
        n = sum(counts) + 3 + extra_pages
        free = torch.randperm(n).tolist()
        table = torch.full((n_slots, max([1, *counts])), -1, dtype=torch.int32)
        for slot, c in zip(self.order, counts):
            table[slot, :c] = torch.tensor([free.pop() for _ in range(c)], dtype=torch.int32)
        self.table_host = table
        self.codes = {k: torch.randint(0, 256, (n, nkv, PAGE, hd), dtype=torch.uint8) for k in "kv"}
        self.exps = {k: torch.randint(100, 140, (n, nkv, PAGE), dtype=torch.uint8) for k in "kv"}
        self.ring_rows, self.keep_first, self.n_slots = ring, keep if ring else 0, n_slots

    def put(self, i, pos, name, codes, exps):
        r = cache_row(pos, self.ring_rows, self.keep_first)
        page = int(self.table_host[self.order[i], r // PAGE])
        self.codes[name][page, :, r % PAGE] = codes
        self.exps[name][page, :, r % PAGE] = exps

    def to(self, dev):
        self.page_table = self.table_host.to(dev)
        self.k, self.v = (self.codes[n].to(dev).view(F8) for n in "kv")
        self.k_exp, self.v_exp = (self.exps[n].to(dev) for n in "kv")
        return self


def step(view, lens, dev, most=None, pad=0):
    slots = torch.tensor(view.order + [-1] * pad, dtype=torch.int32, device=dev)
    return SimpleNamespace(n_seqs=len(lens) + pad, slots=slots, len_after=torch.tensor(list(lens) + [0] * pad, dtype=torch.int32, device=dev),
                           max_len_after=most or max(lens), aux={})


# ---------------------------------------------------------------------------------------------- storing

def store_batch(view, before, new, dev):
    pos = [b + i for b, n in zip(before, new) for i in range(n)]
    seq = [i for i, n in enumerate(new) for _ in range(n)]
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    return SimpleNamespace(positions=t(pos), seq_of_token=t(seq), slots=t(view.order), len_after=t([b + n for b, n in zip(before, new)]))


def hard_rows(T, width):
    """Rows with large and small values, zeros, borders between codes, infinities and NaN."""
    x = torch.randn(T, width) * torch.exp2(torch.randint(-20, 20, (T, 1)).float())
    x[::5] = torch.randint(-480, 481, x[::5].shape).float() / 16          # many ties between codes
    if T > 3:
        x[3, ::7] = 0.0
        x[1] = 0.0
        x[2, 5], x[2, 70], x[2, 150] = math.inf, -math.inf, math.nan
    return x.to(torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv,before,new,ring,keep", [
    (256, 8, 4, [0, 0, 0], [1, 65, 130], 0, 0),
    (256, 2, 1, [700, 63, 64], [1, 1, 1], 0, 0),
    (128, 3, 3, [0, 0], [500, 64], 128, 0),
    (64, 5, 5, [0, 0], [333, 40], 128, 70),
    (64, 4, 1, [127, 128, 300], [1, 1, 1], 128, 3),
])
@pytest.mark.parametrize("rounded", [False, True])
def test_store(K, hd, nq, nkv, before, new, ring, keep, rounded):
    """Codes, exponents and rounded rows are exactly the format's; what no token of the step takes stays as it was."""
    after = [b + n for b, n in zip(before, new)]
    view = View(after, nkv, hd, ring, keep)
    T = sum(new)
    x = hard_rows(T, (nq + 2 * nkv) * hd)
    wide = torch.full((T, x.shape[1] + 24), 7.0, dtype=torch.bfloat16, device=DEV)       # (rows of a wider tensor)
    wide[:, : x.shape[1]] = x.to(DEV)
    codes, exps = quantise(x[:, nq * hd:].view(T, 2, nkv, hd))
    want = View.__new__(View)
    want.__dict__.update(view.__dict__)
    want.codes, want.exps = ({n: t.clone() for n, t in d.items()} for d in (view.codes, view.exps))
    t = 0
    for i, (b, n) in enumerate(zip(before, new)):
        for p in range(b, b + n):                            # (a later token takes an earlier one's ring row)
            for j, name in enumerate("kv"):
                want.put(i, p, name, codes[t, j], exps[t, j])
            t += 1
    view.to(DEV)
    back = torch.full((T, 2 * nkv * hd + 8), -5.0, dtype=torch.bfloat16, device=DEV)
    K.store_kv8(wide[:, : x.shape[1]], store_batch(view, before, new, DEV), nq, nkv, hd, view,
                rounded=back[:, : 2 * nkv * hd] if rounded else None)
    assert torch.equal(view.k.view(torch.uint8).cpu(), want.codes["k"]) and torch.equal(view.v.view(torch.uint8).cpu(), want.codes["v"])
    assert torch.equal(view.k_exp.cpu(), want.exps["k"]) and torch.equal(view.v_exp.cpu(), want.exps["v"])
    if rounded:
        got = back[:, : 2 * nkv * hd].double().cpu().view(T, 2, nkv, hd)
        assert torch.equal(got.nan_to_num(123.0), values(codes, exps).nan_to_num(123.0))
        assert bool((back[:, 2 * nkv * hd:] == -5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv", [(64, 3, 3), (128, 8, 2), (256, 8, 4)])
@pytest.mark.parametrize("rot,pairing", [(1.0, "half"), (1.0, "adjacent"), (0.25, "half"), (0.0, "half")])
@pytest.mark.parametrize("splits", [0, 1, 19])
def test_rotate_and_store(K, hd, nq, nkv, rot, pairing, splits):
    """One kernel gives the rows, codes and exponents that the rotation and the store give, to the bit: a ring with kept tokens, padding
    rows, rows of zeros and of infinities."""
    before, ring, keep = [0, 63, 64, 700, 129, 5, 8], 192, 5
    lens = [n + 1 for n in before]
    rot_dim = int(hd * rot) // 2 * 2
    width = (nq + 2 * nkv) * hd
    src = hard_rows(len(lens) + 2, width).to(DEV)
    parts = (src.float()[None] * torch.rand(splits, 1, 1, device=DEV)).contiguous() if splits else None
    inv = (10000.0 ** (-torch.arange(rot_dim // 2).float() / max(1, rot_dim // 2))).to(DEV)
    got = []
    for fused in (False, True):
        torch.manual_seed(3)
        view = View(lens, nkv, hd, ring, keep)
        b = store_batch(view, before, [1] * len(lens), DEV)
        pad = lambda t, v: torch.cat([t, torch.full((2,), v, dtype=torch.int32, device=DEV)])
        b.positions, b.slots, b.len_after = pad(b.positions, 0), pad(b.slots, -1), pad(b.len_after, 0)
        b.seq_of_token = torch.arange(len(lens) + 2, dtype=torch.int32, device=DEV)
        view.to(DEV)
        wide = torch.full((len(lens) + 2, width + 8), 7.0, dtype=torch.bfloat16, device=DEV)
        qkv = wide[:, :width]
        if not splits:
            qkv.copy_(src)
        if fused:
            K.rope_store_kv8(qkv, b, inv, nq, nkv, hd, rot_dim, pairing, view, parts=parts)
        else:
            K.rope_cache_write(qkv, b.positions, inv, nq, nkv, hd, rot_dim, pairing, parts=parts)
            K.store_kv8(qkv, b, nq, nkv, hd, view)
        got.append([wide.view(torch.int16), *(t.view(torch.uint8) for t in (view.k, view.v, view.k_exp, view.v_exp))])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    K.check_device_errors(DEV)


@pytest.mark.gpu
def test_store_extremes(K):
    """The largest and the smallest bfloat16 values: no code overflows, exponents stay in range."""
    hd, nkv = 64, 1
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    rows = torch.zeros(6, 3 * hd)
    rows[0, 64:], rows[1, 64:], rows[2, 64:130] = big, tiny, -big
    rows[3, 64:] = torch.linspace(-448, 448, 128)
    rows[4, 64], rows[5, 64] = 449.0, 448.0
    x = rows.to(torch.bfloat16)
    view = View([6], nkv, hd)
    view.to(DEV)
    K.store_kv8(x.to(DEV), store_batch(view, [0], [6], DEV), 1, nkv, hd, view)
    codes, exps = quantise(x[:, hd:].view(6, 2, nkv, hd))
    page = int(view.table_host[view.order[0], 0])
    for j, (c, e) in enumerate(((view.k, view.k_exp), (view.v, view.v_exp))):
        assert torch.equal(c.view(torch.uint8).cpu()[page, :, :6], codes[:, j].transpose(0, 1))
        assert torch.equal(e.cpu()[page, :, :6], exps[:, j].transpose(0, 1))


@pytest.mark.gpu
def test_store_leaves_padding_and_bad_pages(K):
    """Padding rows (slot -1) and tokens whose page-table entry is no page are not stored."""
    hd, nkv = 128, 2
    view = View([10, 20], nkv, hd)
    view.table_host[view.order[1], 0] = -1
    view.to(DEV)
    b = store_batch(view, [9, 19], [1, 1], DEV)
    b.slots[0] = -1
    x = torch.randn(2, 6 * hd, device=DEV).to(torch.bfloat16)
    before = view.k.view(torch.uint8).clone(), view.v.view(torch.uint8).clone(), view.k_exp.clone(), view.v_exp.clone()
    K.store_kv8(x, b, 2, nkv, hd, view)
    for was, now in zip(before, (view.k.view(torch.uint8), view.v.view(torch.uint8), view.k_exp, view.v_exp)):
        assert torch.equal(was, now)


# ---------------------------------------------------------------------------------------------- attention of single tokens

def visible(pos, window, mask, keep):
    return [p for p in range(pos + 1) if not window or p < keep or (p // window == pos // window if mask == "chunk" else p > pos - window)]


def fill(view, lens, nkv, hd, k_scale=1.0, v_scale=None):
    """Random rows of every position that the cache still holds; returns per sequence {position: (k, v)} as 64-bit values."""
    out = []
    for i, n in enumerate(lens):
        lo = max(0, n - view.ring_rows) if view.ring_rows else 0
        held = sorted(set(range(min(view.keep_first, n))) | set(range(lo, n)))
        x = torch.randn(len(held), 2, nkv, hd)
        x[:, 0, :, ::17] *= 6.0
        x[:, 0] *= k_scale
        if v_scale is not None:
            x[:, 1] *= torch.exp2(torch.randint(-v_scale, v_scale + 1, (len(held), nkv, 1)).float())
        codes, exps = quantise(x.to(torch.bfloat16))
        for j, p in enumerate(held):
            view.put(i, p, "k", codes[j, 0], exps[j, 0])
            view.put(i, p, "v", codes[j, 1], exps[j, 1])
        val = values(codes, exps)
        out.append({p: val[j] for j, p in enumerate(held)})
    return out


def plain_attention(q, held, lens, nq, nkv, hd, scale, cap, window, mask, keep, sinks):
    """(outputs [B, nq, hd], sums of p |v| over the softmax's sum, the largest sum of |q k| scale) in 64 bits."""
    outs, mags, big = [], [], 0.0
    for i, n in enumerate(lens):
        if n == 0:
            outs.append(torch.zeros(nq, hd, dtype=torch.float64))
            mags.append(torch.zeros(nq, hd, dtype=torch.float64))
            continue
        kv = torch.stack([held[i][p] for p in visible(n - 1, window, mask, keep)])          # [n, 2, nkv, hd]
        qq = q[i].double().view(nkv, nq // nkv, hd)
        k, v = kv[:, 0], kv[:, 1]
        z = torch.einsum("hgd,nhd->hgn", qq, k) * scale
        big = max(big, float(torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs()).max()) * abs(scale))
        if cap:
            z = cap * torch.tanh(z / cap)
        if sinks is not None:
            z = torch.cat([z, sinks.double().view(nkv, -1, 1)], -1)
        p = torch.softmax(z, -1)[..., : kv.shape[0]]
        outs.append(torch.einsum("hgn,nhd->hgd", p, v).reshape(nq, hd))
        mags.append(torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(nq, hd))
    return torch.stack(outs), torch.stack(mags), big


def bound(ref, mag, big, hd):
    """How far a result may be off: half a step of its bfloat16 rounding (2^-8 of it) and, of the sum of p |v|, a half-precision
    or bfloat16 rounding of every weight (2^-8 at most), the weights' own error (a score's: 32-bit sums of hd products, each off by
    2^-23 of the sum of magnitudes for every 16 of them, twice for the maximum's; exponentials: 2^-20) and the 32-bit sums (2^-20)."""
    score = 2.0 * (hd / 16 + 2) * 2.0 ** -23 * big
    return ref.abs() * 2.0 ** -8 + mag * (2.0 ** -8 + 2 * score + 2.0 ** -18) + 1e-30


def check_decode(K, lens, nq, nkv, hd, cap=0.0, window=0, mask="window", keep=0, sinks=False, k_scale=1.0, v_scale=None, q_scale=2.0, pad=0,
                 gate=False):
    ring = pages_for(window) * PAGE if window else 0
    view = View(lens, nkv, hd, ring, keep)
    held = fill(view, lens, nkv, hd, k_scale, v_scale)
    view.to(DEV)
    B = len(lens)
    q = (torch.randn(B + pad, nq * hd) * q_scale).to(torch.bfloat16)
    sk = torch.randn(nq) * 2 if sinks else None
    scale = hd ** -0.5
    ref, mag, big = plain_attention(q, held, lens, nq, nkv, hd, scale, cap, window, mask, view.keep_first, sk)
    wide = torch.zeros(B + pad, nq * hd + 40, dtype=torch.bfloat16, device=DEV)            # (queries inside packed rows)
    wide[:, : nq * hd] = q.to(DEV)
    out = torch.full((B + pad, nq * hd + 8), 9.0, dtype=torch.bfloat16, device=DEV)
    logits = torch.randn(B + pad, nq, device=DEV) if gate else None
    K.attn_decode(out[:, : nq * hd], wide[:, : nq * hd], view, step(view, lens, DEV, pad=pad), nq, nkv, hd, scale, cap, window, mask=mask,
                  sinks=sk.to(DEV) if sinks else None, gate=logits)
    got = out[:B, : nq * hd].double().cpu().view(B, nq, hd)
    lim = bound(ref, mag, big, hd)
    if gate:
        s = torch.sigmoid(logits[:B].double().cpu())[..., None]
        ref, lim = ref * s, lim * s + 2.0 ** -7 * (ref * s).abs()      # (the gate rounds the row a second time)
    assert bool(((got - ref).abs() <= lim).all()), float(((got - ref).abs() / lim).max())
    assert bool((out[:, nq * hd:] == 9.0).all())
    assert bool((out[B:, : nq * hd] == 0.0).all())            # (padding rows give zeros)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 4), (3, 1), (8, 1), (12, 1), (16, 1), (40, 2)])
def test_decode_heads(K, hd, nq, nkv):
    check_decode(K, [1, 64, 65, 200, 63], nq, nkv, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [2], [64], [65], [1000], [4097], [1, 1, 1, 1, 1, 1, 1], [3000, 1, 5, 64, 700, 129, 2]])
@pytest.mark.parametrize("cap,sinks", [(0.0, False), (30.0, True)])
def test_decode_lengths(K, lens, cap, sinks):
    check_decode(K, lens, 8, 4, 128, cap=cap, sinks=sinks, pad=1)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["window", "chunk"])
@pytest.mark.parametrize("window,keep", [(1, 0), (33, 0), (64, 0), (100, 5), (128, 64), (200, 70)])
def test_decode_windows(K, mask, window, keep):
    check_decode(K, [1, 32, 33, 34, 64, 100, 101, 128, 199, 200, 201, 500, 777], 6, 2, 64, window=window, mask=mask, keep=keep, sinks=keep > 0)


@pytest.mark.gpu
def test_decode_many_sequences(K):
    """More (sequence, kv head) units than blocks; a sequence without a token among them."""
    lens = [int(x) for x in torch.randint(0, 300, (150,))]
    lens[3] = 0
    check_decode(K, lens, 4, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_more_pages_than_stages(K, hd):
    """Blocks whose segments are longer than the ring of pages in shared memory, one unit after the other, and one long unit."""
    check_decode(K, [1500 + 37 * i for i in range(30)], 16, 8, hd, window=1400)
    check_decode(K, [40000], 2, 1, hd)


@pytest.mark.gpu
def test_decode_scales(K):
    """Values whose rows differ by 2^40 in size, keys and queries of large and small size."""
    check_decode(K, [400, 90], 8, 2, 128, v_scale=20)
    check_decode(K, [300, 5], 4, 1, 256, k_scale=2.0 ** 30, q_scale=2.0 ** -30)
    check_decode(K, [300, 5], 4, 1, 64, k_scale=2.0 ** -30, q_scale=2.0 ** 31)
    check_decode(K, [300, 5], 4, 1, 64, k_scale=40.0, cap=20.0)


@pytest.mark.gpu
def test_decode_gate(K):
    check_decode(K, [300, 5, 70], 4, 2, 128, gate=True)


@pytest.mark.gpu
def test_decode_nan_reaches_its_own_sequence_only(K):
    """A NaN in a visible key makes that sequence's heads of its kv head NaN; one in a key that the window hides changes nothing."""
    lens, nq, nkv, hd = [100, 100], 4, 2, 64
    view = View(lens, nkv, hd, 64, 0)
    held = fill(view, lens, nkv, hd)
    q = torch.randn(2, nq * hd).to(torch.bfloat16)
    ref, mag, big = plain_attention(q, held, lens, nq, nkv, hd, 0.125, 0.0, 40, "window", 0, None)
    hidden, seen = 50, 80
    for name in "kv":
        page = int(view.table_host[view.order[0], hidden % 64 // PAGE])
        view.codes[name][page, :, hidden % 64, 3] = 0x7F
    view.to(DEV)
    out = torch.empty(2, nq * hd, dtype=torch.bfloat16, device=DEV)
    args = (nq, nkv, hd, 0.125, 0.0, 40)
    K.attn_decode(out, q.to(DEV), view, step(view, lens, DEV), *args)
    got = out.double().cpu().view(2, nq, hd)
    assert bool(((got - ref).abs() <= bound(ref, mag, big, hd)).all())
    page = int(view.table_host[view.order[0], 0])
    view.k.view(torch.uint8)[page, 1, seen % 64, 7] = 0xFF
    K.attn_decode(out, q.to(DEV), view, step(view, lens, DEV), *args)
    got = out.double().cpu().view(2, nq, hd)
    assert bool(torch.isnan(got[0, 2:]).all()) and bool(((got - ref).abs() <= bound(ref, mag, big, hd))[0, :2].all())
    assert bool(((got - ref).abs() <= bound(ref, mag, big, hd))[1].all())


@pytest.mark.gpu
def test_decode_far_pages(K):
    """Pages whose bytes lie beyond 2^31 from the first."""
    nq, nkv, hd, lens = 4, 2, 256, [130, 65]
    n = (1 << 31) // (nkv * PAGE * hd) + 70
    view = View(lens, nkv, hd)
    held = fill(view, lens, nkv, hd)
    shift = n - view.codes["k"].shape[0]
    view.to(DEV)
    far = {}
    for name in ("k", "v", "k_exp", "v_exp"):
        t = getattr(view, name)
        t = t.view(torch.uint8)
        far[name] = torch.zeros(n, *t.shape[1:], dtype=torch.uint8, device=DEV)
        far[name][shift:] = t
    view.k, view.v, view.k_exp, view.v_exp = far["k"].view(F8), far["v"].view(F8), far["k_exp"], far["v_exp"]
    view.page_table = torch.where(view.page_table >= 0, view.page_table + shift, view.page_table)
    q = torch.randn(2, nq * hd).to(torch.bfloat16)
    ref, mag, big = plain_attention(q, held, lens, nq, nkv, hd, 0.0625, 0.0, 0, "window", 0, None)
    out = torch.empty(2, nq * hd, dtype=torch.bfloat16, device=DEV)
    K.attn_decode(out, q.to(DEV), view, step(view, lens, DEV), nq, nkv, hd, 0.0625, 0.0, 0)
    assert bool(((out.double().cpu().view(2, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())
    # and the store reaches them
    b = store_batch(view, [129, 64], [1, 1], DEV)
    x = torch.randn(2, (nq + 2 * nkv) * hd).to(torch.bfloat16)
    K.store_kv8(x.to(DEV), b, nq, nkv, hd, view)
    codes, exps = quantise(x[:, nq * hd:].view(2, 2, nkv, hd))
    page = int(view.page_table[view.order[0], 2])
    assert page * nkv * PAGE * hd > 1 << 31
    assert torch.equal(view.k[page, :, 1].view(torch.uint8).cpu(), codes[0, 0]) and torch.equal(view.v_exp[page, :, 1].cpu(), exps[0, 1])


@pytest.mark.gpu
def test_store_then_attend_captured_and_replayed(K):
    """The two together, captured once and replayed with other lengths and tokens, on a stream of their own."""
    nq, nkv, hd, B = 8, 2, 128, 3
    view = View([200, 200, 200], nkv, hd)
    lens0 = [70, 5, 128]
    held = fill(view, lens0, nkv, hd)
    view.to(DEV)
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    b = step(view, [1] * B, DEV, most=200)
    b.positions, b.seq_of_token = pos, torch.arange(B, dtype=torch.int32, device=DEV)
    qkv = torch.zeros(B, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(B, nq * hd, dtype=torch.bfloat16, device=DEV)

    def run():
        b.aux.clear()
        K.store_kv8(qkv, b, nq, nkv, hd, view)
        K.attn_decode(out, qkv[:, : nq * hd], view, b, nq, nkv, hd, 0.1, 0.0, 0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()                       # (length 1: writes row 0, which the loop below writes again)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(B):              # put back what the warm-up wrote
        for name in "kv":
            page = int(view.table_host[view.order[i], 0])
            getattr(view, name).view(torch.uint8)[page, :, 0] = view.codes[name][page, :, 0].to(DEV)
            getattr(view, name + "_exp")[page, :, 0] = view.exps[name][page, :, 0].to(DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    lens = list(lens0)
    for _ in range(4):
        x = torch.randn(B, (nq + 2 * nkv) * hd).to(torch.bfloat16)
        codes, exps = quantise(x[:, nq * hd:].view(B, 2, nkv, hd))
        for i in range(B):
            held[i][lens[i]] = values(codes[i], exps[i])
        lens = [n + 1 for n in lens]
        qkv.copy_(x.to(DEV))
        pos.copy_(torch.tensor([n - 1 for n in lens], dtype=torch.int32))
        b.len_after.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        ref, mag, big = plain_attention(x[:, : nq * hd], held, lens, nq, nkv, hd, 0.1, 0.0, 0, "window", 0, None)
        assert bool(((out.double().cpu().view(B, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())


# ---------------------------------------------------------------------------------------------- refusals

def test_refusals(K):
    """Wrong types, shapes and layouts are refused before anything reaches the device."""
    nq, nkv, hd = 4, 2, 64
    view = View([70], nkv, hd).to("cpu")
    b = store_batch(view, [0], [70], "cpu")
    x = torch.zeros(70, (nq + 2 * nkv) * hd, dtype=torch.bfloat16)
    with pytest.raises(K.KernelError, match="bfloat16 rows"):
        K.store_kv8(x.float(), b, nq, nkv, hd, view)
    with pytest.raises(K.KernelError, match="bfloat16 rows"):
        K.store_kv8(x[:, 1:], b, nq, nkv, hd, view)
    with pytest.raises(K.KernelError, match="positions"):
        K.store_kv8(x[:5], b, nq, nkv, hd, view)
    with pytest.raises(K.KernelError, match="rounded"):
        K.store_kv8(x, b, nq, nkv, hd, view, rounded=torch.zeros(70, 3, dtype=torch.bfloat16))
    with pytest.raises(K.KernelError, match="CUDA device"):
        K.store_kv8(x, b, nq, nkv, hd, view)
    inv = torch.ones(hd // 2)
    for bad, match in ((dict(qkv=x.float()), "bfloat16 rows"), (dict(pairing="none"), "pairing"), (dict(rot_dim=32), "frequencies"),
                       (dict(qkv=x[:5]), "positions"), (dict(parts=torch.zeros(0, 70, x.shape[1])), "parts"),
                       (dict(parts=torch.zeros(2, 70, x.shape[1], dtype=torch.bfloat16)), "parts"), (dict(inv_freq=inv.double()), "inv_freq"),
                       ({}, "CUDA device")):
        args = dict(dict(qkv=x, inv_freq=inv, rot_dim=hd, pairing="half", parts=None), **bad)
        with pytest.raises(K.KernelError, match=match):
            K.rope_store_kv8(args["qkv"], b, args["inv_freq"], nq, nkv, hd, args["rot_dim"], args["pairing"], view, parts=args["parts"])
    d = step(view, [70], "cpu")
    q, out = torch.zeros(1, nq * hd, dtype=torch.bfloat16), torch.zeros(1, nq * hd, dtype=torch.bfloat16)
    with pytest.raises(K.KernelError, match="slopes"):
        K.attn_decode(out, q, view, d, nq, nkv, hd, 1.0, 0.0, 0, slopes=torch.zeros(nq))
    with pytest.raises(K.KernelError, match="keys' size"):
        K.attn_decode(out, q, view, d, nq, nkv, hd, 1.0, 0.0, 0, dv=32)
    with pytest.raises(K.KernelError, match="bfloat16 queries"):
        K.attn_decode(out.float(), q, view, d, nq, nkv, hd, 1.0, 0.0, 0)
    with pytest.raises(K.KernelError, match="sinks"):
        K.attn_decode(out, q, view, d, nq, nkv, hd, 1.0, 0.0, 0, sinks=torch.zeros(3))
    with pytest.raises(K.KernelError, match="pages must be"):
        K.attn_decode(out, q, view, d, nq, 1, hd, 1.0, 0.0, 0)
    view.k_exp = view.k_exp.float()
    with pytest.raises(K.KernelError, match="uint8 exponents"):
        K.attn_decode(out, q, view, d, nq, nkv, hd, 1.0, 0.0, 0)


@pytest.mark.gpu
def test_refusals_of_the_library(K):
    nq, nkv, hd = 4, 2, 64
    view = View([70], nkv, hd).to(DEV)
    d = step(view, [70], DEV)
    q, out = torch.zeros(1, nq * hd, dtype=torch.bfloat16, device=DEV), torch.zeros(1, nq * hd, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(K.KernelError, match="heads"):
        K.attn_decode(out, q, view, d, nq, nkv, hd, 1.0, 0.0, 0) if nq % nkv else K.attn_decode(out[:, :192], q, view, d, 3, nkv, hd, 1.0, 0.0, 0)
    odd = View([70], nkv, 96).to(DEV)
    with pytest.raises(K.KernelError, match="head_dim 96"):
        K.attn_decode(torch.zeros(1, nq * 96, dtype=torch.bfloat16, device=DEV), torch.zeros(1, nq * 96, dtype=torch.bfloat16, device=DEV), odd, d, nq, nkv,
                      96, 1.0, 0.0, 0)
    x = torch.zeros(70, (nq + 2 * nkv) * hd + 4, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(K.KernelError, match="16-byte"):
        K.store_kv8(x[:, 4:], store_batch(view, [0], [70], DEV), nq, nkv, hd, view)
    ringed = View([70], nkv, hd, 128, 0).to(DEV)
    with pytest.raises(K.KernelError, match="ring"):
        K.attn_decode(out, q, ringed, d, nq, nkv, hd, 1.0, 0.0, 300)
