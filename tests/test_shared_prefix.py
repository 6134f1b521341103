"""Decode attention of sequences that share their first cache pages, in a 16-bit and in an 8-bit cache, against plain attention
in 64 bits over every sequence's own keys."""
from types import SimpleNamespace

import pytest
import torch

from test_cache8 import DEV, F8, PAGE, bound, pages_for, plain_attention, quantise, values


@pytest.fixture(scope="module")
def K():
    from airframe_b200 import kernels
    return kernels


class Family:
    """Sequences (group, shared pages, length) over one cache: the members of a group have the group's pages in front of their own.
    A group of None shares nothing."""

    def __init__(self, seqs, nkv, hd, bits, width=0):
        self.seqs, self.bits = seqs, bits
        self.lens = [n for _, _, n in seqs]
        n_slots = len(seqs) + 2
        self.order = torch.randperm(n_slots)[: len(seqs)].tolist()
        trunk = {}
        for g, p, _ in seqs:
            if g is not None:
                trunk[g] = max(trunk.get(g, 0), p)
        total = sum(trunk.values()) + sum(pages_for(n) for n in self.lens) + 2
        free = torch.randperm(total).tolist()
        trunk = {g: [free.pop() for _ in range(p)] for g, p in trunk.items()}
        self.table = torch.full((n_slots, max([width, *(pages_for(n) for n in self.lens)])), -1, dtype=torch.int32)
        x = {k: torch.randn(total, nkv, PAGE, hd) for k in "kv"}
        x["k"][..., ::17] *= 5.0
        if bits == 8:
            x["v"] *= torch.exp2(torch.randint(-6, 7, (total, nkv, PAGE, 1)).float())
        x = {k: t.to(torch.bfloat16) for k, t in x.items()}
        held = []
        for i, (g, p, n) in enumerate(seqs):
            own = pages_for(n) - (p if g is not None else 0)
            pages = (trunk[g][:p] if g is not None else []) + [free.pop() for _ in range(own)]
            self.table[self.order[i], : len(pages)] = torch.tensor(pages, dtype=torch.int32)
            held.append(pages)
        if bits == 8:
            self.codes = {k: quantise(t) for k, t in x.items()}
            for i, pages in enumerate(held):                     # any bytes behind a sequence's end
                if self.lens[i] % PAGE:
                    for c, e in self.codes.values():
                        c[pages[-1], :, self.lens[i] % PAGE:] = torch.randint(0, 256, c[pages[-1], :, self.lens[i] % PAGE:].shape, dtype=torch.uint8)
            val = {k: values(c, e) for k, (c, e) in self.codes.items()}
        else:
            val = {k: t.double() for k, t in x.items()}
        self.held = []
        for i, pages in enumerate(held):
            kv = [torch.cat([val[k][q] for q in pages], 1)[:, : self.lens[i]] for k in "kv"]      # [nkv, n, hd]
            both = torch.stack(kv).permute(2, 0, 1, 3)
            self.held.append({p: both[p] for p in range(self.lens[i])})
        self.page_table, self.ring_rows = self.table.to(DEV), 0
        self.keep_first = 0
        if bits == 8:
            self.k, self.v = (self.codes[n][0].to(DEV).view(F8) for n in "kv")
            self.k_exp, self.v_exp = (self.codes[n][1].to(DEV) for n in "kv")
        else:
            self.k, self.v = (x[n].to(DEV) for n in "kv")

    def step(self, most=None, pad=0):
        return SimpleNamespace(n_seqs=len(self.seqs) + pad, slots=torch.tensor(self.order + [-1] * pad, dtype=torch.int32, device=DEV),
                               len_after=torch.tensor(self.lens + [0] * pad, dtype=torch.int32, device=DEV), max_len_after=most or max(self.lens), aux={})

    def lead(self, pad=0):
        """(lead, pages) of the rows, on the device."""
        first = {}
        lead, pages = [], []
        for i, (g, p, _) in enumerate(self.seqs):
            lead.append(i if g is None else first.setdefault(g, i))
            pages.append(0 if g is None else p)
        t = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        return t(lead + list(range(len(lead), len(lead) + pad))), t(pages + [0] * pad)


def check(K, seqs, nq, nkv, hd, bits, cap=0.0, sinks=False, pad=0, lead=None, pages=None, gate=False, q_scale=2.0):
    f = Family(seqs, nkv, hd, bits)
    B = len(seqs)
    q = (torch.randn(B + pad, nq * hd) * q_scale).to(torch.bfloat16)
    sk = torch.randn(nq) if sinks else None
    ref, mag, big = plain_attention(q, f.held, f.lens, nq, nkv, hd, hd ** -0.5, cap, 0, "window", 0, sk)
    l, p = f.lead(pad)
    if lead is not None:
        l = torch.tensor(lead, dtype=torch.int32, device=DEV)
    if pages is not None:
        p = torch.tensor(pages, dtype=torch.int32, device=DEV)
    out = torch.full((B + pad, nq * hd + 8), 9.0, dtype=torch.bfloat16, device=DEV)
    logits = torch.randn(B + pad, nq, device=DEV) if gate else None
    K.attn_decode_shared(out[:, : nq * hd], q.to(DEV), f, f.step(pad=pad), nq, nkv, hd, hd ** -0.5, cap, l, p, max(1, int(p.max())),
                         sinks=sk.to(DEV) if sinks else None, gate=logits)
    got = out[:B, : nq * hd].double().cpu().view(B, nq, hd)
    lim = bound(ref, mag, big, hd)
    if gate:
        s = torch.sigmoid(logits[:B].double().cpu())[..., None]
        ref, lim = ref * s, lim * s + 2.0 ** -7 * (ref * s).abs()
    assert bool(((got - ref).abs() <= lim).all()), float(((got - ref).abs() / lim).max())
    assert bool((out[:, nq * hd:] == 9.0).all()) and bool((out[B:, : nq * hd] == 0.0).all())
    K.check_device_errors(DEV)


pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("nq,nkv", [(4, 4), (8, 4), (3, 1), (24, 2)])
def test_heads(K, bits, hd, nq, nkv):
    check(K, [(0, 3, 200), (0, 3, 193), (0, 3, 300)], nq, nkv, hd, bits, pad=1)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("prefix", [1, 2, 5, 40])
@pytest.mark.parametrize("cap,sinks", [(0.0, False), (30.0, True)])
def test_prefixes(K, bits, prefix, cap, sinks):
    n = prefix * PAGE
    check(K, [(0, prefix, n + 1), (0, prefix, n + 64), (0, prefix, n + 65)], 8, 2, 128, bits, cap=cap, sinks=sinks)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("members,nq,nkv", [(16, 8, 1), (17, 8, 1), (70, 4, 2), (33, 20, 1)])
def test_many_members(K, bits, members, nq, nkv):
    """Rows of a kv head that fill a tile, pass it by a sequence, and fill several."""
    check(K, [(0, 4, 257 + 3 * i) for i in range(members)], nq, nkv, 64, bits)


@pytest.mark.parametrize("bits", [16, 8])
def test_groups(K, bits):
    """Several groups in any order, sequences of none, a group of one, an empty sequence, unequal claims inside a group."""
    seqs = [(0, 2, 129), (1, 5, 321), (None, 0, 70), (0, 2, 500), (2, 3, 400), (1, 5, 400), (None, 0, 1), (0, 2, 130), (1, 4, 300)]
    check(K, seqs, 6, 2, 128, bits, pad=3)
    check(K, seqs, 6, 2, 256, bits, cap=20.0, sinks=True)


@pytest.mark.parametrize("bits", [16, 8])
def test_many_groups(K, bits):
    """More units than blocks: blocks take several items, one after the other."""
    seqs = [(i % 40, 1 + i % 4, 300 + i) for i in range(120)]
    check(K, seqs, 16, 8, 64, bits)


@pytest.mark.parametrize("bits", [16, 8])
def test_claims_are_bounded(K, bits):
    """More pages claimed than a sequence has before its token's page, leads outside the batch, negative claims: still each
    sequence's own attention."""
    seqs = [(0, 3, 200), (0, 3, 193), (0, 3, 260)]
    check(K, seqs, 4, 2, 64, bits, pages=[100, 3, 3])
    check(K, seqs, 4, 2, 64, bits, lead=[7, -1, 2])
    check(K, seqs, 4, 2, 64, bits, pages=[-5, 3, 3])
    check(K, seqs, 4, 2, 64, bits, lead=[2, 2, 2])
    check(K, seqs, 4, 2, 64, bits, pages=[0, 0, 0])


@pytest.mark.parametrize("bits", [16, 8])
def test_gate_and_large_queries(K, bits):
    check(K, [(0, 3, 200), (0, 3, 250)], 4, 2, 128, bits, gate=True)
    check(K, [(0, 9, 600), (0, 9, 700)], 4, 1, 64, bits, q_scale=30.0)


def test_far_from_the_first_page(K):
    """Keys that grow along the prefix: the reference maximum moves again and again."""
    for bits in (16, 8):
        seqs = [(0, 30, 30 * PAGE + 5), (0, 30, 30 * PAGE + 90)]
        f = Family(seqs, 1, 128, bits)
        nq, hd = 4, 128
        q = torch.zeros(2, nq * hd)
        q[:, ::hd] = 200.0
        q = q.to(torch.bfloat16)
        ramp = torch.arange(30 * PAGE, dtype=torch.float32) / 128      # (the first channel of the key at each position)
        for page in range(30):
            pid = int(f.table[f.order[0], page])
            rows = torch.zeros(1, PAGE, hd)
            rows[0, :, 0] = ramp[page * PAGE:(page + 1) * PAGE]
            rows = rows.to(torch.bfloat16)
            if bits == 8:
                c, e = quantise(rows)
                f.k.view(torch.uint8)[pid], f.k_exp[pid] = c.to(DEV), e.to(DEV)
                val = values(c, e)
            else:
                f.k[pid] = rows.to(DEV)
                val = rows.double()
            for held in f.held:
                for r in range(PAGE):
                    held[page * PAGE + r] = torch.stack([val[:, r], held[page * PAGE + r][1]])
        ref, mag, big = plain_attention(q, f.held, f.lens, nq, 1, hd, 0.1, 0.0, 0, "window", 0, None)
        out = torch.empty(2, nq * hd, dtype=torch.bfloat16, device=DEV)
        l, p = f.lead()
        K.attn_decode_shared(out, q.to(DEV), f, f.step(), nq, 1, hd, 0.1, 0.0, l, p, 30)
        assert bool(((out.double().cpu().view(2, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_items(K, bits, hd):
    """A block's item of several pages, in which the reference maximum moves with every page, with every second one, once and never:
    20 groups of 2 with 8 kv heads are more units than SMs, so that no unit is cut."""
    pages, nq, nkv = 11, 8, 8
    f = Family([(i % 20, pages, pages * PAGE + 3 + i) for i in range(40)], nkv, hd, bits)
    q = torch.randn(40, nq * hd) * 0.1
    q[:, ::hd] = 200.0
    q = q.to(torch.bfloat16)
    for g in range(20):
        up = torch.arange(pages * PAGE).float() / 128
        ramp = (up, -up, torch.where(torch.arange(pages * PAGE) // PAGE % 2 == 0, up, -up), up * (torch.arange(pages * PAGE) // PAGE == 6))[g % 4]
        for page in range(pages):
            pid = int(f.table[f.order[g], page])
            if bits == 8:
                rows = values(f.codes["k"][0][pid], f.codes["k"][1][pid]).float()
            else:
                rows = f.k[pid].float().cpu()
            rows[..., 0] = ramp[page * PAGE:(page + 1) * PAGE]
            rows = rows.to(torch.bfloat16)
            if bits == 8:
                c, e = quantise(rows)
                f.k.view(torch.uint8)[pid], f.k_exp[pid] = c.to(DEV), e.to(DEV)
                rows = values(c, e)
            else:
                f.k[pid] = rows.to(DEV)
                rows = rows.double()
            for held in (f.held[g], f.held[g + 20]):
                for r in range(PAGE):
                    held[page * PAGE + r] = torch.stack([rows[:, r], held[page * PAGE + r][1]])
    ref, mag, big = plain_attention(q, f.held, f.lens, nq, nkv, hd, 0.1, 0.0, 0, "window", 0, None)
    out = torch.empty(40, nq * hd, dtype=torch.bfloat16, device=DEV)
    l, p = f.lead()
    K.attn_decode_shared(out, q.to(DEV), f, f.step(), nq, nkv, hd, 0.1, 0.0, l, p, pages)
    got, lim = out.double().cpu().view(40, nq, hd), bound(ref, mag, big, hd)
    assert bool(((got - ref).abs() <= lim).all()), float(((got - ref).abs() / lim).max())
    K.check_device_errors(DEV)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_and_replayed(K, bits):
    """A captured step replayed with other groups and lengths: the plan is made anew on the device."""
    nq, nkv, hd = 4, 2, 128
    f = Family([(0, 4, 300), (0, 4, 290), (1, 2, 200), (1, 2, 140)], nkv, hd, bits, width=8)
    b = f.step(most=512)
    lead, pages = f.lead()
    q = torch.zeros(4, nq * hd, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(4, nq * hd, dtype=torch.bfloat16, device=DEV)

    def run():
        b.aux.clear()
        K.attn_decode_shared(out, q, f, b, nq, nkv, hd, 0.1, 0.0, lead, pages, 8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    whole = list(f.lens)
    for lens, claim in (([300, 290, 200, 140], [4, 4, 2, 2]), ([290, 257, 129, 140], [4, 4, 2, 1]), ([300, 290, 0, 140], [3, 4, 2, 2])):
        x = torch.randn(4, nq * hd).to(torch.bfloat16)
        q.copy_(x.to(DEV))
        b.len_after.copy_(torch.tensor(lens, dtype=torch.int32))
        pages.copy_(torch.tensor(claim, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        ref, mag, big = plain_attention(x, f.held, lens, nq, nkv, hd, 0.1, 0.0, 0, "window", 0, None)
        assert bool(((out.double().cpu().view(4, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())
    assert whole == f.lens


def test_same_result_alone_and_on_another_stream(K):
    """A row's result does not depend on the run, nor on the stream."""
    for bits in (16, 8):
        f = Family([(0, 8, 600), (0, 8, 700), (0, 8, 513)], 2, 128, bits)
        q = torch.randn(3, 8 * 128).to(torch.bfloat16).to(DEV)
        l, p = f.lead()
        outs = []
        for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                out = torch.empty(3, 8 * 128, dtype=torch.bfloat16, device=DEV)
                K.attn_decode_shared(out, q, f, f.step(), 8, 2, 128, 0.1, 0.0, l, p, 8)
            torch.cuda.synchronize()
            outs.append(out)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("hd,seqs", [(64, [(i % 40, 1 + i % 4, 300 + i) for i in range(120)]), (128, [(0, 40, 3000 + i) for i in range(20)]),
                                     (256, [(i % 3, 40 + i % 3, 3000 + i) for i in range(24)])])
def test_same_result_every_time(K, bits, hd, seqs):
    """Blocks of several items, units of many items, several groups: fifty runs give the same bits."""
    f = Family(seqs, 8, hd, bits)
    q = (torch.randn(len(seqs), 16 * hd) * 2).to(torch.bfloat16).to(DEV)
    l, p = f.lead()
    first = None
    for _ in range(50):
        out = torch.empty(len(seqs), 16 * hd, dtype=torch.bfloat16, device=DEV)
        K.attn_decode_shared(out, q, f, f.step(), 16, 8, hd, 0.1, 0.0, l, p, 43)
        first = out if first is None else first
        assert torch.equal(out, first)


def test_other_paths(K):
    """Sizes that the shared kernels do not take (32 bits, odd head sizes) go to the ordinary attention; rings are refused."""
    f = Family([(0, 3, 200), (0, 3, 193)], 2, 64, 16)
    l, p = f.lead()
    q = torch.randn(2, 4 * 64).to(torch.bfloat16)
    ref, _, _ = plain_attention(q, f.held, f.lens, 4, 2, 64, 0.125, 0.0, 0, "window", 0, None)
    f.k, f.v = f.k.float(), f.v.float()
    out = torch.empty(2, 4 * 64, device=DEV)
    K.attn_decode_shared(out, q.float().to(DEV), f, f.step(), 4, 2, 64, 0.125, 0.0, l, p, 3)
    assert float((out.double().cpu().view(2, 4, 64) - ref).abs().max()) < 1e-5
    f.ring_rows = 128
    with pytest.raises(K.KernelError, match="no ring"):
        K.attn_decode_shared(out, q.float().to(DEV), f, f.step(), 4, 2, 64, 0.125, 0.0, l, p, 3)
    f.ring_rows = 0
    with pytest.raises(K.KernelError, match="lead"):
        K.attn_decode_shared(out, q.float().to(DEV), f, f.step(), 4, 2, 64, 0.125, 0.0, l[:1], p, 3)


@pytest.mark.parametrize("bits", [16, 8])
def test_two_streams_at_once(K, bits):
    """Steps of two batches (shared prefixes, and sequences on their own) that run side by side give what each gives alone."""
    jobs = []
    for hd, seqs in ((128, [(0, 20, 1400 + 9 * i) for i in range(12)]), (256, [(i % 3, 6, 500 + 31 * i) for i in range(9)])):
        nq, nkv = 8, 4
        f = Family(seqs, nkv, hd, bits)
        q = torch.randn(len(seqs), nq * hd).to(torch.bfloat16).to(DEV)
        lead, pages = f.lead()

        def run(f=f, q=q, lead=lead, pages=pages, hd=hd, most=max(p for _, p, _ in seqs)):
            outs = [torch.empty_like(q) for _ in range(3)]
            for layer in range(2):                   # (the second with the first one's plan)
                if layer == 0:
                    b = f.step()
                K.attn_decode_shared(outs[layer], q, f, b, 8, 4, hd, 0.1, 0.0, lead, pages, most)
                K.attn_decode(outs[2], q, f, b, 8, 4, hd, 0.1, 0.0, 0)
            return outs

        jobs.append((run, run(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(15):
        for run, _, stream in jobs:
            with torch.cuda.stream(stream):
                got.append(run())
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for x, y in zip(outs, jobs[i % 2][1]):
            assert torch.equal(x, y)
    K.check_device_errors(DEV)


@pytest.mark.parametrize("bits", [16, 8])
def test_far_pages(K, bits):
    """Shared pages, and the sequences' own, whose bytes lie beyond 2^32 (16 bits) and 2^31 (8 bits) from the cache's first."""
    nq, nkv, hd = 8, 4, 256
    f = Family([(0, 5, 400), (0, 5, 321), (0, 5, 350)], nkv, hd, bits)
    n = (1 << 31) // (nkv * PAGE * hd) + 70
    shift = n - f.k.shape[0]
    for name in ("k", "v", "k_exp", "v_exp") if bits == 8 else ("k", "v"):
        t = getattr(f, name)
        plain = t.view(torch.uint8) if bits == 8 else t
        far = torch.zeros(n, *t.shape[1:], dtype=plain.dtype, device=DEV)
        far[shift:] = plain
        setattr(f, name, far.view(F8) if t.dtype == F8 else far)
    f.page_table = torch.where(f.page_table >= 0, f.page_table + shift, f.page_table)
    q = torch.randn(3, nq * hd).to(torch.bfloat16)
    ref, mag, big = plain_attention(q, f.held, f.lens, nq, nkv, hd, 0.0625, 0.0, 0, "window", 0, None)
    out = torch.empty(3, nq * hd, dtype=torch.bfloat16, device=DEV)
    l, p = f.lead()
    K.attn_decode_shared(out, q.to(DEV), f, f.step(), nq, nkv, hd, 0.0625, 0.0, l, p, 5)
    assert bool(((out.double().cpu().view(3, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())
    K.check_device_errors(DEV)


@pytest.mark.parametrize("bits", [16, 8])
def test_prefix_of_what_is_not_finite(K, bits):
    """NaN in a group's shared pages reaches that group's outputs and no other's."""
    nq, nkv, hd = 4, 2, 64
    f = Family([(0, 3, 200), (1, 3, 230), (0, 3, 250), (1, 3, 199)], nkv, hd, bits)
    ref, mag, big = plain_attention(q := torch.randn(4, nq * hd).to(torch.bfloat16), f.held, f.lens, nq, nkv, hd, 0.1, 0.0, 0, "window", 0, None)
    page = int(f.table[f.order[0], 1])
    if bits == 8:
        f.v.view(torch.uint8)[page, 1, 7, 3] = 0x7f           # (a NaN code)
    else:
        f.v[page, 1, 7, 3] = float("nan")
    out = torch.empty(4, nq * hd, dtype=torch.bfloat16, device=DEV)
    l, p = f.lead()
    K.attn_decode_shared(out, q.to(DEV), f, f.step(), nq, nkv, hd, 0.1, 0.0, l, p, 3)
    got, lim = out.double().cpu().view(4, nq, hd), bound(ref, mag, big, hd)
    struck = torch.zeros(4, nq, hd, dtype=torch.bool)
    struck[0::2, nq // 2:, 3] = True                          # (the second kv head's query heads of the first group, that dim)
    assert bool(got[struck].isnan().all()) and bool(((got - ref).abs() <= lim)[~struck].all())
    K.check_device_errors(DEV)


@pytest.mark.parametrize("bits", [16, 8])
def test_many_groups_in_any_order(K, bits):
    """Hundreds of rows whose groups' members lie among one another in no order, rows alone between them: a row's place is its own."""
    nq, nkv, hd = 2, 1, 64
    rng = torch.Generator().manual_seed(3)
    groups = torch.randint(0, 60, (333,), generator=rng).tolist()
    seqs = [(g, 2, 129 + (7 * i) % 60) for i, g in enumerate(groups)]
    f = Family(seqs, nkv, hd, bits)
    q = torch.randn(len(seqs), nq * hd).to(torch.bfloat16)
    ref, mag, big = plain_attention(q, f.held, f.lens, nq, nkv, hd, 0.125, 0.0, 0, "window", 0, None)
    lead, pages = f.lead()
    out = torch.empty(len(seqs), nq * hd, dtype=torch.bfloat16, device=DEV)
    K.attn_decode_shared(out, q.to(DEV), f, f.step(), nq, nkv, hd, 0.125, 0.0, lead, pages, 2)
    assert bool(((out.double().cpu().view(-1, nq, hd) - ref).abs() <= bound(ref, mag, big, hd)).all())
    K.check_device_errors(DEV)
