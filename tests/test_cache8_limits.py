"""Limits of the 8-bit cache's attention and of shared prefixes: rows and pages of odd addresses, refusals that come before any
launch, plans of calls that were refused, positions and lengths beyond a page table."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from test_cache8 import PAGE, View, bound, fill, plain_attention, step

DEV = "cuda:0"


@pytest.fixture(scope="module")
def K():
    from airframe_b200 import kernels
    return kernels


def refusal(K, entry, block):
    """What the library says to a call that it must not let reach the device (there is none here, or nothing to read at these addresses)."""
    lib = K._lib()
    lib.af_last_error.restype = ctypes.c_char_p
    assert getattr(lib, entry)(block) != 0
    return lib.af_last_error().decode()


# ---------------------------------------------------------------------------------------------- rows of queries

def decode8_block(K, **over):
    """The argument block of af_attn_decode8 for one step of two sequences, 4 heads in 2 groups of 64."""
    a = dict(out=0x10000, q=0x20000, k=0x30000, v=0x40000, k_exp=0x50000, v_exp=0x60000, table=0x70000, slots=0x80000, lens=0x90000,
             scratch=0xa0000, plan=0xb0000, sinks=0, err=0xc0000, stream=0, out_stride=256, q_stride=256, n_pages=4, max_pages=2, batch=2,
             nq=4, nkv=2, hd=64, window=0, keep=0, ring_rows=0, n_splits=4, plan_ints=1 << 20, scale=1.0, cap=0.0)
    assert set(over) <= set(a)
    return K._DECODE8.pack(*dict(a, **over).values())


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of nothing: only where there is no device to send them to")
@pytest.mark.parametrize("over,match", [
    (dict(q=0x20004), "16-byte"), (dict(q=0x20008), "16-byte"), (dict(q_stride=258), "16-byte"), (dict(q_stride=260), "16-byte"),
    (dict(k_exp=0x50008), "alignment"), (dict(v=0x40004), "alignment"), (dict(nq=3), "heads"), (dict(hd=96), "head_dim 96"),
    (dict(keep=3), "kept"), (dict(ring_rows=128), "ring"), (dict(n_splits=0), "splits"), (dict(n_pages=1 << 26), "pages")])
def test_decode8_refuses_before_a_launch(K, over, match):
    said = refusal(K, "af_attn_decode8", decode8_block(K, **over))
    assert "af_attn_decode8:" in said and match in said


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of nothing: only where there is no device to send them to")
@pytest.mark.parametrize("q,q_stride,out,out_stride", [(0x20002, 256, 0x10000, 256), (0x20000, 257, 0x10000, 256), (0x20000, 256, 0x10002, 256),
                                                       (0x20000, 256, 0x10000, 257)])
def test_decode_of_16_bits_refuses_odd_rows(K, q, q_stride, out, out_stride):
    """The 16-bit split kernel, which takes what the shared one leaves, reads queries and writes outputs in words of 4 bytes."""
    I, P, L, F = ctypes.c_int, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_float
    lib = K._lib()
    lib.af_last_error.restype = ctypes.c_char_p
    assert lib.af_attn_decode_kept(P(out), L(out_stride), P(q), L(q_stride), P(0x30000), P(0x40000), L(4), P(0x70000), I(2), P(0x80000), P(0x90000),
                                   I(2), I(4), I(2), I(64), F(1.0), F(0.0), I(0), I(0), I(0), I(4), P(0xa0000), P(0xb0000), P(0), P(0xc0000), P(0)) != 0
    assert "4-byte" in lib.af_last_error().decode()


def shared_block(K, **over):
    """The argument block of af_attn_decode_shared for the same step."""
    a = dict(out=0x10000, q=0x20000, k=0x30000, v=0x40000, k_exp=0x50000, v_exp=0x60000, table=0x70000, slots=0x80000, lens=0x90000,
             lead=0xd0000, pages=0xe0000, own=0xa0000, pre=0xf0000, plan=0xb0000, sinks=0, err=0xc0000, stream=0, out_stride=256,
             q_stride=256, n_pages=4, max_pages=2, batch=2, nq=4, nkv=2, hd=64, n_splits=4, plan_ints=1 << 20, bits=8, scale=1.0, cap=0.0)
    assert set(over) <= set(a)
    return K._SHARED.pack(*dict(a, **over).values())


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses of nothing: only where there is no device to send them to")
@pytest.mark.parametrize("over,match", [
    (dict(k_exp=0x50004), "exponents"), (dict(v_exp=0x60008), "exponents"), (dict(v_exp=0), "exponents"), (dict(q=0x20008), "16-byte"),
    (dict(q_stride=260), "16-byte"), (dict(n_splits=0), "splits"), (dict(bits=4), "bits"), (dict(hd=96), "head_dim 96"), (dict(nq=3), "heads"),
    (dict(pre=0), "scratch"), (dict(bits=16, k=0x30008), "16-byte")])
def test_shared_refuses_before_a_launch(K, over, match):
    said = refusal(K, "af_attn_decode_shared", shared_block(K, **over))
    assert "af_attn_decode_shared:" in said and match in said


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv", [(64, 4, 2), (128, 8, 2), (256, 16, 1)])
@pytest.mark.parametrize("offset,pad", [(0, 2), (2, 0), (4, 4), (1, 7), (8, 16)])
def test_decode8_rows_that_begin_anywhere(K, hd, nq, nkv, offset, pad):
    """Queries whose rows begin on 2, 4 or 8 bytes (a slice, an odd stride) give the bits that aligned rows give, and so do one
    sequence's rows and those that the shared kernels do not take."""
    lens = [130, 1, 70]
    view = View(lens, nkv, hd)
    fill(view, lens, nkv, hd)
    view.to(DEV)
    q = torch.randn(3, nq * hd, dtype=torch.bfloat16, device=DEV)
    odd = torch.empty(3, offset + nq * hd + pad, dtype=torch.bfloat16, device=DEV)[:, offset: offset + nq * hd]
    odd.copy_(q)
    want, got = torch.empty_like(q), torch.empty_like(q)
    K.attn_decode(want, q, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, 0)
    K.attn_decode(got, odd, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, 0)
    assert torch.equal(got, want)
    lead, pages = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1, 2], [0, 0, 0]))
    if offset * 2 % 16 or odd.stride(0) % 8:
        K.attn_decode_shared(got.zero_(), odd, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, lead, pages, 1)
        assert torch.equal(got, want)
    one = View([130], nkv, hd)
    fill(one, [130], nkv, hd)
    one.to(DEV)
    K.attn_decode(want[:1], q[:1], one, step(one, [130], DEV), nq, nkv, hd, 0.1, 0.0, 0)
    K.attn_decode(got[:1], odd[:1], one, step(one, [130], DEV), nq, nkv, hd, 0.1, 0.0, 0)
    assert torch.equal(got[:1], want[:1])
    K.check_device_errors(DEV)


@pytest.mark.gpu
def test_exponents_of_an_odd_address_are_refused(K):
    """Pages' exponents that do not begin on 16 bytes: an error by both attentions, and the next call works."""
    nq, nkv, hd, lens = 4, 2, 64, [200, 193]
    view = View(lens, nkv, hd)
    fill(view, lens, nkv, hd)
    view.to(DEV)
    q, out = torch.randn(2, nq * hd, dtype=torch.bfloat16, device=DEV), torch.zeros(2, nq * hd, dtype=torch.bfloat16, device=DEV)
    lead, pages = torch.arange(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    whole = view.v_exp
    room = torch.zeros(whole.numel() + 16, dtype=torch.uint8, device=DEV)
    view.v_exp = room[4: 4 + whole.numel()].view(whole.shape).copy_(whole)
    b = step(view, lens, DEV)
    with pytest.raises(K.KernelError, match="exponents"):
        K.attn_decode_shared(out, q, view, b, nq, nkv, hd, 0.1, 0.0, lead, pages, 1)
    with pytest.raises(K.KernelError, match="alignment"):
        K.attn_decode(out, q, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, 0)
    assert not out.any()
    view.v_exp = whole
    K.attn_decode_shared(out, q, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, lead, pages, 1)
    assert bool(out.any())
    K.check_device_errors(DEV)


class Pages16:
    """A layer's view of a bfloat16 cache, slots and pages in order."""

    def __init__(self, lens, nkv, hd):
        self.pages_per_seq = -(-max(lens) // PAGE)
        n = len(lens) * self.pages_per_seq
        self.k, self.v = (torch.randn(n, nkv, PAGE, hd, device=DEV).to(torch.bfloat16) for _ in range(2))
        self.page_table = torch.arange(n, dtype=torch.int32, device=DEV).view(len(lens), -1).contiguous()
        self.ring_rows, self.keep_first, self.order = 0, 0, list(range(len(lens)))


@pytest.mark.gpu
@pytest.mark.parametrize("offset,pad", [(1, 0), (0, 1), (3, 4), (2, 2)])
@pytest.mark.parametrize("lens", [[130, 1, 70], [3000, 1500, 5000]])
def test_decode_of_16_bits_with_odd_rows(K, offset, pad, lens):
    """Queries and outputs in rows that begin on 2 or 4 bytes: the aligned rows' bits, also through the shared entry."""
    nq, nkv, hd = 8, 2, 128
    view = Pages16(lens, nkv, hd)
    odd = lambda: torch.zeros(3, offset + nq * hd + pad, dtype=torch.bfloat16, device=DEV)[:, offset: offset + nq * hd]
    q = torch.randn(3, nq * hd, dtype=torch.bfloat16, device=DEV)
    want, q2, got = torch.empty_like(q), odd().copy_(q), odd()
    K.attn_decode(want, q, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, 0)
    K.attn_decode(got, q2, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, 0)
    assert torch.equal(got, want)
    lead, pages = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1, 2], [0, 0, 0]))
    got.zero_()
    K.attn_decode_shared(got, q2, view, step(view, lens, DEV), nq, nkv, hd, 0.1, 0.0, lead, pages, 1)
    assert torch.equal(got, want)
    K.check_device_errors(DEV)


# ---------------------------------------------------------------------------------------------- plans

class Refusing:
    """A library that refuses its first call and records whether each call was to make a plan."""

    def __init__(self, plan_word):
        self.made, self.word = [], plan_word

    def __getattr__(self, name):
        def entry(block):
            self.made.append(ctypes.cast(block, ctypes.POINTER(ctypes.c_longlong))[self.word] > 0)
            return -1 if len(self.made) == 1 else 0
        return (lambda: b"no") if name == "af_last_error" else entry


@pytest.mark.parametrize("shared", [False, True])
def test_a_refused_call_leaves_no_plan(K, monkeypatch, shared):
    """A step's plan is made by its first call that the library takes: one that was refused has made none for the next to read."""
    nq, nkv, hd = 4, 2, 64
    lib = Refusing(26)               # (the word that says how long a plan to make, in both blocks)
    for name, fake in (("_lib", lambda: lib), ("_here", lambda *a: 0), ("_current_device", lambda: 0), ("_raw_stream", lambda d: 0),
                       ("_error_pointer", lambda d: 0), ("_plan_ints", lambda *a: 64), ("sm_count", lambda: 148)):
        monkeypatch.setattr(K, name, fake)
    view = View([200, 200], nkv, hd).to("cpu")
    b = step(view, [200, 200], "cpu")
    q = torch.zeros(2, nq * hd, dtype=torch.bfloat16)
    out, lead, pages = torch.empty_like(q), torch.zeros(2, dtype=torch.int32), torch.full((2,), 3, dtype=torch.int32)

    def call():
        if shared:
            K.attn_decode_shared(out, q, view, b, nq, nkv, hd, 0.1, 0.0, lead, pages, 3)
        else:
            K.attn_decode8(out, q, view, b, nq, nkv, hd, 0.1, 0.0, 0)

    with pytest.raises(K.KernelError):
        call()
    assert not b.aux
    call()
    call()
    assert lib.made == [True, True, False] and len(b.aux) == 1


# ---------------------------------------------------------------------------------------------- one behind the other

@pytest.mark.gpu
@pytest.mark.parametrize("rotates", [False, True])
def test_layers_of_stores_of_many_tokens_and_attention(K, rotates):
    """A store of many tokens directly in front of the attention that reads them, in layers that share one step's plan: the bits that
    the same calls give one at a time (a store of more tokens than sequences is complete before the attention starts)."""
    nq, nkv, hd, layers, lens = 4, 2, 128, 8, [1500, 700, 64, 2000]
    T = sum(lens)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    views = [View(lens, nkv, hd).to(DEV) for _ in range(layers)]
    for v in views:                                       # (one group of layers: the same table and slots)
        v.page_table, v.order = views[0].page_table, views[0].order
    store = SimpleNamespace(positions=t([p for n in lens for p in range(n)]), seq_of_token=t([i for i, n in enumerate(lens) for _ in range(n)]),
                            slots=t(views[0].order), len_after=t(lens))
    x = [torch.randn(T, (nq + 2 * nkv) * hd, device=DEV).to(torch.bfloat16) for _ in range(layers)]
    q = torch.randn(4, nq * hd, device=DEV).to(torch.bfloat16)
    inv = torch.zeros(hd // 2, device=DEV)                # (a rotation by nothing)

    def run(apart):
        outs = torch.empty(layers, 4, nq * hd, dtype=torch.bfloat16, device=DEV)
        b = step(views[0], lens, DEV)
        for v in views:
            v.k.view(torch.uint8).zero_(), v.v.view(torch.uint8).zero_(), v.k_exp.fill_(100), v.v_exp.fill_(100)
        K.attn_decode(outs[0], q, views[0], b, nq, nkv, hd, 0.1, 0.0, 0)          # (the plan)
        for i, v in enumerate(views):
            if rotates:
                K.rope_store_kv8(x[i].clone(), store, inv, nq, nkv, hd, hd, "half", v)
            else:
                K.store_kv8(x[i], store, nq, nkv, hd, v)
            if apart:
                torch.cuda.synchronize()
            K.attn_decode(outs[i], q, v, b, nq, nkv, hd, 0.1, 0.0, 0)
        return outs

    want = run(True)
    for _ in range(30):
        assert torch.equal(run(False), want)
    K.check_device_errors(DEV)


def test_stores_say_how_many_sequences_they_are_of(K, monkeypatch):
    """The entries learn the number of sequences, by which a store of more tokens lets nothing start before it is complete."""
    said = []

    class Lib:
        def __getattr__(self, name):
            return lambda block: said.append(ctypes.cast(block, ctypes.POINTER(ctypes.c_longlong))[{"af_store_kv8": 22, "af_rope_store_kv8": 26}[name]]) or 0

    for name, fake in (("_lib", Lib), ("_here", lambda *a: 0), ("_raw_stream", lambda d: 0)):
        monkeypatch.setattr(K, name, fake)
    view = View([70, 5, 9], 2, 64).to("cpu")
    t = lambda v: torch.tensor(v, dtype=torch.int32)
    b = SimpleNamespace(positions=t([1] * 7), seq_of_token=t([0] * 7), slots=t(view.order), len_after=t([70, 5, 9]))
    x = torch.zeros(7, 8 * 64, dtype=torch.bfloat16)
    K.store_kv8(x, b, 4, 2, 64, view)
    K.rope_store_kv8(x, b, torch.ones(32), 4, 2, 64, 64, "half", view)
    assert said == [3, 3]


# ---------------------------------------------------------------------------------------------- beyond the page table

@pytest.mark.gpu
@pytest.mark.parametrize("pos", [-1, -64, -65, -1000, 128, 1000, 2 ** 31 - 1])
def test_store_of_positions_outside_the_table(K, pos):
    """A token whose position lies before the first or behind the table's last page is not stored; its neighbours are, and other
    sequences' pages stay as they were."""
    hd, nkv, nq = 128, 2, 2
    view = View([128, 128, 128], nkv, hd).to(DEV)
    order = view.order
    x = torch.randn(3, (nq + 2 * nkv) * hd, device=DEV).to(torch.bfloat16)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)

    def stored(places):
        for name in "kv":
            getattr(view, name).view(torch.uint8).copy_(view.codes[name])
            getattr(view, name + "_exp").copy_(view.exps[name])
        b = SimpleNamespace(positions=t([places[i] for i in range(3)]), seq_of_token=t([0, 1, 2]), slots=t(order), len_after=t([128] * 3))
        rounded = torch.empty(3, 2 * nkv * hd, dtype=torch.bfloat16, device=DEV)
        K.store_kv8(x, b, nq, nkv, hd, view, rounded=rounded)
        return [view.k.view(torch.uint8).clone(), view.v.view(torch.uint8).clone(), view.k_exp.clone(), view.v_exp.clone(), rounded]

    whole, got = stored([5, 70, 127]), stored([5, pos, 127])
    page = int(view.table_host[order[1], 1])
    for w, g, name in zip(whole[:4], got[:4], ("k", "v", "k", "v")):
        was = (view.codes if w.dim() == 4 else view.exps)[name].to(DEV)
        w[page, :, 6] = was[page, :, 6]                    # (what position 70 wrote)
        assert torch.equal(w, g)
    assert torch.equal(whole[4], got[4])
    inv = torch.ones(hd // 2, device=DEV)
    b = SimpleNamespace(positions=t([pos] * 3), seq_of_token=t([0, 1, 2]), slots=t(order), len_after=t([128] * 3))
    K.rope_store_kv8(x.clone(), b, inv, nq, nkv, hd, hd, "half", view)
    assert torch.equal(view.k.view(torch.uint8), got[0]) and torch.equal(view.v_exp, got[3])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_lengths_beyond_the_table(K, hd):
    """A length that the page table has no entries for reads no page of its own; the step's other sequences are as they should be."""
    nq, nkv = 4, 2
    lens = [128, 100, 128]
    view = View(lens, nkv, hd)
    held = fill(view, lens, nkv, hd)
    view.to(DEV)
    q = torch.randn(3, nq * hd).to(torch.bfloat16)
    ref, mag, big = plain_attention(q, held, lens, nq, nkv, hd, 0.1, 0.0, 0, "window", 0, None)
    ok = lambda out: bool(((out.double().cpu().view(3, nq, hd) - ref).abs() <= bound(ref, mag, big, hd))[0::2].all())
    lead, pages = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0, 1, 2], [0, 0, 0]))
    for long in (129, 64 * 60, 64 * 3000 + 7):
        out = torch.empty(3, nq * hd, dtype=torch.bfloat16, device=DEV)
        K.attn_decode(out, q.to(DEV), view, step(view, [128, long, 128], DEV), nq, nkv, hd, 0.1, 0.0, 0)
        assert ok(out)
        K.attn_decode_shared(out.zero_(), q.to(DEV), view, step(view, [128, long, 128], DEV), nq, nkv, hd, 0.1, 0.0, lead, pages, 1)
        assert ok(out)
    K.check_device_errors(DEV)


# ---------------------------------------------------------------------------------------------- what is beside the 8-bit cache

@pytest.mark.gpu
def test_heads_that_are_no_multiple_are_refused(K):
    nq, nkv, hd = 3, 2, 64
    view = View([70], nkv, hd).to(DEV)
    q = torch.zeros(1, nq * hd, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(K.KernelError, match="heads"):
        K.attn_decode(torch.empty_like(q), q, view, step(view, [70], DEV), nq, nkv, hd, 1.0, 0.0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [63, 64, 300, 1200])
def test_rotation_of_prompts_alone_has_the_bits_of_the_rotation_with_its_store(K, dtype, tokens):
    """A rotary encoding reads the step's table of cosines and sines from so many rows on whether or not it stores: the same rows as
    without the table, and as with the store."""
    from airframe_b200.config import PartSpec
    from airframe_b200.parts import BuildContext, build_part
    nq, nkv, hd = 4, 2, 128
    rope = build_part("position", PartSpec("rope", {"theta": 10000.0, "rotary_dim": hd, "pairing": "half"}), BuildContext(dtype, torch.device(DEV)))
    rope.load({})
    x = torch.randn(tokens, (nq + 2 * nkv) * hd, device=DEV).to(dtype)
    pos = torch.arange(tokens, dtype=torch.int32, device=DEV) * 7
    n_pages = -(-int(tokens) * 7 // PAGE)
    kv = SimpleNamespace(k=torch.zeros(n_pages, nkv, PAGE, hd, dtype=dtype, device=DEV), v=torch.zeros(n_pages, nkv, PAGE, hd, dtype=dtype, device=DEV),
                         page_table=torch.arange(n_pages, dtype=torch.int32, device=DEV)[None], ring_rows=0, keep_first=0)
    batch = lambda: SimpleNamespace(positions=pos, seq_of_token=torch.zeros_like(pos), slots=torch.zeros(1, dtype=torch.int32, device=DEV),
                                    len_after=torch.full((1,), tokens * 7, dtype=torch.int32, device=DEV), aux={})
    alone, stored, plain = x.clone(), x.clone(), x.clone()
    rope.encode(alone, batch(), nq, nkv, hd)
    assert rope.encode_and_store(stored, batch(), nq, nkv, hd, kv)
    K.rope_cache_write(plain, pos, rope.inv_freq, nq, nkv, hd, hd, "half")
    assert torch.equal(alone, plain) and torch.equal(alone, stored)
