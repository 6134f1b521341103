"""Forked sequences and caches of 8 bits through the engine, the generation loop and the command line: what the cache keeps of
them, that they give what separate sequences give, and that a prompt runs once."""
import pytest
import torch

import plain_gemma2 as plain
import replay
import tiny_fiferax
import tiny_retudra
from test_cache8 import quantise, values
from test_generate_loop import FakeEngine, P, ScriptSampler
from tiny import CONFIGS, WIDE_D, make_folder
from tolerances import BF16_SPLITS, FP32_SPLITS, VS_PLAIN, rel_err

from airframe_b200.cache import CacheFull, IndexPool, PoolError, SequenceCache
from airframe_b200.config import ConfigError, config_from_dict
from airframe_b200.engine import GenerationLoop, Model, RequestError, StepEntry
from airframe_b200.parts import KVNeed, StateNeed

F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------- bookkeeping, no GPU

def test_pool_shares_and_gives_back():
    p = IndexPool(3, "page")
    a = p.take()
    p.share(a)
    p.share(a)
    assert p.owners(a) == 3 and p.n_held == 1 and p.owners(2) == 0
    p.give_back(a)
    p.give_back(a)
    assert p.is_held(a) and p.n_free == 2
    p.give_back(a)
    assert not p.is_held(a) and p.n_free == 3
    with pytest.raises(PoolError):
        p.give_back(a)
    with pytest.raises(PoolError):
        p.share(a)


def test_fork_shares_whole_pages_and_copies_the_rest():
    full, ring, eight = KVNeed(2, 16), KVNeed(1, 8, 100, keep_first=3), KVNeed(1, 64, eight_bits=True)
    c = SequenceCache([(full, None, None), (ring, StateNeed((3,)), None), (eight, (StateNeed((2, 2)), StateNeed((1,), "int32")), None)], 64 * 40, 1024,
                      torch.float32, "cpu", max_sequences=4)
    a = c.take_slot()
    c.reserve({a: 150})
    c.commit({a: 150})
    for g in c.groups.values():
        for t in (g.k, g.v):
            t.copy_(torch.randint(0, 100, t.shape).to(t.dtype))
        if g.k_exp is not None:
            g.k_exp.random_(0, 255)
            g.v_exp.random_(0, 255)
    for st in c.states.values():
        if st is not None:
            st.copy_(torch.randint(0, 9, st.shape))
    free = {n: g.pages.n_free for n, g in c.groups.items()}
    b = c.fork(a)
    assert c.length(b) == 150
    f, r, e = c.groups[full], c.groups[ring], c.groups[eight]
    assert f.held[b][:2] == f.held[a][:2] and f.held[b][2] != f.held[a][2] and f.pages.owners(f.held[a][0]) == 2
    assert not set(r.held[a]) & set(r.held[b]) and len(r.held[b]) == len(r.held[a]) == 3
    assert free[full] - f.pages.n_free == 1 and free[ring] - r.pages.n_free == 3
    for g in c.groups.values():
        assert g.table_host[b, : len(g.held[b])].tolist() == g.held[b]
        for x, y in zip(g.held[a], g.held[b]):
            assert torch.equal(g.k[:, x].float(), g.k[:, y].float()) and torch.equal(g.v[:, x].float(), g.v[:, y].float())
            if g.k_exp is not None:
                assert torch.equal(g.k_exp[:, x], g.k_exp[:, y]) and torch.equal(g.v_exp[:, x], g.v_exp[:, y])
    for st in c.states.values():
        if st is not None:
            assert torch.equal(st[a], st[b])
    # the original ends: the shared pages stay with the fork, and are free when it ends too
    c.free_slot(a)
    assert f.pages.owners(f.held[b][0]) == 1
    c.reserve({b: 193})
    c.free_slot(b)
    assert all(g.pages.n_held == 0 for g in c.groups.values()) and c.slots.n_held == 0


def test_fork_refusals_change_nothing():
    need = KVNeed(1, 8)
    c = SequenceCache([(need, None, None)], 64 * 4, 256, torch.float32, "cpu", max_sequences=3)
    a = c.take_slot()
    with pytest.raises(ValueError, match="no tokens"):
        c.fork(a)
    with pytest.raises(PoolError):
        c.fork(2)
    c.reserve({a: 200})
    c.commit({a: 200})
    assert c.groups[need].pages.n_free == 0
    with pytest.raises(CacheFull):
        c.fork(a)                                    # (the begun page needs a copy)
    assert c.slots.n_held == 1 and c.groups[need].pages.owners(c.groups[need].held[a][0]) == 1
    c.free_slot(a)
    b = c.take_slot()
    c.reserve({b: 192})
    c.commit({b: 192})
    x, y = c.fork(b), c.fork(b)                      # (whole pages only: nothing to copy)
    assert c.groups[need].pages.n_held == 3
    with pytest.raises(CacheFull):
        c.fork(b)                                    # (no slot)
    assert c.groups[need].pages.owners(c.groups[need].held[b][0]) == 3
    for s in (b, x, y):
        c.free_slot(s)
    assert c.groups[need].pages.n_held == 0


@pytest.mark.parametrize("broken", ["index_copy_", "index_select", "copy_"])
def test_a_fork_whose_copy_fails_changes_nothing(monkeypatch, broken):
    """No memory for a page's copy or a state's: the slot and the pages taken so far go back, owners and claims are as before."""
    full, ring = KVNeed(2, 16), KVNeed(1, 8, 100)
    c = SequenceCache([(full, None, None), (ring, StateNeed((3,)), None)], 64 * 40, 1024, torch.float32, "cpu", max_sequences=4)
    a = c.take_slot()
    c.reserve({a: 150})
    c.commit({a: 150})
    b = c.fork(a)
    held = {n: ([list(h) for h in g.held], g.table_host.clone(), g.pages.n_free) for n, g in c.groups.items()}
    whole, calls = getattr(torch.Tensor, broken), []

    def fails(self, *args, **kw):
        calls.append(1)
        if len(calls) == (1 if broken == "copy_" else 3):        # (of the second group of layers, or its state)
            raise torch.OutOfMemoryError("no memory")
        return whole(self, *args, **kw)

    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, broken, fails)
        with pytest.raises(torch.OutOfMemoryError):
            c.fork(a)
    assert c.slots.n_held == 2
    for n, g in c.groups.items():
        assert g.held == held[n][0] and torch.equal(g.table_host, held[n][1]) and g.pages.n_free == held[n][2]
    assert c.groups[full].pages.owners(c.groups[full].held[a][0]) == 2 and c.shared_claims([a, b])[:2] == ([0, 0], [2, 2])
    d = c.fork(a)
    for s in (a, b, d):
        c.free_slot(s)
    assert c.slots.n_held == 0 and all(g.pages.n_held == 0 for g in c.groups.values())


def test_shared_claims():
    c = SequenceCache([(KVNeed(1, 8), None, None)], 64 * 100, 2000, torch.float32, "cpu", max_sequences=8)
    a, z = c.take_slot(), c.take_slot()
    for s, n in ((a, 200), (z, 300)):
        c.reserve({s: n})
        c.commit({s: n})
    assert c.shared_claims([a, z]) is None
    b = c.fork(a)                                    # shares 3 pages with a
    c.reserve({a: 400})
    c.commit({a: 400})
    d = c.fork(a)                                    # shares 6 with a, 3 with b
    e = c.fork(b)                                    # 3
    y = c.fork(z)                                    # another family: 4
    assert c.shared_claims([a, b])[:3] == ([0, 0], [3, 3], [(2, 3)])
    assert c.shared_claims([z, d, a])[:3] == ([0, 1, 1], [0, 6, 6], [(2, 6)])
    assert c.shared_claims([y, b, -1, d, z, e, None])[:3] == ([0, 1, 2, 1, 0, 1, 6], [4, 3, 0, 3, 4, 3, 0], [(2, 4), (3, 3)])
    assert c.shared_claims([a, z]) is None
    held = c.groups[KVNeed(1, 8)].held
    assert held[a][:6] == held[d][:6] and held[a][:3] == held[b][:3] == held[e][:3]
    c.free_slot(a)                                   # its slot is another sequence's now
    n = c.take_slot()
    assert n == a and c.shared_claims([n, b, e])[:3] == ([0, 1, 1], [0, 3, 3], [(2, 3)])


def test_claims_are_of_the_groups_that_keep_all_keys():
    """Their longest rows decide; without such a group nothing is read once."""
    ring, small, large = KVNeed(1, 8, 64), KVNeed(1, 8), KVNeed(2, 8, eight_bits=True)
    for needs, want in (([ring], None), ([ring, small], small), ([large, ring, small], large)):
        c = SequenceCache([(n, None, None) for n in needs], 64 * 100, 2000, torch.float32, "cpu", max_sequences=4)
        a = c.take_slot()
        c.reserve({a: 200})
        c.commit({a: 200})
        claims = c.shared_claims([a, c.fork(a)])
        assert claims is None if want is None else claims[3] == want


def _claiming(spec, dtype=torch.bfloat16, kv_dtype=None):
    from airframe_b200.engine import Engine
    model = Model(spec, dtype, "cpu", kv_dtype)
    model.loaded = True
    return Engine(model, 64 * 600, 64 * 70, max_sequences=60)


def _family(eng, family, n, pages):
    """n forks of one sequence (the bookkeeping alone: nothing is copied)."""
    slots = [eng.take_slot() for _ in range(n)]
    for s in slots:
        eng.cache.lens[s], eng.cache._family[s] = 64 * pages, (family, pages)
    return slots


def _claims_of(spec, dtype=torch.bfloat16):
    """What an engine of this model claims for 40 forks of 64 pages each (far beyond what the rule asks for)."""
    eng = _claiming(spec, dtype)
    return eng._claims(_family(eng, 0, 40, 64))


def test_rope_stores_into_views_without_exponents(monkeypatch):
    """A view of cache pages that knows nothing of 8 bits goes to the rotation and store of the compute dtype, as it did."""
    from types import SimpleNamespace
    from airframe_b200 import kernels
    from airframe_b200.config import PartSpec
    from airframe_b200.parts import BuildContext, build_part
    rope = build_part("position", PartSpec("rope", {"theta": 10000.0, "rotary_dim": 16, "pairing": "half"}), BuildContext(torch.bfloat16, torch.device("cpu")))
    went = []
    monkeypatch.setattr(kernels, "rope_cache_write", lambda *a, **k: went.append(k["kcache"]))
    t = torch.zeros(3, dtype=torch.int32)
    batch = SimpleNamespace(positions=t, seq_of_token=t, slots=t, len_after=t, aux={})
    kv = SimpleNamespace(k="pages", v="pages", page_table=t.view(1, 3), ring_rows=0, keep_first=0)
    assert rope.encode_and_store(torch.zeros(3, 4 * 16, dtype=torch.bfloat16), batch, 2, 1, 16, kv) and went == ["pages"]


def test_padding_counts_as_rows_of_a_step():
    """More rows than the 8-bit cache's attention plans for are refused before anything changes, padding or not."""
    from airframe_b200.engine import StepError
    eng = _claiming(config_from_dict(CONFIGS["D"]).model_spec(), kv_dtype=F8)
    s = eng.take_slot()
    eng.cache.reserve({s: 64})
    eng.cache.commit({s: 64})
    held = eng.cache.pages_held()
    with pytest.raises(StepError, match="up to 2048 sequences"):
        eng.step([StepEntry(s, [1], [0])], pad_to=2049)
    assert eng.length(s) == 64 and eng.cache.pages_held() == held


def test_a_model_without_a_layer_that_shares_claims_nothing():
    """Shared steps have graphs of their own: a model whose kernels would be the ordinary ones again makes none (32 bits, head sizes
    that the shared kernels do not take, latent attention, score slopes, windows alone)."""
    import test_toy_parts
    import tiny_banitar
    from airframe_b200.config import PartSpec
    from airframe_b200.parts import unregister_part
    big = lambda size=256: config_from_dict(dict(CONFIGS["D"], max_position_embeddings=64 * 70, num_attention_heads=8, num_key_value_heads=8,
                                                head_dim=size)).model_spec()
    assert _claims_of(big()) == ([0] * 40, [64] * 40)
    assert _claims_of(big(), torch.float32) is None and _claims_of(big(96)) is None
    windows = big()
    for layer in windows.layers:
        layer.mixer.params["window"] = 128
    assert _claims_of(windows) is None
    test_toy_parts._register()
    try:
        slopes = big()
        for layer in slopes.layers:
            layer.mixer.params["position"] = PartSpec("toy_distance_slopes", {"base": 2.0, "heads": 8})
        assert _claims_of(slopes) is None
    finally:
        for kind in (("feed_forward", "toy_top1_experts"), ("position", "toy_learned_offset"), ("position", "toy_distance_slopes")):
            unregister_part(*kind)
    latent = config_from_dict(tiny_banitar.CONFIGS[next(iter(tiny_banitar.CONFIGS))]).model_spec()
    assert Model(latent, torch.bfloat16, "cpu").shared_needs() == set()


def test_shared_pages_pay_where_enough_is_read_again():
    from airframe_b200.kernels import attn_decode_shared_pays as pays
    for eight in (False, True):
        assert not pays([(2, 16)], 4, 256, eight) and not pays([(64, 1)], 8, 128, eight)
        assert pays([(32, 64)], 4, 256, eight) and pays([(8, 256)], 8, 128, eight)
        assert pays([(32, 256), (2, 16)], 4, 128, eight)
    assert pays([(3, 1024)], 4, 256) and not pays([(3, 1024)], 4, 256, True)
    assert not pays([], 4, 256)


def test_groups_that_gain_nothing_are_left_to_themselves():
    """A pair in 8 bits costs more together than apart: it neither joins nor keeps a large group from being read once."""
    from airframe_b200.kernels import attn_decode_shared_pays as pays
    assert pays([(32, 256)], 8, 128, True) and pays([(32, 256), (2, 4096)], 8, 128, True) and not pays([(2, 4096)], 8, 128, True)
    assert pays([(4, 64)], 8, 128, False, torch.bfloat16, 40, True) and not pays([(2, 4096)], 8, 128, True, torch.bfloat16, 40, True)
    eng = _claiming(config_from_dict(dict(CONFIGS["D"], max_position_embeddings=64 * 70, num_attention_heads=8, num_key_value_heads=8, head_dim=128)).model_spec(),
                    kv_dtype=F8)
    many = _family(eng, 0, 40, 64)
    pair, other = _family(eng, 1, 2, 60), _family(eng, 2, 2, 60)
    slots = [pair[0], many[0], other[0], other[1], *many[1:], pair[1]]
    lead, pages = eng._claims(slots)
    assert pages == [0, 64, 0, 0] + [64] * 39 + [0] and lead[4:-1] == [1] * 39
    assert eng._claims(pair + other) is None


def test_the_faster_way_of_pairs_and_of_many_groups():
    """Where both ways were measured, the faster one: pairs of long prompts by head size, many small groups of short ones."""
    from airframe_b200.kernels import attn_decode_shared_pays as pays
    assert not pays([(2, 512)], 4, 256) and pays([(2, 1024)], 4, 256) and pays([(2, 512)], 8, 128)
    assert not pays([(2, 16)] * 64, 4, 256) and not pays([(2, 16)] * 64, 8, 128) and not pays([(2, 64)] * 16, 4, 256) and pays([(4, 128)] * 4, 4, 256)
    assert not pays([(8, 8)] * 64, 8, 128) and not pays([(8, 24)] * 32, 8, 128, True) and not pays([(8, 32)] * 64, 4, 256, True)


def test_batches_are_planned_in_linear_time(monkeypatch):
    """A request is asked about a bounded number of times, however many are in its batch, and the batches are those that ``fits`` allows."""
    import random
    from airframe_b200.sampling import SamplingParams
    rng = random.Random(5)
    asked = []
    whole = SequenceCache.pages_wanted
    monkeypatch.setattr(SequenceCache, "pages_wanted", lambda self, *a: (asked.append(1), whole(self, *a))[1])
    monkeypatch.setattr(SequenceCache, "fits", None)
    for completions in (1, 3, 700):
        class Eng:
            cache = SequenceCache([(KVNeed(1, 8), None, None), (KVNeed(1, 8, 200, keep_first=3), None, None)], 64 * 900, 4000, torch.float32, None,
                                  max_sequences=800)
            max_context = 4000
            vocab_size = 100
        prompts = [p for p in ([1] * rng.randint(1, 700) for _ in range(2100 // completions)) for _ in range(completions)]
        params = SamplingParams(max_tokens=90)
        asked.clear()
        batches = GenerationLoop(Eng(), None).plan_batches(prompts, params, completions)
        assert len(asked) <= 2 * len(prompts)
        assert [i for b in batches for i in b] == list(range(len(prompts)))
        monkeypatch.undo()
        held = lambda b: [min(len(prompts[i]) + 89, 4000) for i in b]
        shared = lambda b: [len(prompts[i]) if i % completions and i > b[0] else 0 for i in b]
        for k, b in enumerate(batches):
            assert Eng.cache.fits(held(b), shared(b))
            if k + 1 < len(batches):                      # (and none could have taken the next request too)
                more = b + [batches[k + 1][0]]
                pages = sum((n + 63) // 64 - s // 64 for n, s in zip(held(more), shared(more)))
                assert not Eng.cache.fits(held(more), shared(more)) or pages > Eng.cache.total_pages
        monkeypatch.setattr(SequenceCache, "pages_wanted", lambda self, *a: (asked.append(1), whole(self, *a))[1])
        monkeypatch.setattr(SequenceCache, "fits", None)


def test_a_fork_of_a_ring_has_its_rows():
    """Every page of a window, the kept first tokens' and the begun page of all keys are copied, in every layer of a group."""
    ring, kept, full = KVNeed(1, 8, 192), KVNeed(2, 4, 128, keep_first=3), KVNeed(1, 8)
    c = SequenceCache([(ring, None, None), (kept, None, None), (full, None, None), (ring, None, None)], 64 * 100, 2000, torch.float32, "cpu", max_sequences=4)
    a = c.take_slot()
    c.reserve({a: 700})
    c.commit({a: 700})
    for g in c.groups.values():
        g.k.copy_(torch.randn(g.k.shape))
        g.v.copy_(torch.randn(g.v.shape))
    before = {n: (g.k.clone(), g.v.clone()) for n, g in c.groups.items()}
    b = c.fork(a)
    for n, g in c.groups.items():
        assert len(g.held[b]) == len(g.held[a]) and (n.window is None or not set(g.held[a]) & set(g.held[b]))
        for t, old in ((g.k, before[n][0]), (g.v, before[n][1])):
            assert torch.equal(t[:, g.held[b]], old[:, g.held[a]]) and torch.equal(t[:, g.held[a]], old[:, g.held[a]])
            others = [p for p in range(t.shape[1]) if p not in g.held[b]]
            assert torch.equal(t[:, others], old[:, others])


def test_batches_of_completions_share_only_what_is_in_the_batch():
    """Requests of one prompt that fall into two batches: the second batch's first one holds the whole prompt again."""
    from airframe_b200.engine import GenerationLoop
    from airframe_b200.sampling import SamplingParams

    class Eng:
        cache = SequenceCache([(KVNeed(1, 8), None, None)], 64 * 12, 2000, torch.float32, None, max_sequences=8)
        max_context = 2000
        vocab_size = 100
    loop = GenerationLoop(Eng(), None)
    params = SamplingParams(max_tokens=65)
    prompts = [[1] * 256] * 6 + [[2] * 256] * 6          # 4 whole pages each, one page of their own: 4 + 6 and 4 + 6 of 12
    got = loop.plan_batches(prompts, params, 6)
    assert got == [list(range(6)), list(range(6, 12))]
    got = loop.plan_batches([[1] * 320] * 9, params, 9)   # 5 whole pages: 5 + 7 fit
    assert got == [list(range(7)), [7, 8]]
    Eng.max_step_sequences = 3
    assert loop.plan_batches([[1] * 64] * 7, SamplingParams(max_tokens=1), 7) == [[0, 1, 2], [3, 4, 5], [6]]


@pytest.mark.gpu
def test_a_step_of_too_many_sequences_is_refused(tmp_path):
    """The 8-bit cache's attention plans for a number of sequences: more are refused before anything changes, and a loop makes batches."""
    from airframe_b200.engine import StepEntry, StepError
    from airframe_b200.sampling import SamplingParams
    cfg = dict(CONFIGS["D"], max_position_embeddings=512)
    rt = _runtime(tmp_path, cfg, "bfloat16", kv_dtype="float8_e4m3")
    eng = rt.engine
    assert eng.max_step_sequences == 2048 and _runtime(tmp_path, cfg, "bfloat16").engine.max_step_sequences is None
    eng.max_step_sequences = 2
    slots = [eng.take_slot() for _ in range(3)]
    with pytest.raises(StepError, match="up to 2 sequences"):
        eng.step([StepEntry(s, [1, 2, 3], [2]) for s in slots])
    assert [eng.length(s) for s in slots] == [0, 0, 0]
    eng.step([StepEntry(s, [1, 2, 3], [2]) for s in slots[:2]])
    eng.step([StepEntry(slots[2], [1, 2, 3], [2])])
    with pytest.raises(StepError, match="up to 2 sequences"):
        eng.decode_rows(slots, torch.ones(3, dtype=torch.int32, device=eng.device))
    assert [eng.length(s) for s in slots] == [3, 3, 3]
    for s in slots:
        eng.free_slot(s)
    outs = rt.generate([[1, 2], [3], [4, 5, 6], [7]], SamplingParams(max_tokens=3, temperature=0.0, ignore_eos=True))
    assert [len(o) for o in outs] == [3] * 4


def test_fits_counts_shared_pages_once():
    full, ring = KVNeed(1, 8), KVNeed(1, 8, 64)
    c = SequenceCache([(full, None, None), (ring, None, None)], 64 * 10, 2000, torch.float32, None, max_sequences=4)
    assert not c.fits([320, 320, 320]) and c.fits([320, 320, 320], [0, 300, 300])
    assert not c.fits([320] * 5, [0, 300, 300, 300, 300])             # (slots)


def test_refused_builds():
    spec = lambda name: config_from_dict(CONFIGS[name]).model_spec()
    with pytest.raises(ConfigError, match="8 bits"):
        Model(spec("A"), torch.bfloat16, "cpu", F8)                    # head size 16
    with pytest.raises(ConfigError, match="8 bits"):
        Model(spec("D"), torch.float32, "cpu", F8)
    with pytest.raises(ConfigError, match="kv_dtype"):
        Model(spec("D"), torch.bfloat16, "cpu", torch.float8_e5m2)
    import test_toy_parts
    from airframe_b200.config import PartSpec
    from airframe_b200.parts import unregister_part
    test_toy_parts._register()
    try:
        slopes = spec("D")
        slopes.layers[0].mixer.params["position"] = PartSpec("toy_distance_slopes", {"base": 2.0, "heads": slopes.layers[0].mixer.params["num_heads"]})
        with pytest.raises(ConfigError, match="slopes"):
            Model(slopes, torch.bfloat16, "cpu", F8)
    finally:
        for kind in (("feed_forward", "toy_top1_experts"), ("position", "toy_learned_offset"), ("position", "toy_distance_slopes")):
            unregister_part(*kind)
    needs = Model(spec("D"), torch.bfloat16, "cpu", F8).cache_needs()
    assert all(n[0].eight_bits for n in needs)
    from airframe_b200.engine.runtime import _kv_dtype
    with pytest.raises(ValueError, match="kv_dtype"):
        _kv_dtype("int8")
    with pytest.raises(ValueError, match="other head sizes, bits"):
        SequenceCache([(KVNeed(2, 64), None, None), (KVNeed(2, 64, eight_bits=True), None, 0)], 640, 512)


class ForkingEngine(FakeEngine):
    def fork(self, slot, n=1):
        new = []
        for _ in range(n):
            s = self.take_slot()
            self.lens[s] = self.lens[slot]
            self.forks.append((slot, s))
            new.append(s)
        return new

    def step(self, entries, borrow=False):
        super().step(entries, borrow)
        return torch.tensor([e.slot for e in entries])


def test_loop_runs_a_prompt_once():
    eng = ForkingEngine()
    eng.forks = []
    script = {0: [5, 9], 1: [6, 7, 8, 1], 2: [9], 3: [4, 4, 4, 4], 4: [3, 9], 5: [2, 2, 9]}
    loop = GenerationLoop(eng, ScriptSampler(script), stop_token_ids=[9])
    out = loop.generate([[1, 2, 3], [7]], P(max_tokens=4), completions=3)
    assert out == [[5], [6, 7, 8, 1], [], [4, 4, 4, 4], [3], [2, 2]]
    assert eng.steps[0] == [(0, [1, 2, 3]), (1, [7])]                   # two prompts, six sequences
    assert eng.forks == [(0, 2), (0, 3), (1, 4), (1, 5)] and eng.pool.n_held == 0
    assert loop.finish_reasons == ["stop", "length", "stop", "length", "stop", "stop"]
    with pytest.raises(RequestError):
        loop.generate([[1]], P(max_tokens=1), completions=0)


def test_loop_plans_completions():
    """Slots end a batch inside a prompt's completions: the next batch runs the prompt again."""
    eng = ForkingEngine(slots=2)
    eng.forks = []
    loop = GenerationLoop(eng, ScriptSampler({i: [i] for i in range(3)}))
    assert loop.generate([[1, 2]], P(max_tokens=1), completions=3) == [[0], [1], [2]]
    assert loop.batches_run == [[0, 1], [2]] and len(eng.steps) == 2
    # and shared pages count once where the cache says so
    eng.cache = SequenceCache([(KVNeed(1, 8), None, None)], 64 * 8, 1000, torch.float32, None, max_sequences=9)
    eng.max_context = 1000
    loop = GenerationLoop(eng, None)
    assert loop.plan_batches([[1] * 300] * 4, P(max_tokens=30), 4) == [[0, 1], [2, 3]]       # 6 pages and, the 4 whole ones shared, 2: of 8
    assert loop.plan_batches([[1] * 300] * 4, P(max_tokens=30)) == [[0], [1], [2], [3]]


# ---------------------------------------------------------------------------------------------- on the GPU

def _runtime(tmp_path, cfg, dtype, **kw):
    from airframe_b200.engine import GpuRuntime
    return GpuRuntime.load(make_folder(cfg, seed=5, store_dtype="bfloat16", root=tmp_path), dtype=dtype, max_tokens=64 * 60, **kw)


def _forked(rt, prompt, tails, graphs=True):
    """The prompt once, forked for every tail; logits at the tails' tokens, a step for all a time."""
    eng = rt.engine
    eng.use_graphs = graphs and eng.model.graph_safe
    s = eng.take_slot()
    rt.step([StepEntry(s, prompt, [])])
    slots = [s] + eng.fork(s, len(tails) - 1)
    got = [[] for _ in tails]
    for i in range(max(map(len, tails))):
        live = [r for r, t in enumerate(tails) if i < len(t)]
        logits = rt.step([StepEntry(slots[r], [tails[r][i]], [0]) for r in live])
        for k, r in enumerate(live):
            got[r].append(logits[k].cpu())
        for r, t in enumerate(tails):
            if i + 1 == len(t):
                eng.free_slot(slots[r])
    assert eng.cache.slots.n_held == 0 and all(n == 0 for n in eng.cache.pages_held().values())
    return [torch.stack(g) for g in got]


@pytest.mark.gpu
@pytest.mark.parametrize("name,dtype,kv", [("H", "bfloat16", None), ("D", "bfloat16", None), ("C", "bfloat16", None), ("A", "float32", None),
                                           ("H", "bfloat16", "float8_e4m3"), ("D", "bfloat16", "float8_e4m3")])
@pytest.mark.parametrize("graphs", [True, False])
def test_forks_go_on_like_separate_sequences(tmp_path, monkeypatch, name, dtype, kv, graphs):
    """Forks with other tails (shared pages, copied begun pages and rings; one ends early) against sequences of their own."""
    from airframe_b200 import kernels
    monkeypatch.setattr(kernels, "attn_decode_shared_pays", lambda *a: True)
    cfg = dict(CONFIGS[name], max_position_embeddings=512)
    rt = _runtime(tmp_path, cfg, dtype, kv_dtype=kv)
    shared = []
    whole = kernels.attn_decode_shared
    monkeypatch.setattr(kernels, "attn_decode_shared", lambda *a, **k: (shared.append(1), whole(*a, **k))[1])
    V = cfg["vocab_size"]
    prompt = replay.random_ids(V, 200, 3)
    tails = [replay.random_ids(V, n, 40 + n) for n in (70, 3, 70, 69)]
    got = _forked(rt, prompt, tails, graphs)
    assert shared                                              # (the layers that keep all keys went that way)
    limit = FP32_SPLITS if dtype == "float32" else BF16_SPLITS
    for t, g in zip(tails, got):
        rt.engine.use_graphs = False
        ref = replay.run_tail(rt, prompt + t, len(t))[-len(t):]
        assert rel_err(g, ref) < limit


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [None, "float8_e4m3"])
def test_the_rule_in_the_engine(tmp_path, monkeypatch, kv):
    """Twenty forks behind 45 pages go through the shared kernels by the rule's own word, three behind 2 pages and a pair beside the
    twenty do not; all of them give what sequences of their own give."""
    from airframe_b200 import kernels
    from airframe_b200.engine import GpuRuntime
    cfg = dict(CONFIGS["D"], max_position_embeddings=4096)
    rt = GpuRuntime.load(make_folder(cfg, seed=5, store_dtype="bfloat16", root=tmp_path), max_tokens=64 * 160, kv_dtype=kv)
    eng, V, shared = rt.engine, cfg["vocab_size"], []
    whole = kernels.attn_decode_shared
    monkeypatch.setattr(kernels, "attn_decode_shared", lambda *a, **k: (shared.append(a), whole(*a, **k))[1])

    def forks(prompt, n):
        s = eng.take_slot()
        rt.step([StepEntry(s, prompt, [])])
        return [s] + eng.fork(s, n - 1)

    few = replay.random_ids(V, 140, 5)
    tails = [replay.random_ids(V, 3, 100 + i) for i in range(20)]
    _forked(rt, few, tails[:3])
    assert not shared
    prompt, other = replay.random_ids(V, 64 * 45 + 10, 6), replay.random_ids(V, 64 * 3 + 5, 7)
    many, pair = forks(prompt, 20), forks(other, 2)
    slots, mine = [pair[0], *many, pair[1]], [tails[0], *tails, tails[1]]
    eng.use_graphs = True
    got = torch.stack([rt.step([StepEntry(s, [t[i]], [0]) for s, t in zip(slots, mine)]).cpu() for i in range(3)])
    assert shared
    graph = next(g for k, g in eng._graphs.items() if isinstance(k, tuple) and k[-1] == "shared")
    Bp = eng.padded_batch(22)
    pages = graph["dynamic"][5 * Bp: 5 * Bp + 22].tolist()
    assert pages == [0] + [45] * 20 + [0]
    for s in slots:
        eng.free_slot(s)
    eng.use_graphs = False
    for r, ids in ((0, other), (1, prompt), (9, prompt), (21, other)):
        ref = replay.run_tail(rt, ids + mine[r], 3)[-3:]
        assert rel_err(got[:, r], ref) < BF16_SPLITS


@pytest.mark.gpu
@pytest.mark.parametrize("make,cfg", [(tiny_fiferax.make_folder, tiny_fiferax.CONFIGS["A"]), (tiny_retudra.make_folder, tiny_retudra.CONFIGS["A"])])
def test_forks_of_sequences_with_states(tmp_path, make, cfg):
    from airframe_b200.engine import GpuRuntime
    rt = GpuRuntime.load(make(cfg, seed=5, root=tmp_path), dtype="float32", max_tokens=64 * 30)
    V = rt.model.spec.vocab_size
    prompt = replay.random_ids(V, 50, 3)
    tails = [replay.random_ids(V, n, 40 + n) for n in (12, 9)]
    for t, g in zip(tails, _forked(rt, prompt, tails)):
        assert rel_err(g, replay.run_tail(rt, prompt + t, len(t))[-len(t):]) < FP32_SPLITS


# An 8-bit value is off by half a step at most, 2^-4 of itself (e4m3): logits are held to that fraction of the largest, beside what
# the bfloat16 engine is held to; two ways of cutting the work round bfloat16 rows that differ in their last bit to neighbouring
# codes here and there: the same bound.
EIGHT_BITS = 2.0 ** -4


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["H", "D", "E", "F"])
def test_engine_with_a_cache_of_8_bits(tmp_path, monkeypatch, name):
    """Against the plain model with its keys and values rounded as the cache rounds them, and one step against single tokens."""
    cfg_d = CONFIGS[name]
    folder = make_folder(cfg_d, seed=11, store_dtype="bfloat16", root=tmp_path)
    cfg, w = plain.read_model_folder(folder)
    ids = replay.random_ids(cfg["vocab_size"], 150, 8)
    attention = plain.attention

    def rounded(q, k, v, *a):
        k, v = (values(*quantise(t.to(torch.bfloat16))).to(t.dtype) for t in (k, v))
        return attention(q, k, v, *a)

    monkeypatch.setattr(plain, "attention", rounded)
    ref = plain.logits(cfg, w, ids)
    from airframe_b200.engine import GpuRuntime
    rt = GpuRuntime.load(folder, max_tokens=64 * 24, kv_dtype="float8_e4m3")
    full = rt.engine.cache
    assert all(v.kv.k.dtype == F8 for v in full.views)
    one = replay.run_whole(rt, ids)
    assert rel_err(one, ref) < VS_PLAIN["bfloat16"] + EIGHT_BITS
    assert rel_err(replay.run_tail(rt, ids, 100), one) < EIGHT_BITS
    bits16 = GpuRuntime.load(folder, max_tokens=64 * 24)
    assert full.bytes_allocated() < 0.52 * bits16.engine.cache.bytes_allocated()


@pytest.mark.gpu
@pytest.mark.parametrize("module,name", [("banitar", "B"), ("banitar", "C"), ("banitar", "F"), ("fiferax", "B"), ("fiferax", "C"), ("retudra", "B"),
                                         ("retudra", "E"), ("zatasun", "B")])
def test_the_other_architectures_with_a_cache_of_8_bits(tmp_path, monkeypatch, module, name):
    """Attention with norms of queries and keys, gates, sinks, biases, chunks, kept first tokens, padded heads and stretched rotations, beside
    latent attention and states: a prompt in one step against single tokens, captured steps against ones kernel by kernel, and forks (shared
    pages where a layer keeps all keys).  A router may choose other experts for a token whose row differs in its last bit: a tenth of the
    positions may be such."""
    import importlib
    from airframe_b200 import kernels
    from airframe_b200.engine import GpuRuntime
    mod = importlib.import_module("tiny_" + module)
    rt = GpuRuntime.load(mod.make_folder(mod.CONFIGS[name], seed=5, root=tmp_path), max_tokens=64 * 40, kv_dtype="float8_e4m3")
    eng = rt.engine
    assert any(g.need.eight_bits for g in eng.cache.groups.values())
    ids = replay.random_ids(rt.model.spec.vocab_size, 330, 3)
    whole = replay.run_whole(rt, ids)
    tail = replay.run_tail(rt, ids, 100)

    def near(got, ref):
        each = (got.double() - ref.double()).abs().amax(1) / ref.double().abs().max()
        assert float(each.quantile(0.9)) < BF16_SPLITS

    near(tail, whole)
    eng.use_graphs = False
    assert torch.equal(replay.run_tail(rt, ids, 100), tail)
    eng.use_graphs = rt.model.graph_safe
    monkeypatch.setattr(kernels, "attn_decode_shared_pays", lambda *a: True)
    for g in _forked(rt, ids[:200], [ids[200:230], ids[200:260], ids[200:]]):
        near(g, whole[200: 200 + len(g)])


@pytest.mark.gpu
def test_completions_of_a_prompt(tmp_path, monkeypatch):
    """The same tokens as so many requests of their own (whose generators are seeded alike), greedy and drawn; prompt steps once."""
    from airframe_b200 import kernels
    from airframe_b200.engine import GpuRuntime
    from airframe_b200.sampling import SamplingParams
    monkeypatch.setattr(kernels, "attn_decode_shared_pays", lambda *a: True)
    cfg = dict(CONFIGS["A"], max_position_embeddings=512)
    rt = GpuRuntime.load(make_folder(cfg, seed=5, store_dtype="float32", root=tmp_path), dtype="float32", max_tokens=64 * 60)
    prompts = [replay.random_ids(256, 130, 1), replay.random_ids(256, 7, 2)]
    for params in (SamplingParams(max_tokens=20, temperature=0.0, repetition_penalty=1.0, ignore_eos=True),
                   SamplingParams(max_tokens=20, temperature=1.5, repetition_penalty=1.0, ignore_eos=True),
                   SamplingParams(max_tokens=20, temperature=1.5, repetition_penalty=1.2)):
        separate = rt.generate([p for p in prompts for _ in range(3)], params)
        seen = []
        got = rt.generate(prompts, params, on_token=lambda i, t: seen.append(i), completions=3)
        assert [c for of_prompt in got for c in of_prompt] == separate
        assert set(seen) <= set(range(6))
        assert rt.generate(prompts[0], params, completions=3) == separate[:3]
    assert rt.engine.cache.slots.n_held == 0 and all(n == 0 for n in rt.engine.cache.pages_held().values())


@pytest.mark.gpu
def test_command_line(tmp_path, capsys):
    from airframe_b200.cli.simple_flight import main
    folder = make_folder(WIDE_D, seed=3, store_dtype="bfloat16", root=tmp_path)
    argv = ["--model", str(folder), "2,17,3", "--max-tokens", "5", "--temperature", "0.9", "--ignore-eos"]
    assert main(argv + ["--completions", "3", "--kv-dtype", "float8_e4m3"]) == 0
    text = capsys.readouterr().out
    assert all(f"Output {i}:" in text for i in range(3)) and "15 tokens" in text
    with pytest.raises(SystemExit):
        main(argv + ["--completions", "0"])
