"""The 8-bit cache without a GPU: the plain statement against independent ones, the cache's bookkeeping with a keep rule,
what is refused."""
import numpy as np
import pytest
import torch

import go_tinygrad_b200 as lib
import plain_e4m3 as plain
from conftest import TINY_A
from go_tinygrad_b200.cache import (Cache, CacheFull, CacheMisuse, E4M3KVView, E4M3Storage, KeepRule, KVRequest, StateRequest)
from go_tinygrad_b200.engine.schedule import RequestTooLarge, plan_batches
from go_tinygrad_b200.kernels import KernelError, ops


# ------------------------------------------------------------------ the plain statement
def test_plain_codes_are_torchs():
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.standard_normal(20000) * 10.0 ** rng.integers(-4, 3, 20000), np.arange(-448, 449) / 1.0,
                        np.arange(-64, 65) * 2.0 ** -10, [0.0, 448.0, -448.0, 464.0 - 32.0]])
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(plain.nearest(x), want.astype(np.float64))
    assert np.isnan(plain.nearest(np.array([np.inf, -np.inf, np.nan]))).all()


@pytest.mark.parametrize("most,want", [(448.0, 1.0), (448.0001, 2.0), (224.0, 0.5), (0.0, 2.0 ** -126), (1e-45, 2.0 ** -126),
                                       (3.3e38, 2.0 ** 120), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7), (2.0, 2.0 ** -7)])
def test_plain_scale(most, want):
    assert plain.needed([0.0, -most, np.nan, np.inf]) == want


def test_plain_blocks_do_not_depend_much_on_the_cut():
    """Values stored row by row and all at once: a code may round a second time where it falls below 2^-6, by half a step of
    2^-9 scales at most."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((150, 8)) * np.geomspace(1e-3, 30.0, 150)[:, None]
    whole, single = plain.Rows(8), plain.Rows(8)
    whole.append(x)
    for r in x:
        single.append(r[None])
    assert whole.scales == single.scales
    step = np.repeat(whole.scales, 64)[:150, None] * 2.0 ** -9
    near = np.maximum(np.abs(x) * 2.0 ** -4, step / 2)
    assert (np.abs(whole.values() - x) <= near * (1 + 1e-12)).all()
    assert (np.abs(single.values() - x) <= near * (1 + 2.0 ** -4) + step / 2).all()


def test_plain_choice():
    assert plain.chosen([5, 1, 1, 0, 1, 9], 4, 1) == [0, 1, 2, 5]
    assert plain.chosen([5, 1, 1, 0], 4, 1) == [0, 1, 2, 3]
    assert plain.chosen([0.0] * 6, 2, 2) == [4, 5]
    assert plain.chosen([0.0] * 6, 2, 0) == [0, 1]


# ------------------------------------------------------------------ the cache's bookkeeping
def make_cache(max_tokens=64 * 12, keep=KeepRule(100, 20), requests=None, **more):
    requests = requests or [[KVRequest(2, 16, e4m3=True)], [KVRequest(2, 16, e4m3=True)], [KVRequest(1, 32, e4m3=True)]]
    return Cache(requests, [None] * len(requests), max_tokens=max_tokens, max_slots=3, dtype=torch.bfloat16, device="cpu", kv_format="e4m3",
                 keep=keep, **more)


def test_storage_of_a_group():
    cache = make_cache()
    first = cache.groups[0].e4m3
    assert first.k.shape == (2, 12, 2, 64, 16) and first.v.shape == (2, 12, 2, 16, 64) and first.scales.shape == (2, 12, 2, 2)
    assert first.weights.shape == (2, 12, 2, 64) and first.dropped.shape == (3,)
    a, b = cache.handles[0].kv, cache.handles[1].kv
    assert a.format == "e4m3" and a.k.data_ptr() != b.k.data_ptr() and a.k.dtype == torch.float8_e4m3fn
    assert a.head_dim == 16 and a.n_kv_heads == 2 and cache.handles[2].kv.head_dim == 32
    plain_cache = Cache([[KVRequest(2, 16, e4m3=True)]], [None], max_tokens=64 * 12, max_slots=3, dtype=torch.bfloat16, device="cpu")
    assert plain_cache.handles[0].kv.format is None
    # 8 bits a value, a scale and 64 weights a block of a head: less than 3/4 of bfloat16 even at 16 channels
    assert make_cache(requests=[[KVRequest(2, 16, e4m3=True)]]).bytes() < 0.75 * plain_cache.bytes()
    without = make_cache(keep=None).groups[0].e4m3
    assert without.weights is None and without.dropped is None


def test_rows_and_positions_part_when_rows_are_evicted(monkeypatch):
    cache = make_cache()
    calls = []

    def evict(storage, slots, lengths, max_length, budget, recent, kept=None):
        calls.append((slots.tolist(), lengths.tolist(), max_length, budget, recent))
        return torch.zeros(1)
    monkeypatch.setattr(ops, "kv_evict_e4m3", evict)
    a, b = cache.open_sequence(), cache.open_sequence()
    cache.reserve_many([(a, 300), (b, 90)])
    assert cache.free_pages() == [5, 5]
    cache.advance(a, 300)
    cache.advance(b, 90)
    cache.evict_due([a, b])                                # a holds 300 >= 164, b stays
    assert calls == [([a], [300], 300, 100, 20)] * 2       # once for each group
    assert cache.length(a) == 300 and cache.held(a) == 100 and cache.held(b) == 90
    assert cache.free_pages() == [8, 8]                    # two pages hold 100 rows
    calls.clear()
    for _ in range(63):
        cache.reserve(a, cache.length(a) + 1)
        cache.advance(a, 1)
        cache.evict_due([a, b])
    assert not calls and cache.held(a) == 163 and cache.length(a) == 363 and cache.free_pages() == [7, 7]
    cache.reserve(a, 364)
    cache.advance(a, 1)
    cache.evict_due([a, b])
    assert [c[1] for c in calls] == [[164]] * 2 and cache.held(a) == 100 and cache.length(a) == 364
    assert cache.evict([b], budget=10, recent=5) and cache.held(b) == 10 and cache.length(b) == 90
    with pytest.raises(CacheMisuse, match="rolled back"):
        cache.truncate(b, 89)
    cache.truncate(b, 90)
    cache.close_sequence(a)
    cache.close_sequence(b)
    assert cache.free_pages() == [12, 12]
    assert cache.held(cache.open_sequence()) == 0


def test_sequences_longer_than_the_cache_holds():
    cache = make_cache(max_position=10 ** 6)
    assert cache.max_sequence == 10 ** 6 and cache.max_held == 64 * 12
    a = cache.open_sequence()
    with pytest.raises(CacheFull, match="768"):
        cache.reserve(a, 769)
    cache.reserve(a, 768)
    cache.advance(a, 768)
    with pytest.raises(CacheFull):
        cache.reserve(a, 769)
    short = make_cache(max_position=200, keep=KeepRule(50, 10))
    b = short.open_sequence()
    with pytest.raises(CacheFull, match="200"):
        short.reserve(b, 201)


def test_what_a_cache_refuses():
    with pytest.raises(ValueError, match="not known"):
        Cache([[KVRequest(1, 16)]], [None], max_tokens=64, dtype=torch.float32, device="cpu", kv_format="int4")
    with pytest.raises(ValueError, match="gather no attention weights"):
        Cache([[KVRequest(1, 16, e4m3=True)]], [None], max_tokens=640, dtype=torch.float32, device="cpu", keep=KeepRule(10, 5))
    with pytest.raises(ValueError, match="does not read from an e4m3 cache"):
        make_cache(requests=[[KVRequest(1, 16, e4m3=True)], [KVRequest(1, 16)]])
    with pytest.raises(ValueError, match="one size"):
        make_cache(requests=[[KVRequest(1, 16, value_dim=8, e4m3=True)]])
    with pytest.raises(ValueError, match="forget by themselves"):
        make_cache(requests=[[KVRequest(1, 16, window=64, e4m3=True)]])
    make_cache(requests=[[KVRequest(1, 16, window=64, e4m3=True)]], keep=None)
    with pytest.raises(ValueError, match="keeps up to 864"):
        make_cache(keep=KeepRule(800, 10))
    for bad in ((0, 0, 64), (10, 11, 64), (10, -1, 64), (10, 5, 0)):
        with pytest.raises(ValueError, match="keep rule"):
            KeepRule(*bad)
    cache = make_cache()
    a = cache.open_sequence()
    with pytest.raises(CacheMisuse, match="each named once"):
        cache.evict([a, a])
    with pytest.raises(CacheMisuse, match="each named once"):
        cache.evict([2])
    with pytest.raises(ValueError, match="recent"):
        cache.evict([a], budget=3, recent=4)
    assert cache.evict([]) == []
    with pytest.raises(CacheMisuse, match="keep rule"):
        make_cache(keep=None).evict([])
    stated = make_cache(requests=[[KVRequest(1, 16, e4m3=True), StateRequest("h", (4,))]])       # state of fixed size beside it
    assert stated.handles[0].state("h").shape == (3, 4)


def test_batches_of_an_evicting_cache():
    assert plan_batches([100, 100], [10000, 10000], max_tokens=512, max_batch=8, max_held=200) == [[0, 1]]
    assert plan_batches([300, 100], [10000, 10000], max_tokens=512, max_batch=8, max_held=200) == [[0], [1]]   # a prompt is held whole once
    with pytest.raises(RequestTooLarge):
        plan_batches([600], [10], max_tokens=512, max_batch=8, max_held=200)
    assert plan_batches([100], [20], max_tokens=128, max_batch=8, max_held=200) == [[0]]


# ------------------------------------------------------------------ refusals of the entry points
def view(pages=4, heads=2, dim=16, slots=3, weights=True, **swap):
    t = dict(k=torch.zeros(pages, heads, 64, dim).to(torch.float8_e4m3fn), v=torch.zeros(pages, heads, dim, 64).to(torch.float8_e4m3fn),
             scales=torch.ones(pages, 2, heads), block_table=torch.zeros(slots, 4, dtype=torch.int32),
             weights=torch.zeros(pages, heads, 64) if weights is True else None if weights is False else weights, dropped=torch.zeros(slots, dtype=torch.int32))
    t.update(swap)
    return E4M3KVView(t["k"], t["v"], t["scales"], t["block_table"], weights=t["weights"], dropped=t["dropped"])


@pytest.mark.parametrize("swap,what", [
    (dict(k=torch.zeros(4, 2, 64, 16)), "float8"),
    (dict(k=torch.zeros(4, 2, 32, 16).to(torch.float8_e4m3fn)), "keys must be"),
    (dict(v=torch.zeros(4, 2, 64, 16).to(torch.float8_e4m3fn)), "values must be"),
    (dict(scales=torch.ones(4, 2, 2, dtype=torch.float64)), "scales must be"),
    (dict(scales=torch.ones(4, 2, 3)), "scales must be"),
    (dict(weights=torch.zeros(4, 2, 32)), "weights must be"),
    (dict(k=torch.zeros(4, 2, 16, 64).to(torch.float8_e4m3fn).transpose(2, 3)), "in one piece"),
    (dict(k=torch.zeros(4 * 2 * 64 * 16 + 8).to(torch.float8_e4m3fn)[8:].view(4, 2, 64, 16)), "16-byte boundary"),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int64)), "block table"),
    (dict(block_table=torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)), "row by row"),
    (dict(dropped=torch.zeros(2, dtype=torch.int32)), "dropped"),
])
def test_a_view_refuses(swap, what):
    with pytest.raises(ValueError, match=what):
        view(**swap)


def step_tensors(lengths, dtype=torch.float32, width=8 * 16):
    n = sum(lengths)
    cu = torch.tensor([0] + list(np.cumsum(lengths)), dtype=torch.int32)
    return torch.zeros(n, width, dtype=dtype), cu, torch.arange(len(lengths), dtype=torch.int32), torch.zeros(len(lengths), dtype=torch.int32)


def test_the_store_refuses():
    kv = view()
    qkv, cu, slots, start = step_tensors([2, 1])
    q = torch.zeros(3, 4 * 16)

    def call(what, qkv=qkv, cos_sin=None, heads=4, store=2, kv=kv, cu=cu, slots=slots, start=start, longest=2, q=q, **more):
        with pytest.raises(KernelError, match=what):
            ops.kv_store_e4m3(qkv, cos_sin, heads, store, kv, cu, slots, start, longest, q, **more)
    call("no CUDA device")                                 # all is well but for the machine
    call("view of an e4m3 cache", kv=object())
    call("dtype", qkv=qkv.half())
    call("unit inner stride", qkv=torch.zeros(8 * 16, 3).t())
    call("int32", slots=slots.long())
    call("cumulative lengths", cu=cu[:2].contiguous())
    call("heads, not 1", store=1)
    call("too narrow", qkv=torch.zeros(3, 7 * 16))
    call("longest run", longest=0)
    call("pairing", pairing="spiral")
    call("cos_sin must be", cos_sin=torch.zeros(3, 4, 2))
    call("must be even", cos_sin=torch.zeros(3, 2, 2), rotary_dim=5)
    call("must be even", cos_sin=torch.zeros(3, 9, 2), rotary_dim=18)
    call("q_out must be", q=torch.zeros(3, 3 * 16))
    call("q_out must be", q=torch.zeros(3, 4 * 16, dtype=torch.bfloat16))


def test_the_attention_refuses():
    kv = view()
    _, cu, slots, start = step_tensors([2, 1])
    q, out = torch.zeros(3, 4 * 16), torch.zeros(3, 4 * 16)

    def call(what, q=q, out=out, kv=kv, cu=cu, slots=slots, start=start, longest=2, heads=4, max_kv_len=2, **more):
        with pytest.raises(KernelError, match=what):
            ops.attention_e4m3(q, out, kv, cu, slots, start, longest, heads, 0.25, max_kv_len=max_kv_len, **more)
    call("no CUDA device")
    call("view of an e4m3 cache", kv=None)
    call("dtype", q=q.half(), out=out.half())
    call("of one dtype", out=out.bfloat16())
    call("of one dtype", q=q[:, :48])
    call("of one dtype", out=out[:2])
    call("cannot share", heads=3, q=torch.zeros(3, 48), out=torch.zeros(3, 48))
    call("must be positive", longest=0)
    call("must be positive", max_kv_len=0)
    call("window", window=-1)
    call("int32", start=start.long())
    ops.attention_e4m3(q[:0], out[:0], kv, torch.zeros(1, dtype=torch.int32), slots[:0], start[:0], 0, 4, 0.25, max_kv_len=0)   # nothing to do


def test_the_eviction_refuses():
    def storage(weights=True):
        kv = view(weights=weights)
        return E4M3Storage(kv.k[None], kv.v[None], kv.scales[None], kv.block_table, weights=kv.weights[None] if weights else None, dropped=kv.dropped)
    slots, lengths = torch.tensor([0, 1], dtype=torch.int32), torch.tensor([100, 60], dtype=torch.int32)

    def call(what, s=None, slots=slots, lengths=lengths, longest=100, budget=70, recent=7, kept=None):
        with pytest.raises(KernelError, match=what):
            ops.kv_evict_e4m3(s or storage(), slots, lengths, longest, budget, recent, kept)
    call("no CUDA device")
    call("storage of an e4m3 cache", s=view())
    call("gathers no attention weights", s=storage(False))
    call("int32", lengths=lengths.long())
    call("int32", lengths=lengths[:1])
    call("budget 0", budget=0, recent=0)
    call("recent 71", recent=71)
    call("holds no 257 rows", longest=257)
    call("kept must be", kept=torch.zeros(1, 2, 2, 69, dtype=torch.int32))


def test_models_and_generation_refuse():
    """A model whose mixers read no such cache; options for a cache that is passed."""
    from go_tinygrad_b200.engine.generate import generate
    from go_tinygrad_b200.engine.model import Model
    from go_tinygrad_b200.parts.base import Runtime
    from go_tinygrad_b200.config.registry import find_architecture
    arch = find_architecture(TINY_A)
    model = Model(arch.plan(arch.read_config(TINY_A)), Runtime(torch.device("cpu"), torch.bfloat16))
    cache = model.new_cache(640, 2, kv_format="e4m3", keep=KeepRule(100, 10))
    assert all(h.kv.format == "e4m3" for h in cache.handles) and cache.max_sequence == 1024 and cache.max_held == 640
    with pytest.raises(ValueError, match="has its own"):
        generate(model, [[1]], 1, cache=cache, kv_format="e4m3")
    assert lib.KeepRule is KeepRule
