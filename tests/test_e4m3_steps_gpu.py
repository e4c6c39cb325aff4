"""Steps of whole models over the 8-bit cache: a looped design whose values are its keys, with state beside the cache; layers that
see a window and give pages back; steps on the device that do not stop the host."""
import numpy as np
import pytest
import torch

import go_tinygrad_b200 as lib
import plain_e4m3 as plain
from conftest import make_prompts
from go_tinygrad_b200.cache import KeepRule
from go_tinygrad_b200.engine.decode import DecodeBatch
from test_e4m3_gpu import BF16, DEV, F32, HALF_STEP
from test_ropovik_gpu import CONFIG_P

pytestmark = pytest.mark.gpu


class Order:
    """An op hook that keeps queries, projected keys and values, and attention outputs of one step in the order of the runs."""

    def __init__(self):
        self.runs, self.values = [], None

    def __call__(self, step, layer, op, tensor):
        if op == "v":
            self.values = tensor.double().cpu().numpy().copy()
        elif op == "q_attn":
            self.runs.append({"v": self.values, "q_attn": tensor.double().cpu().numpy().copy()})
        elif op == "attn" and self.runs and "attn" not in self.runs[-1]:
            self.runs[-1]["attn"] = tensor.double().cpu().numpy().copy()


def mixers_in_order(model):
    """(mixer, cache entry) of every run that keeps keys and values."""
    found = []
    for i, entry in enumerate(model.plan.schedule):
        mixer = getattr(model.blocks[entry.layer], "mixer", None)
        if hasattr(mixer, "n_kv"):
            found.append((mixer, i))
    return found


def rows_of(cache, entry, slot, n):
    """Keys, values, weights and value scales of a sequence's rows in one run's cache, by head; rows whose page has been given back
    are zeros."""
    kv = cache.handles[entry].kv
    group = next(g for g in cache.groups if g.e4m3 is not None and g.e4m3.k.data_ptr() <= kv.k.data_ptr() < g.e4m3.k.data_ptr() + g.storage.numel())
    out = []
    for h in range(kv.n_kv_heads):
        k, v, w, vs = np.zeros((n, kv.head_dim)), np.zeros((n, kv.head_dim)), np.zeros(n), np.zeros(n)
        for i in range((n + 63) // 64):
            page, m = group.pages_of[slot][i], min(64, n - 64 * i)
            if page < 0:
                continue
            s = kv.scales[page, :, h].double().cpu().numpy()
            at = slice(64 * i, 64 * i + m)
            k[at] = kv.k.view(torch.uint8)[page, h].view(torch.float8_e4m3fn).double().cpu().numpy()[:m] * s[0]
            v[at] = kv.v.view(torch.uint8)[page, h].view(torch.float8_e4m3fn).double().cpu().numpy().T[:m] * s[1]
            vs[at] = s[1]
            if kv.weights is not None:
                w[at] = kv.weights[page, h].double().cpu().numpy()[:m]
        out.append((k, v, w, vs))
    return out


def checked_step(model, cache, entries, dtype, carried, window=0):
    """One step; every run's attention against the plain statement over the rows that its cache holds, its new values against the
    nearest codes, gathered weights against those before (`carried`).  Evictions are left to the caller.  Bounds as in
    test_steps_of_a_model_over_an_evicting_cache."""
    watch = Order()
    model.op_hook = watch
    evict_due, cache.evict_due = cache.evict_due, lambda slots: None
    held = {e.slot: cache.held(e.slot) for e in entries}
    try:
        logits = lib.step(model, cache, entries)
    finally:
        model.op_hook = None
        del cache.evict_due
    assert torch.isfinite(logits).all()
    bf = dtype == "bfloat16"
    runs = mixers_in_order(model)
    assert len(runs) == len(watch.runs)
    for (mixer, entry), seen in zip(runs, watch.runs):
        heads, n_kv, hd, o = mixer.n_heads, mixer.n_kv, mixer.head_dim, 0
        for e in entries:
            m, h = len(e.tokens), held[e.slot]
            q, attn = (seen[x][o: o + m].reshape(m, n_kv, heads // n_kv, hd) for x in ("q_attn", "attn"))
            vals = seen["v"][o: o + m].reshape(m, n_kv, hd)
            # (the step gives back, at its end, the pages that the next token's window does not reach)
            first = max(0, h + m - window + 1) // 64 * 64 if window else 0
            for j, (k, v, w, vs) in enumerate(rows_of(cache, entry, e.slot, h + m)):
                there = np.arange(h, h + m) >= first
                off = np.abs(v[h:] - vals[:, j])[there]
                assert (off <= np.maximum(np.abs(vals[:, j]) * 2.0 ** -4, vs[h:, None] * 2.0 ** -10)[there]).all()
                for i in range(m):
                    if window and h + i - window + 1 < first:
                        continue
                    want, _ = plain.attend(q[i: i + 1, j], k, v, h + i, mixer.scale, window)
                    size, _ = plain.attend(q[i: i + 1, j], k, np.abs(v), h + i, mixer.scale, window)
                    delta = (hd + 4) * 2.0 ** -23 * (np.abs(q[i, j]) @ np.abs(k).T).max() * mixer.scale
                    rel = 4 * delta + 2.0 ** -20 + (h + m) * 2.0 ** -23
                    bound = size * (rel + (2.0 ** -11 if bf else 0)) + np.abs(want) * HALF_STEP[BF16 if bf else F32] * (1 + 2.0 ** -7)
                    assert (np.abs(attn[i, j] - want[0]) <= bound + 1e-30).all(), (entry, j, i)
                if carried is not None:
                    _, gathered = plain.attend(q[:, j], k, v, h, mixer.scale, window)
                    before = carried.get((entry, e.slot, j), np.zeros(0))
                    total = np.concatenate([before, np.zeros(m)]) + gathered
                    delta = (hd + 4) * 2.0 ** -23 * (np.abs(q[:, j]) @ np.abs(k).T).max() * mixer.scale
                    rel = 4 * delta + 2.0 ** -20 + (h + m) * 2.0 ** -23
                    assert (np.abs(w - total) <= gathered * (rel + m * heads * 2.0 ** -24) + total * 2.0 ** -23 + 1e-30).all(), (entry, j)
                    carried[(entry, e.slot, j)] = w
            o += m
    return logits


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_looped_design_whose_values_are_its_keys(tmp_path, dtype):
    """Heads of 32, 24 and 16 channels, each run of a looped stretch with rows of its own, recurrent state beside them: prompts,
    chunks and single tokens with evictions in between."""
    folder = str(tmp_path)
    lib.write_random_model(folder, CONFIG_P, seed=3, dtype="bfloat16", std=0.15, norm_std=0.1)
    model = lib.Model.load(folder, dtype=dtype, device="cuda")
    keep = KeepRule(70, 20, slack=30)
    cache = model.new_cache(64 * 12, 2, kv_format="e4m3", keep=keep)
    assert len(mixers_in_order(model)) == 2 * 3 + 1
    rng = np.random.default_rng(6)
    tokens = rng.integers(0, CONFIG_P["vocab"], 400).tolist()
    slots, carried, at = [cache.open_sequence() for _ in range(2)], {}, 0

    def step(lengths):
        nonlocal at
        entries = []
        for s, m in zip(slots, lengths):
            if m:
                entries.append(lib.StepEntry(s, tokens[at: at + m], [m - 1]))
                at += m
        checked_step(model, cache, entries, dtype, carried)
        for s in slots:
            if cache.held(s) >= keep.most:
                before = {key: w for key, w in carried.items() if key[1] == s}
                cache.evict_due([s])
                for (entry, _, j), w in before.items():
                    rows = plain.chosen(w.tolist(), keep.budget, keep.recent)
                    after = rows_of(cache, entry, s, keep.budget)[j][2]
                    assert np.array_equal(after, w[rows]), (entry, j)
                    carried[(entry, s, j)] = after
    step([130, 9])
    assert [cache.held(s) for s in slots] == [70, 9]
    for _ in range(32):
        step([1, 1])
    step([5, 70])
    step([1, 0])
    step([0, 2])
    assert [cache.length(s) for s in slots] == [168, 113] and all(cache.held(s) < keep.most for s in slots)
    # as recorded steps and in the open
    results = []
    for use_graph in (True, False):
        made = model.new_cache(64 * 12, 2, kv_format="e4m3", keep=keep)
        results.append([r.tokens for r in lib.generate(model, [tokens[:90], tokens[90:100]], 60, stop=[], cache=made, use_graph=use_graph)])
    assert all(len(t) == 60 for t in results[0]) and (dtype == "bfloat16" or results[0] == results[1])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,window", [("A", 70), ("B", 64)])
def test_layers_that_see_a_window_give_pages_back(model_folders, name, dtype, window):
    """Pages behind the window return to the pool and are taken by another sequence; what is seen stays what it was."""
    model = lib.Model.load(model_folders[name], dtype=dtype, device="cuda")
    for block in model.blocks:
        block.mixer.window = block.mixer.cache_window = window
    cache = model.new_cache(64 * 10, 2, kv_format="e4m3")
    tokens = make_prompts(name, [900], seed=6)[0]
    slots, at = [cache.open_sequence() for _ in range(2)], 0
    free = cache.free_pages()[0]
    for lengths in ([200, 3], [1, 1], [150, 1], [1, 60], [1, 100], [2, 1], [1, 1]):
        entries = []
        for s, m in zip(slots, lengths):
            entries.append(lib.StepEntry(s, tokens[at: at + m], [m - 1]))
            at += m
        checked_step(model, cache, entries, dtype, None, window=window)
    assert [cache.length(s) for s in slots] == [356, 167]
    assert cache.free_pages()[0] >= free - 2 * ((window + 63) // 64 + 1)          # what two windows touch is all that is held


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_device_steps_do_not_stop_the_host(model_folders, dtype):
    """Steps that feed back their own tokens, across evictions and into pages taken anew: no call waits for the device."""
    model = lib.Model.load(model_folders["A"], dtype=dtype, device="cuda")
    keep = KeepRule(64, 16, slack=20)
    prompts = make_prompts("A", [70, 5, 60], seed=8)

    def run(watched):
        cache = model.new_cache(64 * 16, 3, kv_format="e4m3", keep=keep)
        slots = [cache.open_sequence() for _ in prompts]
        lib.step(model, cache, [lib.StepEntry(s, p, []) for s, p in zip(slots, prompts)])
        batch = DecodeBatch(model, cache, slots, [0, 1, 2], lib.Sampler())
        tokens = [batch.step_host([5, 6, 7], [1, 1, 1])]
        picked = [torch.empty_like(batch.sampled) for _ in range(60)]
        for t in picked[:3]:                               # the step is recorded
            batch.step_device()
            t.copy_(batch.sampled)
        batch.reserve_ahead(60)
        torch.cuda.synchronize()
        mode = torch.cuda.get_sync_debug_mode()
        evictions, evict = [], cache.evict
        cache.evict = lambda which, *a, **kw: (evictions.append(list(which)), evict(which, *a, **kw))[1]
        try:
            if watched:
                torch.cuda.set_sync_debug_mode("error")
            for t in picked[3:]:
                batch.step_device()
                t.copy_(batch.sampled)
        finally:
            torch.cuda.set_sync_debug_mode(mode)
            del cache.evict
        assert len(evictions) >= 4 and all(cache.held(s) < keep.most for s in slots)
        return tokens + [t.tolist() for t in picked]
    assert run(True) == run(False)


@pytest.mark.parametrize("kv_format", [None, "e4m3"])
def test_block_tables_copied_on_another_stream(model_folders, kv_format):
    """Pages taken for two sequences, whose rows one stream's step copies for both; the other's step, on a stream of its own, waits for
    the copy and for nothing else."""
    model = lib.Model.load(model_folders["A"], dtype="float32", device="cuda")
    prompts = make_prompts("A", [130, 90], seed=11)
    want = [lib.step(model, c, [lib.StepEntry(c.open_sequence(), p, [len(p) - 1])]) for p in prompts for c in [model.new_cache(64 * 8, 2, kv_format=kv_format)]]
    for _ in range(3):
        cache = model.new_cache(64 * 8, 2, kv_format=kv_format)
        slots = [cache.open_sequence() for _ in prompts]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in prompts]
        cache.reserve_many([(s, len(p)) for s, p in zip(slots, prompts)])
        with torch.cuda.stream(streams[0]):
            torch.cuda._sleep(20_000_000)                  # the copy waits behind this
            cache.flush_tables()
        got = []
        for stream, s, p in zip(streams[::-1], slots[::-1], prompts[::-1]):
            with torch.cuda.stream(stream):
                got.append(lib.step(model, cache, [lib.StepEntry(s, p, [len(p) - 1])]))
            stream.synchronize()                           # (a model's steps share its workspace)
        for a, b in zip(got[::-1], want):
            assert torch.equal(a, b)
