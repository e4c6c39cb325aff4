"""The kernels of the 8-bit cache against the plain statement in 64 bits: storing, attention (decode steps, prompts, chunks), the
gathered weights, eviction, and a run of them together through the engine."""
import math

import numpy as np
import pytest
import torch

import go_tinygrad_b200 as lib
import plain_e4m3 as plain
from conftest import make_prompts
from go_tinygrad_b200.cache import E4M3KVView, E4M3Storage, KeepRule
from go_tinygrad_b200.engine.decode import DecodeBatch
from go_tinygrad_b200.kernels import KernelError, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAN = 0x7F
F32, BF16 = torch.float32, torch.bfloat16
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8}           # of a rounding, relative to the value


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cut(lengths):
    return ints([0] + [int(c) for c in np.cumsum(lengths)])


class Pages:
    """Sequences scattered over the pages of one run's cache (pages in no order, slots in no order, NaN codes wherever nothing was
    stored), and the plain statement's rows beside them."""

    def __init__(self, held, n_kv, hd, seed=0, weights=False, dropped=None, spare_pages=3, room=64):
        self.rng = np.random.default_rng(seed)
        self.held, self.n_kv, self.hd = list(held), n_kv, hd
        per = [(h + room + 63) // 64 for h in held]
        total = sum(per) + spare_pages
        order = self.rng.permutation(total).tolist()
        self.slots = self.rng.permutation(len(held) + 2)[: len(held)].tolist()
        table = np.zeros((len(held) + 2, max(per) + 1), dtype=np.int32)
        self.pages = []
        for slot, n in zip(self.slots, per):
            self.pages.append([order.pop() for _ in range(n)])
            table[slot, :n] = self.pages[-1]
        self.table = torch.from_numpy(table).to(DEV)
        # a page stride larger than a page, as a cache of several planes has
        raw = torch.full((2, total, n_kv * 64 * hd + 32), NAN, dtype=torch.uint8, device=DEV)
        fp8 = raw[:, :, : n_kv * 64 * hd].view(torch.float8_e4m3fn)
        self.k = fp8[0].unflatten(1, (n_kv, 64, hd))
        self.v = fp8[1].unflatten(1, (n_kv, hd, 64))
        self.scales = torch.full((total, 2, n_kv), 2.0 ** -126, device=DEV)
        self.weights = torch.full((total, n_kv, 64), 7.0, device=DEV) if weights else None
        self.dropped = None
        if dropped is not None:
            self.dropped = torch.zeros(len(held) + 2, dtype=torch.int32, device=DEV)
            self.dropped[torch.tensor(self.slots, device=DEV)] = ints(dropped)
        self.gone = [0] * len(held) if dropped is None else list(dropped)
        self.rows = [[(plain.Rows(hd), plain.Rows(hd)) for _ in range(n_kv)] for _ in held]
        self.gathered = [np.zeros((n_kv, h)) for h in held]
        for b, h in enumerate(held):
            for j in range(n_kv):
                if h:
                    for r, x in zip(self.rows[b][j], self.fill(h)):
                        r.append(x)
                    self.gathered[b][j] = self.rng.random(h).astype(np.float32)
            self.write(b)

    def fill(self, n):
        loud = np.where(self.rng.random(self.hd) < 0.1, 5.0, 1.0)
        return self.rng.standard_normal((n, self.hd)) * loud, self.rng.standard_normal((n, self.hd)) * 2.0

    def write(self, b):
        """The plain rows of sequence b into the device's cache."""
        n = len(self.rows[b][0][0].codes)
        for j, (k, v) in enumerate(self.rows[b]):
            for lo in range(0, n, 64):
                page, m = self.pages[b][lo // 64], min(64, n - lo)
                self.k[page, j, :m] = torch.from_numpy(k.codes[lo: lo + m]).float().to(DEV).to(torch.float8_e4m3fn)
                self.v[page, j, :, :m] = torch.from_numpy(v.codes[lo: lo + m].T.copy()).float().to(DEV).to(torch.float8_e4m3fn)
                self.scales[page, 0, j], self.scales[page, 1, j] = k.scales[lo // 64], v.scales[lo // 64]
                if self.weights is not None:
                    self.weights[page, j, :m] = torch.from_numpy(self.gathered[b][j, lo: lo + m]).float().to(DEV)

    def view(self, window=None):
        return E4M3KVView(self.k, self.v, self.scales, self.table, window=window, weights=self.weights, dropped=self.dropped)

    def read(self, b, j, n):
        """Codes of the first n rows, keys and values, and their scales, from the device."""
        pages = torch.tensor(self.pages[b][: (n + 63) // 64], device=DEV)
        k = self.k.view(torch.uint8)[pages, j].view(torch.float8_e4m3fn).double().reshape(-1, self.hd)[:n]
        v = self.v.view(torch.uint8)[pages, j].view(torch.float8_e4m3fn).double().transpose(1, 2).reshape(-1, self.hd)[:n]
        s = self.scales[pages, :, j].double().cpu().numpy()
        return (k.cpu().numpy(), s[:, 0]), (v.cpu().numpy(), s[:, 1])

    def read_weights(self, b, j, n):
        pages = torch.tensor(self.pages[b][: (n + 63) // 64], device=DEV)
        return self.weights[pages, j].reshape(-1)[:n].double().cpu().numpy()


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


# ------------------------------------------------------------------ storing
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("held,new,heads,n_kv,hd", [
    ([0], [1], 1, 1, 16), ([63, 64, 1, 130], [1, 1, 1, 1], 4, 2, 64), ([0, 5, 64, 60], [1, 64, 200, 3], 6, 3, 128), ([10, 0, 70], [0, 65, 2], 3, 1, 48),
    ([7], [129], 2, 2, 20), ([33, 62], [2, 2], 8, 8, 112), ([0, 100], [130, 1], 5, 5, 7), ([500] * 9, [1] * 9, 16, 4, 256)])
def test_store_without_rotation(dtype, held, new, heads, n_kv, hd):
    """Nothing rounds but the codes: codes and scales are the plain statement's."""
    p = Pages(held, n_kv, hd, seed=1, weights=True, room=max(new) + 64)
    n = sum(new)
    rng = np.random.default_rng(2)
    x = rng.standard_normal((n, heads + 2 * n_kv, hd)) * np.exp(rng.standard_normal((n, 1, 1)) * 2)
    wide = torch.zeros(n, (heads + 2 * n_kv) * hd + 8, dtype=dtype, device=DEV)
    qkv = wide[:, : (heads + 2 * n_kv) * hd]
    qkv.copy_(torch.from_numpy(x.reshape(n, -1)))
    before = qkv.clone()
    x = qkv.double().cpu().numpy().reshape(x.shape)
    q = torch.full((n, heads * hd), 5.0, dtype=dtype, device=DEV)
    everything = p.k.view(torch.uint8).clone(), p.v.view(torch.uint8).clone()
    ops.kv_store_e4m3(qkv, None, heads, n_kv, p.view(), cut(new), ints(p.slots), ints(held), max(new), q)
    assert torch.equal(qkv, before) and torch.equal(q, qkv[:, : heads * hd])
    o = 0
    for b, (h, m) in enumerate(zip(held, new)):
        for j in range(n_kv):
            for r, block in zip(p.rows[b][j], (x[o: o + m, heads + j], x[o: o + m, heads + n_kv + j])):
                if m:
                    r.append(block)
            for (codes, scales), r in zip(p.read(b, j, h + m), p.rows[b][j]):
                assert same(codes, r.codes) and same(scales, np.asarray(r.scales)), (b, j)
            w = p.read_weights(b, j, h + m)
            assert (w[h:] == 0).all() and same(w[:h].astype(np.float32), p.gathered[b][j].astype(np.float32))
        o += m
        # rows behind the sequence's last are as they were
        if (h + m) % 64:
            page, t = p.pages[b][(h + m) // 64], (h + m) % 64
            assert (p.k.view(torch.uint8)[page, :, t:] == everything[0][page, :, t:]).all()
            assert (p.v.view(torch.uint8)[page, :, :, t:] == everything[1][page, :, :, t:]).all()
    used = sorted(sum(p.pages, []))
    spare = [i for i in range(p.k.shape[0]) if i not in used]
    assert (p.k.view(torch.uint8)[spare] == NAN).all() and (p.v.view(torch.uint8)[spare] == NAN).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pairing", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rot,shared", [(64, 64, False), (128, 64, False), (48, 24, True), (20, 20, False), (96, 2, False), (16, 16, True)])
def test_store_rotates(dtype, pairing, hd, rot, shared):
    """The stored key is the nearest code to the rotated one, as far as the rotation's rounding in float (three roundings of
    |a| + |b| by half a step of 2^-24 each) can tell; `shared`: the values are the keys as projected."""
    heads, n_kv, held, new = 4, 2, [10, 0, 64], [70, 3, 1]
    p = Pages(held, n_kv, hd, seed=3, dropped=[1000, 0, 64])
    n = sum(new)
    rng = np.random.default_rng(4)
    width = heads + (1 if shared else 2) * n_kv
    qkv = torch.from_numpy(rng.standard_normal((n, width * hd)) * 2).to(dtype).to(DEV)
    x = qkv.double().cpu().numpy().reshape(n, width, hd)
    pos = np.concatenate([g + h + np.arange(m) for g, h, m in zip(p.gone, held, new)])
    angle = pos[:, None] * 1000.0 ** (-np.arange(rot // 2) / (rot // 2))
    table = torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1)).float().to(DEV).contiguous()
    cos, sin = table[..., 0].double().cpu().numpy(), table[..., 1].double().cpu().numpy()
    turned = np.stack([plain.rotate(x[i, : heads + n_kv], cos[i], sin[i], pairing) for i in range(n)])
    size = np.stack([plain.rotate(np.abs(x[i, : heads + n_kv]), np.abs(cos[i]), np.abs(sin[i]), pairing) for i in range(n)])
    size = np.abs(x[:, : heads + n_kv]).max(axis=-1, keepdims=True) * 2 + np.abs(size)
    q = torch.empty(n, heads * hd, dtype=dtype, device=DEV)
    start = [g + h for g, h in zip(p.gone, held)]
    ops.kv_store_e4m3(qkv, table, heads, n_kv, p.view(), cut(new), ints(p.slots), ints(start), max(new), q, pairing=pairing, rotary_dim=rot,
                      values_from_keys=shared)
    slack = 3 * 2.0 ** -24 * size
    got = q.double().cpu().numpy().reshape(n, heads, hd)
    want = turned[:, :heads]
    assert (np.abs(got - want) <= np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -7) + slack[:, :heads]).all()
    o = 0
    for b, (h, m) in enumerate(zip(held, new)):
        for j in range(n_kv):
            (codes, scales), (vcodes, vscales) = p.read(b, j, h + m)
            s = np.repeat(scales, 64)[h: h + m, None]
            key, err = turned[o: o + m, heads + j], slack[o: o + m, heads + j]
            off = np.abs(codes[h:] * s - key)
            assert (off <= np.maximum(np.abs(key) * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20) + 2 * err).all()
            values = x[o: o + m, heads + j if shared else heads + n_kv + j]
            r = p.rows[b][j][1]
            r.append(values)
            assert same(vcodes, r.codes) and same(vscales, np.asarray(r.scales))
        o += m


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_store_of_what_is_not_finite(dtype):
    """Infinities and NaN become NaN codes and count for no scale; the largest and smallest numbers of the type have scales of
    their own."""
    n_kv, hd = 1, 32
    p = Pages([3], n_kv, hd, seed=5, room=130)
    qkv = torch.zeros(130, 2 * hd, dtype=dtype, device=DEV)
    qkv[:, 0], qkv[:, 1] = 3.0, -1.0
    qkv[5, 3], qkv[6, 4], qkv[7, 5] = math.inf, -math.inf, math.nan
    qkv[100, 0] = torch.finfo(dtype).max / 4               # block 1 of the keys
    qkv[:, hd:] = 1e-39
    ops.kv_store_e4m3(qkv, None, 0, n_kv, p.view(), cut([130]), ints(p.slots), ints([3]), 130, None)
    k, v = p.rows[0][0]
    k.append(qkv[:, :hd].double().cpu().numpy())
    v.append(qkv[:, hd:].double().cpu().numpy())
    (codes, scales), (vcodes, vscales) = p.read(0, 0, 133)
    assert same(codes, k.codes) and same(scales, np.asarray(k.scales)) and same(vcodes, v.codes) and same(vscales, np.asarray(v.scales))
    assert np.isnan(codes[8, 3]) and np.isnan(codes[9, 4]) and np.isnan(codes[10, 5]) and np.isfinite(codes).sum() == codes.size - 3


def test_store_queries_only():
    """A run that reads another's cache: nothing in it changes."""
    p = Pages([40], 2, 64, seed=6)
    before = p.k.view(torch.uint8).clone(), p.v.view(torch.uint8).clone(), p.scales.clone()
    qkv = torch.randn(1, 4 * 64, device=DEV)
    q = torch.empty(1, 4 * 64, device=DEV)
    ops.kv_store_e4m3(qkv, None, 4, 0, p.view(), cut([1]), ints(p.slots), ints([40]), 1, q)
    assert torch.equal(q, qkv) and torch.equal(before[0], p.k.view(torch.uint8)) and torch.equal(before[1], p.v.view(torch.uint8))
    assert torch.equal(before[2], p.scales)


# ------------------------------------------------------------------ attention
def attention_case(dtype, held, new, heads, n_kv, hd, window=0, weights=False, dropped=None, seed=7, spread=1.5, past_end=0, loose=False):
    """`held`: rows after the step, the new tokens' among them.  Returns the worst error over its bound.

    The bound.  A score is a sum of hd products (exact in the kernels: 8 by 4 significant bits, or 24 by 4) in float, times two
    factors: delta = (hd + 4) 2^-23 sum |q_d k_d| scale covers its roundings in any order, with truncation.  p then is off by a
    relative 2 delta and the exponential's 2^-21, at most; with bfloat16 queries p may be rounded to 11 bits (half a step 2^-11)
    before it is multiplied with values; the sums over n rows are off by n 2^-24 of the sums of absolute values, at most; and
    the result is rounded to its type."""
    p = Pages(held, n_kv, hd, seed=seed, weights=weights, dropped=dropped)
    n, group = sum(new), heads // n_kv
    rng = np.random.default_rng(seed + 1)
    wide = torch.zeros(n + past_end, heads * hd + 16, dtype=dtype, device=DEV)
    q = wide[:, : heads * hd]
    q.copy_(torch.from_numpy(rng.standard_normal((n + past_end, heads * hd)) * spread))
    out = torch.full((n + past_end, heads * hd + 8), 77.0, dtype=dtype, device=DEV)[:, : heads * hd]
    scale = hd ** -0.5
    longest = max(held) if not loose else max(1, max(held) // 3)           # a plan the sequences have outgrown
    start = [g + h - m for g, h, m in zip(p.gone, held, new)]
    # rows behind the sequences' last: nobody's
    ops.attention_e4m3(q, out, p.view(window or None), cut(new), ints(p.slots), ints(start), max(new), heads, scale, max_kv_len=longest,
                       total_kv_len=sum(held) if not loose else 0)
    assert (out[n:] == 77.0).all()
    qs = q.double().cpu().numpy().reshape(-1, n_kv, group, hd)
    got = out.double().cpu().numpy().reshape(-1, n_kv, group, hd)
    worst, worst_w, o = 0.0, 0.0, 0
    for b, (h, m) in enumerate(zip(held, new)):
        for j in range(n_kv):
            k, v = (r.values() for r in p.rows[b][j])
            want, gathered = plain.attend(qs[o: o + m, j], k, v, h - m, scale, window)
            if m:
                delta = (hd + 4) * 2.0 ** -23 * (np.abs(qs[o: o + m, j]) @ np.abs(k).T).max() * scale
                rel = 2 * delta + 2.0 ** -21 + h * 2.0 ** -24
                size, _ = plain.attend(qs[o: o + m, j], k, np.abs(v), h - m, scale, window)
                bound = size * (2 * rel + (2.0 ** -11 if dtype == BF16 else 0.0)) + np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -7) + 1e-30
                worst = max(worst, (np.abs(got[o: o + m, j] - want) / bound).max())
                assert np.isfinite(got[o: o + m, j]).all()
            if weights:
                w = p.read_weights(b, j, h)
                total = p.gathered[b][j] + gathered
                if m:
                    bound = gathered * (2 * rel + m * group * 2.0 ** -24) + total * 2.0 ** -23 + 1e-30
                    worst_w = max(worst_w, (np.abs(w - total) / bound).max())
                else:
                    assert same(w.astype(np.float32), p.gathered[b][j].astype(np.float32))
        o += m
    if weights:                                            # nothing else gathers
        mask = torch.ones_like(p.weights, dtype=torch.bool)
        for b, h in enumerate(held):
            for i in range((h + 63) // 64):
                mask[p.pages[b][i], :, : min(64, h - 64 * i)] = False
        assert (p.weights[mask] == 7.0).all()
    return worst, worst_w


DECODE = [
    ([1], 1, 1, 64), ([2, 1, 64, 65, 63, 128, 129], 4, 2, 64), ([700, 3, 64, 1500], 8, 8, 64), ([300] * 5, 8, 1, 128), ([1000, 17], 32, 8, 128),
    ([257, 511], 16, 1, 64), ([500], 24, 1, 64), ([190, 5000], 4, 4, 64), ([333, 64], 6, 2, 16), ([100, 200], 6, 2, 32), ([130, 64, 1], 3, 1, 48),
    ([90, 900], 10, 5, 80), ([65, 640], 9, 3, 96), ([70, 200], 7, 1, 112), ([64, 200], 40, 1, 128), ([77, 5], 4, 2, 20), ([130], 3, 3, 7),
    ([40, 400], 2, 1, 256), ([3000], 1, 1, 128), ([9000, 40], 2, 1, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("held,heads,n_kv,hd", DECODE)
def test_decode(dtype, weights, held, heads, n_kv, hd):
    worst, worst_w = attention_case(dtype, held, [1] * len(held), heads, n_kv, hd, weights=weights, past_end=2 if hd == 64 else 0)
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 5000])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 3, 1]])
def test_window(dtype, window, new):
    worst, _ = attention_case(dtype, [600, 64, 131], new, 4, 2, 64, window=window)
    assert worst <= 1, worst


PROMPTS = [
    ([1, 2, 3], [1, 2, 3], 4, 2, 64), ([300, 64, 129, 5], [300, 64, 1, 2], 4, 4, 64), ([200, 333], [190, 33], 8, 2, 128), ([150, 64, 9], [0, 60, 9], 4, 1, 64),
    ([700], [700], 2, 1, 128), ([513, 100], [257, 100], 6, 2, 64), ([90, 70], [40, 70], 3, 1, 48), ([130, 40], [130, 7], 4, 2, 16), ([100], [100], 10, 2, 96),
    ([260], [200], 7, 1, 112), ([129], [128], 5, 5, 80), ([140, 64], [129, 64], 6, 3, 32), ([70, 70], [3, 70], 2, 1, 20), ([100], [65], 2, 2, 256),
    ([1300], [16], 16, 2, 64), ([900, 333], [2, 5], 8, 8, 128),
    # long rows that several blocks share, beside sequences that have few or none
    ([2600, 300, 64, 1500], [150, 300, 1, 0], 8, 2, 64), ([3000], [40], 4, 1, 128), ([2100], [700], 2, 1, 80), ([5000, 1100], [33, 600], 1, 1, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("held,new,heads,n_kv,hd", PROMPTS)
def test_prompts_and_chunks(dtype, weights, held, new, heads, n_kv, hd):
    worst, worst_w = attention_case(dtype, held, new, heads, n_kv, hd, weights=weights, past_end=3 if hd == 128 else 0)
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [[1, 1], [100, 33]])
def test_rows_after_an_eviction(dtype, new):
    """Positions far beyond the rows held: the rows are counted from what is left; positions past 2^31 / 64 channels."""
    worst, worst_w = attention_case(dtype, [300, 129], new, 4, 2, 64, weights=True, dropped=[2_000_000_000, 77])
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [[1, 1], [64, 200]])
def test_a_plan_the_sequences_have_outgrown(dtype, new):
    worst, worst_w = attention_case(dtype, [1000, 2300], new, 4, 2, 64, weights=True, loose=True)
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 32])
@pytest.mark.parametrize("new,window,loose", [(1, 100, True), (6, 700, False), (200, 100, True), (200, 100, False), (150, 1, False)])
def test_weights_of_a_window(dtype, hd, new, window, loose):
    """Rows behind the window gather nothing, whether the plan has room for them or not."""
    worst, worst_w = attention_case(dtype, [1300, 300], [new, 1], 4, 2, hd, window=window, weights=True, loose=loose)
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 90])
def test_peaked_scores(dtype, new):
    """Scores of hundreds: one row takes all; and queries of zero: every row the same."""
    for spread in (60.0, 0.0, 1e-3):
        worst, _ = attention_case(dtype, [900], [new], 4, 2, 64, spread=spread)
        assert worst <= 1, (spread, worst)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("new", [1, 70])
def test_scales_far_apart(dtype, hd, new):
    """Blocks of values whose scales are 2^60 apart, the small ones under the scores that win: what a block adds is
    rounded relative to itself, not to a neighbour nobody looks at."""
    n, p = 64 * 4, Pages([64 * 4], 1, hd, seed=11)
    rng = np.random.default_rng(12)
    k, v = p.rows[0][0]
    direction = rng.standard_normal(hd)
    direction /= np.linalg.norm(direction)
    keys = rng.standard_normal((n, hd)) * 0.1
    keys[64:128] += 30 * direction
    k.codes, k.scales, v.codes, v.scales = np.zeros((0, hd)), [], np.zeros((0, hd)), []
    k.append(keys)
    v.append(rng.standard_normal((n, hd)) * np.repeat([2.0 ** 50, 2.0 ** -10, 2.0 ** 40, 1.0], 64)[:, None])
    p.write(0)
    # scores of the winning block lead by 400 or more: the others' share is below 2^-500 of it
    q = torch.from_numpy(np.tile(direction * 20 * math.sqrt(hd), (new, 2)).reshape(new, 2 * hd)).to(dtype).to(DEV)
    if new > 1:
        q[:, :hd] *= 0.97
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([n - new]), new, 2, hd ** -0.5, max_kv_len=n, total_kv_len=n)
    want, _ = plain.attend(q.double().cpu().numpy().reshape(new, 2, hd), k.values(), v.values(), n - new, hd ** -0.5)
    got = out.double().cpu().numpy().reshape(want.shape)
    size, _ = plain.attend(q.double().cpu().numpy().reshape(new, 2, hd), k.values(), np.abs(v.values()), n - new, hd ** -0.5)
    # scores of about 600: delta = (hd + 4) 2^-23 sum |q k| scale
    delta = (hd + 4) * 2.0 ** -23 * (np.abs(q.double().cpu().numpy().reshape(-1, hd)) @ np.abs(k.values()).T).max() * hd ** -0.5
    bound = size * (4 * delta + 2.0 ** -19 + (2.0 ** -11 if dtype == BF16 else 0)) + np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -7)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 70])
def test_queries_as_large_as_their_type_holds(dtype, new):
    """Scores of 2^80 and more: each query sees one row, and its result is that row's values, codes that bfloat16 holds."""
    n, hd = 200, 64
    p = Pages([n], 1, hd, seed=41, weights=True)
    rng = np.random.default_rng(42)
    k, v = p.rows[0][0]
    k.codes, k.scales, v.codes, v.scales = np.zeros((0, hd)), [], np.zeros((0, hd)), []
    k.append(rng.standard_normal((n, hd)) * 2.0 ** -40)
    v.append(rng.standard_normal((n, hd)))
    p.write(0)
    q = torch.from_numpy(rng.uniform(-1, 1, (new, hd)) * 2.0 ** 127.9).to(dtype).to(DEV)
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([n - new]), new, 1, hd ** -0.5, max_kv_len=n)
    scores = q.double().cpu().numpy() @ k.values().T
    sizes = np.abs(q.double().cpu().numpy()) @ np.abs(k.values()).T
    for i in range(new):
        row = scores[i, : n - new + i + 1]
        best = int(row.argmax())
        # which row wins is beyond what rounding a sum of hd products can change
        assert np.delete(row, best).max() < row[best] - 2 * (hd + 4) * 2.0 ** -23 * sizes[i].max()
        assert np.array_equal(out[i].double().cpu().numpy(), v.values()[best]), i
    added = p.read_weights(0, 0, n) - p.gathered[0][0]
    assert np.isfinite(added).all() and added.min() >= -1e-6 and added.max() <= new * (1 + 2.0 ** -20)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("new", [1, 70, 330])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -90])
@pytest.mark.parametrize("order", [(0, 1, 1, 0, 1, 0), (1, 0, 0, 1, 0, 1), (1,) * 16 + (0,) * 20])
def test_blocks_of_zeros_have_their_share_of_the_probability(dtype, hd, new, small, order):
    """Blocks of values that are zero, or next to it, among others, with keys of their own or zero too: their scales are as small
    as scales get, their probabilities are not.  Bound: attention_case's, each channel's sizes summed."""
    n, heads = 64 * len(order), 2
    p = Pages([n], 1, hd, seed=21, weights=True)
    rng = np.random.default_rng(22)
    k, v = p.rows[0][0]
    k.codes, k.scales, v.codes, v.scales = np.zeros((0, hd)), [], np.zeros((0, hd)), []
    keys = rng.standard_normal((n, hd))
    keys[64:128] = 0.0
    k.append(keys)
    v.append(rng.standard_normal((n, hd)) * np.repeat([1.0 if x else small for x in order], 64)[:, None])
    p.write(0)
    q = torch.from_numpy(rng.standard_normal((new, heads * hd))).to(dtype).to(DEV)
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([n - new]), new, heads, hd ** -0.5, max_kv_len=n, total_kv_len=n)
    qs = q.double().cpu().numpy().reshape(new, heads, hd)
    want, gathered = plain.attend(qs, k.values(), v.values(), n - new, hd ** -0.5)
    size, _ = plain.attend(qs, k.values(), np.abs(v.values()), n - new, hd ** -0.5)
    rel = 2 * (hd + 4) * 2.0 ** -23 * (np.abs(qs).reshape(-1, hd) @ np.abs(k.values()).T).max() * hd ** -0.5 + 2.0 ** -21 + n * 2.0 ** -24
    bound = size * (2 * rel + (2.0 ** -11 if dtype == BF16 else 0.0)) + np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -7) + 1e-30
    got = out.double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
    total = p.gathered[0][0] + gathered
    bound = gathered * (2 * rel + new * heads * 2.0 ** -24) + total * 2.0 ** -23 + 1e-30
    assert (np.abs(p.read_weights(0, 0, n) - total) <= bound).all()


@pytest.mark.parametrize("hd", [64, 128, 32])
@pytest.mark.parametrize("window", [1, 64, 700, 1500])
def test_windows_over_long_rows(hd, window):
    """Blocks that share a sequence's pages, of which some queries see none."""
    worst, _ = attention_case(BF16, [2400, 1900], [300, 1900], 2, 1, hd, window=window)
    assert worst <= 1, worst


@pytest.mark.parametrize("window", [0, 3, 70])
@pytest.mark.parametrize("held,new,heads,n_kv,hd", [([400, 1, 130], [400, 1, 100], 8, 2, 64), ([900], [500], 6, 6, 48), ([300, 64], [300, 64], 7, 1, 112),
                                                    ([333, 20], [332, 0], 24, 8, 16)])
def test_many_rows_in_float(window, held, new, heads, n_kv, hd):
    worst, worst_w = attention_case(F32, held, new, heads, n_kv, hd, window=window, weights=not window, past_end=3)
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("longest", [1, 3, 40])
def test_many_sequences_some_without_new_tokens(dtype, longest):
    rng = np.random.default_rng(51)
    new = [int(x) for x in rng.integers(0, longest + 1, 150)]
    new[:3], new[-1] = [0, 0, longest], 0
    held = [int(m + x) for m, x in zip(new, rng.integers(0, 200, 150))]
    worst, worst_w = attention_case(dtype, held, new, 4, 2, 64, weights=True, dropped=[int(x) for x in rng.integers(0, 9, 150)])
    assert worst <= 1 and worst_w <= 1, (worst, worst_w)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_what_is_not_finite_stays_with_who_sees_it(dtype, new):
    """A NaN key spoils the queries that see its row, of its own head alone; NaN behind the window spoils nobody."""
    p = Pages([200, 100], 2, 64, seed=13)
    p.k.view(torch.uint8)[p.pages[0][1], 1, 5] = NAN       # row 69 of sequence 0, head 1
    n = 2 * new
    q = torch.randn(n, 4 * 64, device=DEV).to(dtype)
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new, new]), ints(p.slots), ints([200 - new, 100 - new]), new, 4, 0.125, max_kv_len=200)
    bad = out.isnan().reshape(2, new, 4, 64)
    assert bad[0, :, 2:].all() and not bad[0, :, :2].any() and not bad[1].any()
    ops.attention_e4m3(q, out, p.view(), cut([new, new]), ints(p.slots), ints([200 - new, 100 - new]), new, 4, 0.125, max_kv_len=200, window=50)
    assert not out.isnan().any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 48])
@pytest.mark.parametrize("new", [2, 70])
def test_a_query_that_is_not_a_number_shows_in_the_weights(dtype, hd, new):
    """Those of all rows it sees, under its own key/value head; its result is NaN, its neighbours' are not."""
    p = Pages([200], 2, hd, seed=14, weights=True)
    q = torch.randn(new, 4 * hd, device=DEV).to(dtype)
    q[new // 2 - 1, 2 * hd + 3] = math.nan                 # head 2, of the second group
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([200 - new]), new, 4, hd ** -0.5, max_kv_len=200)
    bad = out.isnan().reshape(new, 4, hd)
    assert bad[new // 2 - 1, 2].all() and bad.sum() == hd
    seen = 200 - new + new // 2 - 1
    w = p.read_weights(0, 1, 200)
    assert np.isnan(w[: seen + 1]).all() and np.isfinite(w[seen + 1:]).all() and np.isfinite(p.read_weights(0, 0, 200)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 128, 48, 20])
@pytest.mark.parametrize("new,window,held", [(2, 0, 200), (5, 0, 200), (60, 0, 200), (130, 0, 200), (3, 40, 200), (100, 40, 200), (700, 0, 900),
                                             (700, 40, 900)])
def test_nan_values_spoil_the_queries_that_see_their_rows(dtype, hd, new, window, held):
    """One channel of one value row is NaN: queries before it are untouched, those at or behind it have NaN in that channel of
    its head (until it is behind the window), and nowhere else."""
    row, channel = held - 1 - new // 2, 11
    p = Pages([held], 2, hd, seed=18)
    p.v.view(torch.uint8)[p.pages[0][row // 64], 1, channel, row % 64] = NAN
    q = torch.randn(new, 4 * hd, device=DEV).to(dtype)
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([held - new]), new, 4, hd ** -0.5, max_kv_len=held, window=window)
    at = held - new + torch.arange(new, device=DEV)
    sees = (at >= row) & ((at - row < window) if window else True)
    want = torch.zeros(new, 2, 2, hd, dtype=torch.bool, device=DEV)
    want[sees, 1, :, channel] = True
    assert torch.equal(out.isnan().reshape(want.shape), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("held,new", [([3000, 70, 1], [1, 1, 1]), ([500, 333], [257, 40])])
def test_the_same_twice_and_alone(dtype, held, new):
    """The same inputs give the same bits; a sequence's result does not depend on another's rows; two calls over one another on
    two streams do not meet."""
    p = Pages(held, 2, 64, seed=14, weights=True)
    q = torch.randn(sum(new), 4 * 64, device=DEV).to(dtype)
    start = ints([h - m for h, m in zip(held, new)])

    def call():
        out = torch.empty_like(q)
        ops.attention_e4m3(q, out, p.view(), cut(new), ints(p.slots), start, max(new), 4, 0.125, max_kv_len=max(held), total_kv_len=sum(held))
        return out
    first = p.weights.clone()
    a = call()
    after = p.weights.clone()
    p.weights.copy_(first)
    assert torch.equal(a, call()) and torch.equal(after, p.weights)
    v = E4M3KVView(p.k, p.v, p.scales, p.table, dropped=p.dropped)          # one that gathers nothing
    outs, streams = [torch.empty_like(q) for _ in range(6)], [torch.cuda.Stream() for _ in range(2)]
    cu, slots = cut(new), ints(p.slots)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            ops.attention_e4m3(q, o, v, cu, slots, start, max(new), 4, 0.125, max_kv_len=max(held), total_kv_len=sum(held))
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured(dtype):
    """Store and attention recorded into a graph and replayed on other data; two graphs, replayed in turn."""
    held, heads, n_kv, hd = [70, 128, 300], 4, 2, 64
    p = Pages(held, n_kv, hd, seed=15, weights=True)
    kv, cu, slots = p.view(), cut([1] * 3), ints(p.slots)
    qkv = torch.randn(3, (heads + 2 * n_kv) * hd, device=DEV).to(dtype)
    start = ints(held)

    def call(q, out):
        ops.kv_store_e4m3(qkv, None, heads, n_kv, kv, cu, slots, start, 1, q)
        ops.attention_e4m3(q, out, kv, cu, slots, start, 1, heads, 0.125, max_kv_len=303, total_kv_len=sum(held))
    bufs = [(torch.empty(3, heads * hd, dtype=dtype, device=DEV), torch.empty(3, heads * hd, dtype=dtype, device=DEV)) for _ in range(3)]
    state = [t.clone() for t in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)]
    call(*bufs[0])
    graphs = []
    for i in (1, 2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(*bufs[i])
        graphs.append(g)
    for seed in range(2):
        qkv.copy_(torch.randn(3, qkv.shape[1], generator=torch.Generator().manual_seed(seed)))
        results = []
        for run in (lambda: call(*bufs[0]), graphs[0].replay, graphs[1].replay):
            for t, s in zip((p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights), state):
                t.copy_(s)
            run()
            results.append((p.weights.clone(), p.scales.clone()))
        torch.cuda.synchronize()
        for i in (1, 2):
            assert torch.equal(bufs[0][1], bufs[i][1]) and all(torch.equal(x, y) for x, y in zip(results[0], results[i]))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 9, 200])
def test_rows_of_any_stride(hd, new):
    """Rows of q and out that start nowhere in particular give what aligned ones give, as far as bfloat16 can tell."""
    p = Pages([300], 2, hd, seed=19)
    q = torch.randn(new, 4 * hd, device=DEV).bfloat16()
    outs = []
    for pad in (0, 1, 8):
        wide_q, wide_out = (torch.zeros(new, 4 * hd + pad, dtype=BF16, device=DEV) for _ in range(2))
        rows, out = wide_q[:, pad:], wide_out[:, pad:]
        rows.copy_(q)
        ops.attention_e4m3(rows, out, p.view(), cut([new]), ints(p.slots), ints([300 - new]), new, 4, hd ** -0.5, max_kv_len=300)
        outs.append(out.double())
        assert (wide_out[:, :pad] == 0).all()
    # two results that are each within half a step (2^-8) and the products' rounding of the same value
    assert ((outs[0] - outs[1]).abs() <= outs[0].abs() * 2.0 ** -7 + 2.0 ** -9).all() and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [64, 48])
@pytest.mark.parametrize("new", [[1, 1, 1], [70, 2, 64]])
def test_kernels_that_begin_early(dtype, hd, new):
    """Steps over the layers of a model, kernels chained (each may begin while the one before it drains) and recorded into a graph, and
    once more one after the other: the same bits everywhere.  The layers share q and the scratch, so what begins too early shows."""
    layers = [Pages([3000 - m, 1200 - m, 300 - m], 2, hd, seed=70 + i, weights=True, dropped=[0, 5, 9], room=400) for i, m in enumerate((3, 60, 128, 7))]
    heads, steps, n = 8, 3, sum(new)
    qkv = [torch.randn(n, (heads + 4) * hd, device=DEV).to(dtype) for _ in layers]
    q, cu = torch.empty(n, heads * hd, dtype=dtype, device=DEV), cut(new)
    views = [p.view() for p in layers]
    starts = [[ints([h + g + m * t for h, g, m in zip(p.held, p.gone, new)]) for t in range(steps)] for p in layers]
    need = max(ops.attention_e4m3_scratch_floats(dtype, 3, n, max(new), heads, v, 3300) for v in views)
    scratch = torch.empty(max(need, 4), device=DEV)

    def run(outs):
        for t in range(steps):
            for i, (p, v) in enumerate(zip(layers, views)):
                ops.kv_store_e4m3(qkv[i], None, heads, 2, v, cu, ints_of[i], starts[i][t], max(new), q)
                ops.attention_e4m3(q, outs[t][i], v, cu, ints_of[i], starts[i][t], max(new), heads, hd ** -0.5, max_kv_len=3300, scratch=scratch)
    ints_of = [ints(p.slots) for p in layers]
    before = [[x.clone() for x in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)] for p in layers]
    results = []
    for chained in (False, True, True):
        for p, b in zip(layers, before):
            for x, y in zip((p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights), b):
                x.copy_(y)
        outs = [[torch.zeros_like(q) for _ in layers] for _ in range(steps)]
        if not chained:
            run(outs)
        else:
            with ops.chained_launches():
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    run(outs)
                g.replay()
        torch.cuda.synchronize()
        results.append([x.clone() for row in outs for x in row] + [x.clone() for p in layers for x in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("new", [1, 4])
def test_a_table_too_wide_to_count_its_steps_in_32_bits(new):
    """Rows of the block table 2^27 entries apart: such a step takes the general kernel, scratch as for any."""
    p = Pages([700, 90], 8, 64, seed=63, weights=True)
    wide = torch.zeros(p.table.shape[0], 1 << 27, dtype=torch.int32, device=DEV)
    wide[:, : p.table.shape[1]] = p.table
    q = torch.randn(2 * new, 16 * 64, device=DEV).bfloat16()
    before, outs, weights = p.weights.clone(), [], []
    for table in (p.table, wide[:, : p.table.shape[1]]):
        p.weights.copy_(before)
        view, out = E4M3KVView(p.k, p.v, p.scales, table, weights=p.weights), torch.empty_like(q)
        ops.attention_e4m3(q, out, view, cut([new, new]), ints(p.slots), ints([700 - new, 90 - new]), new, 16, 0.125, max_kv_len=700)
        outs.append(out.double())
        weights.append(p.weights.double())
    # each within half a step (2^-8) and the products' roundings of the same value
    assert ((outs[0] - outs[1]).abs() <= outs[0].abs() * 2.0 ** -7 + 2.0 ** -9).all()
    # as attention_case has it for each of the two, the largest sum of sizes taken from the norms
    longest = max(np.linalg.norm(r[0].values(), axis=1).max() for rows in p.rows for r in rows)
    delta = 68 * 2.0 ** -23 * q.double().reshape(-1, 64).norm(dim=1).max().item() * longest * 0.125
    rel = 2 * (2 * (2 * delta + 2.0 ** -21 + 700 * 2.0 ** -24) + 2 * new * 2.0 ** -24) + 2.0 ** -22
    assert ((weights[0] - weights[1]).abs() <= rel * weights[0].abs()).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 100])
def test_pages_further_than_32_bits_count(dtype, new):
    """The same sequence in a small cache and at the end of one of 4.4 GB: attention, a step's store and an eviction agree bit by bit."""
    n_kv, hd, held, total = 32, 128, 300, 8400
    p = Pages([held], n_kv, hd, seed=61, weights=True, dropped=[0], room=128)
    raw = torch.zeros(total, 2, n_kv * 64 * hd, dtype=torch.uint8, device=DEV)
    k, v = (raw[:, i].view(torch.float8_e4m3fn) for i in (0, 1))
    k, v = k.unflatten(1, (n_kv, 64, hd)), v.unflatten(1, (n_kv, hd, 64))
    scales, weights = torch.ones(total, 2, n_kv, device=DEV), torch.zeros(total, n_kv, 64, device=DEV)
    here, there = torch.tensor(p.pages[0], device=DEV), torch.arange(total - len(p.pages[0]), total, device=DEV)

    def parts(view):
        return [view.k.view(torch.uint8), view.v.view(torch.uint8), view.scales, view.weights]
    small = p.view()
    table = torch.zeros_like(p.table)
    table[p.slots[0], : len(p.pages[0])] = there.int()
    big = E4M3KVView(k, v, scales, table, weights=weights, dropped=torch.zeros_like(p.dropped))
    for a, b in zip(parts(small), parts(big)):
        b[there] = a[here]
    q = torch.randn(new, n_kv * hd, device=DEV).to(dtype)
    qkv = torch.randn(70, 3 * n_kv * hd, device=DEV).to(dtype)
    outs = []
    for view in (small, big):
        out, stored = torch.empty_like(q), torch.empty(70, n_kv * hd, dtype=dtype, device=DEV)
        ops.attention_e4m3(q, out, view, cut([new]), ints(p.slots), ints([held - new]), new, n_kv, hd ** -0.5, max_kv_len=held)
        ops.kv_store_e4m3(qkv, None, n_kv, n_kv, view, cut([70]), ints(p.slots), ints([held]), 70, stored)
        s = E4M3Storage(view.k[None], view.v[None], view.scales[None], view.block_table, weights=view.weights[None], dropped=view.dropped)
        kept = ops.kv_evict_e4m3(s, ints(p.slots), ints([held + 70]), held + 70, 200, 50)
        outs.append((out, stored, kept))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert all(torch.equal(a[here], b[there]) for a, b in zip(parts(small), parts(big)))


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_waits_that_run_out(hd):
    """The tcgen05 form's give-up path: tiles that never arrive.  The kernel returns, says so, and works again afterwards."""
    p = Pages([300, 70], 2, hd, seed=23, weights=True)
    q = torch.randn(270, 4 * hd, device=DEV).bfloat16()
    before = p.weights.clone()

    def run():
        out = torch.full_like(q, 7.0)
        p.weights.copy_(before)
        ops.attention_e4m3(q, out, p.view(), cut([200, 70]), ints(p.slots), ints([100, 0]), 200, 4, hd ** -0.5, max_kv_len=300)
        return torch.cat([out.float().flatten(), p.weights.flatten()])
    want = run()
    assert ops.bounded_wait_failures() == 0
    try:
        ops.wait_test_hooks("attention_e4m3_tcgen05", True)
        run()
        torch.cuda.synchronize()
        assert ops.bounded_wait_failures() != 0
    finally:
        ops.wait_test_hooks("attention_e4m3_tcgen05", False)
    assert ops.bounded_wait_failures() == 0 and torch.equal(run(), want) and ops.bounded_wait_failures() == 0


def test_other_streams_and_devices_are_checked():
    p = Pages([70], 1, 64, seed=16)
    q = torch.randn(1, 64, device=DEV)
    with pytest.raises(KernelError, match="cache's device"):
        ops.attention_e4m3(q.cpu(), torch.empty(1, 64), p.view(), cut([1]), ints(p.slots), ints([69]), 1, 1, 0.125, max_kv_len=70)
    with pytest.raises(KernelError, match="cache's device"):
        ops.attention_e4m3(q, torch.empty(1, 64), p.view(), cut([1]), ints(p.slots), ints([69]), 1, 1, 0.125, max_kv_len=70)
    with pytest.raises(KernelError, match="cache's device"):
        ops.kv_store_e4m3(torch.zeros(1, 192, device=DEV), None, 1, 1, p.view(), cut([1]), ints(p.slots), ints([70]), 1, torch.empty(1, 64))
    with pytest.raises(KernelError, match="cache's device"):
        ops.kv_store_e4m3(torch.zeros(1, 192, device=DEV), torch.zeros(1, 32, 2), 1, 1, p.view(), cut([1]), ints(p.slots), ints([70]), 1, q)
    scratch = torch.empty(1, device=DEV)
    p = Pages([70], 1, 64, seed=16, weights=True)
    need = ops.attention_e4m3_scratch_floats(F32, 1, 1, 1, 1, p.view(), 70)
    if need > 1:
        with pytest.raises(KernelError, match="scratch needs"):
            ops.attention_e4m3(q, torch.empty_like(q), p.view(), cut([1]), ints(p.slots), ints([69]), 1, 1, 0.125, max_kv_len=70, scratch=scratch)


def test_checked_access():
    """With the debug pass on, a bad slot, page or position is an error and the kernel is not launched."""
    p = Pages([70], 1, 64, seed=17, dropped=[1000])
    q, out = torch.randn(1, 64, device=DEV), torch.empty(1, 64, device=DEV)
    qkv = torch.randn(1, 3 * 64, device=DEV)
    with ops.checked_access():
        good = (p.view(), cut([1]))
        ops.attention_e4m3(q, out, *good, ints(p.slots), ints([1069]), 1, 1, 0.125, max_kv_len=70)
        for slots, start, what in (([9], [1069], "slot"), (p.slots, [5000], "beyond"), (p.slots, [900], "negative")):
            with pytest.raises(KernelError, match=what):
                ops.attention_e4m3(q, out, *good, ints(slots), ints(start), 1, 1, 0.125, max_kv_len=70)
            with pytest.raises(KernelError, match=what):
                ops.kv_store_e4m3(qkv, None, 1, 1, *good, ints(slots), ints(start), 1, q)
        p.table.fill_(99)
        with pytest.raises(KernelError, match="page"):
            ops.attention_e4m3(q, out, *good, ints(p.slots), ints([1069]), 1, 1, 0.125, max_kv_len=70)


# ------------------------------------------------------------------ eviction
def evict_case(lengths, budget, recent, n_kv, hd, entries=2, seed=20, ties=True, weights_of=None):
    runs = [Pages(lengths, n_kv, hd, seed=seed, weights=True, room=64) for _ in range(entries)]
    for e, p in enumerate(runs):                           # same pages, other contents
        p.rng = np.random.default_rng(seed + 100 + e)
        for b, n in enumerate(lengths):
            for j in range(n_kv):
                k, v = plain.Rows(hd), plain.Rows(hd)
                a, c = p.fill(n)
                size = np.exp(p.rng.standard_normal((n, 1)) * 1.5)
                k.append(a * size)
                v.append(c * size)
                p.rows[b][j] = (k, v)
                w = p.rng.random(n).astype(np.float32) ** 6 * 30
                if ties:
                    w = np.where(p.rng.random(n) < 0.5, np.float32(np.floor(w * 4) / 4), w)
                p.gathered[b][j] = w if weights_of is None else weights_of(p.rng, n)
            p.write(b)
    stack = lambda name: torch.stack([getattr(p, name) for p in runs])
    k = torch.stack([p.k.view(torch.uint8) for p in runs]).view(torch.float8_e4m3fn)
    v = torch.stack([p.v.view(torch.uint8) for p in runs]).view(torch.float8_e4m3fn)
    scales, weights, dropped = stack("scales"), stack("weights"), torch.full((len(lengths) + 2,), 5, dtype=torch.int32, device=DEV)
    before = k.view(torch.uint8).clone(), v.view(torch.uint8).clone(), scales.clone(), weights.clone()
    storage = E4M3Storage(k, v, scales, runs[0].table, weights=weights, dropped=dropped)
    kept = ops.kv_evict_e4m3(storage, ints(runs[0].slots), ints(lengths), max(lengths), budget, recent)
    want_dropped = [5] * (len(lengths) + 2)
    for slot, n in zip(runs[0].slots, lengths):
        want_dropped[slot] += max(0, n - budget)
    assert dropped.tolist() == want_dropped
    kept = kept.cpu().numpy()
    for e, p in enumerate(runs):
        p.k, p.v, p.scales, p.weights = k[e], v[e], scales[e], weights[e]
        for b, n in enumerate(lengths):
            for j in range(n_kv):
                rows = plain.chosen(p.gathered[b][j].tolist(), budget, recent)
                assert kept[e, b, j, : len(rows)].tolist() == rows and (kept[e, b, j, len(rows):] == -1).all(), (e, b, j)
                if n > budget:
                    for r in p.rows[b][j]:
                        r.keep(rows)
                (kc, ks), (vc, vs) = p.read(b, j, len(rows))
                for codes, s, r in ((kc, ks, p.rows[b][j][0]), (vc, vs, p.rows[b][j][1])):
                    assert same(s, np.asarray(r.scales)[: len(s)]) and same(codes, r.codes), (e, b, j)
                assert same(p.read_weights(b, j, len(rows)).astype(np.float32), np.asarray(p.gathered[b][j])[rows].astype(np.float32))
        # rows behind the kept ones, and pages of nobody, are as they were
        rows_of = {}
        for b, n in enumerate(lengths):
            for i in range((budget + 63) // 64 if n > budget else 0):
                rows_of[p.pages[b][i]] = min(64, budget - 64 * i)
        for page in range(k.shape[1]):
            t = rows_of.get(page, 0)
            assert torch.equal(k.view(torch.uint8)[e, page, :, t:], before[0][e, page, :, t:])
            assert torch.equal(v.view(torch.uint8)[e, page, :, :, t:], before[1][e, page, :, :, t:])
            assert torch.equal(weights[e, page, :, t:], before[3][e, page, :, t:])
            if not t:
                assert torch.equal(scales[e, page], before[2][e, page])


@pytest.mark.parametrize("lengths,budget,recent,n_kv,hd", [
    ([66], 65, 1, 1, 16), ([128], 64, 64, 2, 64), ([576], 512, 128, 2, 64), ([300, 70, 128, 64], 100, 20, 3, 128), ([200], 199, 0, 1, 48), ([500, 450], 1, 1, 1, 32),
    ([500], 1, 0, 2, 32), ([130, 131], 130, 130, 2, 20), ([1000], 64, 10, 1, 7), ([2112, 2000], 2048, 500, 1, 64), ([5000], 333, 33, 1, 112),
    ([2, 1, 3], 1, 0, 2, 16), ([100], 100, 50, 1, 64), ([4000], 3000, 2999, 1, 256)])
def test_evict(lengths, budget, recent, n_kv, hd):
    evict_case(lengths, budget, recent, n_kv, hd)


@pytest.mark.parametrize("weights_of", [
    lambda rng, n: np.zeros(n, dtype=np.float32),                                                  # nobody was looked at: the first rows stay
    lambda rng, n: np.where(np.arange(n) % 2 == 0, np.float32(1e-42), np.float32(0)).astype(np.float32),        # the smallest numbers there are
    lambda rng, n: np.float32(1) + rng.integers(0, 3, n).astype(np.float32) * np.float32(2.0 ** -23),           # apart by one step
    lambda rng, n: np.where(rng.random(n) < 0.1, np.float32(np.inf), rng.random(n).astype(np.float32)).astype(np.float32),
    lambda rng, n: np.arange(n, dtype=np.float32)], ids=["zeros", "tiny", "near", "infinite", "rising"])
def test_evict_by_weights_of_all_kinds(weights_of):
    evict_case([700, 130], 129, 30, 2, 64, entries=1, weights_of=weights_of)


@pytest.mark.parametrize("hd", [64, 128, 48, 20])
@pytest.mark.parametrize("budget,recent,heavy", [(100, 20, [(10, 50), (900, 935), (1500, 1505)]), (130, 0, [(640, 641), (1000, 1100), (2400, 2429)]),
                                                  (64, 1, [(2490, 2499)]), (300, 300, []), (200, 10, [(i, i + 1) for i in range(0, 2500, 13)])])
def test_evict_over_pages_of_which_nothing_stays(hd, budget, recent, heavy):
    """Rows that stay lie in few pages, far apart, or one or two in every page."""
    def weights_of(rng, n):
        w = rng.random(n).astype(np.float32)
        for lo, hi in heavy:
            w[lo: min(hi, n)] += 10
        return w
    evict_case([2500, 1300, 60], budget, recent, 2, hd, entries=1, weights_of=weights_of)


@pytest.mark.parametrize("hd", [64, 20])
def test_evict_leaves_sequences_longer_than_it_was_told_of(hd):
    p = Pages([300, 200], 2, hd, seed=31, weights=True, dropped=[0, 0])
    s = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None], dropped=p.dropped)
    before = [t.clone() for t in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)]
    kept = ops.kv_evict_e4m3(s, ints(p.slots), ints([300, 200]), 250, 130, 10)
    assert (kept[0, 0] == -1).all() and (kept[0, 1] >= 0).all() and p.dropped[p.slots[0]] == 0 and p.dropped[p.slots[1]] == 70
    pages = torch.tensor(p.pages[0], device=DEV)
    for was, now in zip(before, (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)):
        assert torch.equal(was[pages], now[pages])


def test_evict_keeps_the_code_of_nan():
    p = Pages([200], 1, 64, seed=21, weights=True)
    p.gathered[0][0][:] = np.arange(200)
    p.rows[0][0][0].codes[150, 3] = np.nan
    p.write(0)
    storage = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None])
    kept = ops.kv_evict_e4m3(storage, ints(p.slots), ints([200]), 200, 100, 0)
    assert kept[0, 0, 0].tolist() == list(range(100, 200))
    p.rows[0][0][0].keep(list(range(100, 200)))
    (codes, scales), _ = p.read(0, 0, 100)
    assert same(codes, p.rows[0][0][0].codes) and same(scales, np.asarray(p.rows[0][0][0].scales)) and np.isnan(codes[50, 3])


# ------------------------------------------------------------------ together, through the engine
_models = {}


def get_model(model_folders, name, dtype):
    if (name, dtype) not in _models:
        _models[(name, dtype)] = lib.Model.load(model_folders[name], dtype=dtype, device="cuda")
    return _models[(name, dtype)]


class Watch:
    """An op hook that keeps each layer's queries, projected keys and values, and attention output of one step."""

    def __init__(self):
        self.seen = {}

    def __call__(self, step, layer, op, tensor):
        if op in ("k", "v", "q_attn", "attn"):
            self.seen[(layer, op)] = tensor.double().cpu().numpy().copy()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B"])
def test_steps_of_a_model_over_an_evicting_cache(model_folders, name, dtype):
    """Prompts of unequal lengths, a chunk, single tokens, evictions in between, a sequence that ends and another in its slot:
    after every step each layer's new rows hold the nearest codes, the attention output is that of the rows held, weights add up, and
    an eviction keeps the heaviest and newest.  Rows and weights are carried by the plain statement from the traced values."""
    model = get_model(model_folders, name, dtype)
    cfg = model.config
    heads, n_kv, hd = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    keep = KeepRule(90, 30, slack=16)
    cache = model.new_cache(64 * 12, 3, kv_format="e4m3", keep=keep)
    prompts = make_prompts(name, [150, 20, 88], seed=3)
    slots = [cache.open_sequence() for _ in prompts]
    follow = make_prompts(name, [400], seed=4)[0]
    weights = {}                                           # (slot, layer, head) -> what the rows have gathered
    watch = Watch()
    model.op_hook = watch

    def step(entries):
        held = {e.slot: cache.held(e.slot) for e in entries}
        due = [e.slot for e in entries if cache.held(e.slot) + len(e.tokens) >= keep.most]
        taken = {}
        evict, kept_by_slot = cache.evict, {}

        def spy(which, *a, **kw):                          # the cache as it stands between attention and eviction
            for s in which:
                taken[s] = snapshot(s)
            out = evict(which, *a, **kw)
            for i, s in enumerate(which):
                kept_by_slot[s] = out[0][:, i].cpu().numpy()
            return out
        cache.evict = spy
        try:
            logits = lib.step(model, cache, entries)
        finally:
            del cache.evict
        assert torch.isfinite(logits).all() and sorted(kept_by_slot) == sorted(due)
        o = 0
        for e in entries:
            m, h = len(e.tokens), held[e.slot]
            now = taken.get(e.slot) or snapshot(e.slot)
            for layer in range(cfg.num_hidden_layers):
                q = watch.seen[(layer, "q_attn")][o: o + m].reshape(m, n_kv, heads // n_kv, hd)
                attn = watch.seen[(layer, "attn")][o: o + m].reshape(m, n_kv, heads // n_kv, hd)
                vals = watch.seen[(layer, "v")][o: o + m].reshape(m, n_kv, hd)
                for j in range(n_kv):
                    k, v, s, w = now[(layer, j)]
                    assert len(k) == h + m
                    vs = np.repeat(s[:, 1], 64)[: h + m, None]
                    assert (np.abs(v[h:] - vals[:, j]) <= np.maximum(np.abs(vals[:, j]) * 2.0 ** -4, vs[h:] * 2.0 ** -10)).all()
                    want, gathered = plain.attend(q[:, j], k, v, h, hd ** -0.5)
                    size, _ = plain.attend(q[:, j], k, np.abs(v), h, hd ** -0.5)
                    delta = (hd + 4) * 2.0 ** -23 * (np.abs(q[:, j]) @ np.abs(k).T).max() * hd ** -0.5
                    rel = 4 * delta + 2.0 ** -20 + (h + m) * 2.0 ** -23
                    bf = dtype == "bfloat16"
                    bound = size * (rel + (2.0 ** -11 if bf else 0)) + np.abs(want) * HALF_STEP[BF16 if bf else F32] * (1 + 2.0 ** -7)
                    assert (np.abs(attn[:, j] - want) <= bound + 1e-30).all()
                    before = weights.get((e.slot, layer, j), np.zeros(0))
                    total = np.concatenate([before, np.zeros(m)]) + gathered
                    assert (np.abs(w - total) <= gathered * (rel + m * heads * 2.0 ** -24) + total * 2.0 ** -23 + 1e-30).all()
                    weights[(e.slot, layer, j)] = w
                    if e.slot in kept_by_slot:
                        rows = plain.chosen(w.tolist(), keep.budget, keep.recent)
                        assert kept_by_slot[e.slot][layer, j].tolist() == rows
                        after = snapshot(e.slot, layer, j)
                        assert np.array_equal(after[3], w[rows])
                        # codes round again only where they need the smallest steps
                        for x, y, plane in ((after[0], k[rows], 0), (after[1], v[rows], 1)):
                            assert (np.abs(x - y) <= np.repeat(after[2][:, plane], 64)[: len(rows), None] * 2.0 ** -10).all()
                        weights[(e.slot, layer, j)] = w[rows]
            o += m
        return logits

    def snapshot(slot, only_layer=None, only_head=None):
        got = {}
        n = cache.held(slot) if only_layer is not None else cache.length(slot) - cache._dropped[slot]
        grp = cache.groups[0]
        pages = torch.tensor(grp.pages_of[slot][: (n + 63) // 64], device=DEV)
        st = grp.e4m3
        for layer in range(cfg.num_hidden_layers) if only_layer is None else [only_layer]:
            for j in range(n_kv) if only_head is None else [only_head]:
                s = st.scales[layer, pages, :, j].double()
                k = st.k[layer].view(torch.uint8)[pages, j].view(torch.float8_e4m3fn).double() * s[:, 0, None, None]
                v = st.v[layer].view(torch.uint8)[pages, j].view(torch.float8_e4m3fn).double() * s[:, 1, None, None]
                got[(layer, j)] = (k.reshape(-1, hd)[:n].cpu().numpy(), v.transpose(1, 2).reshape(-1, hd)[:n].cpu().numpy(), s.cpu().numpy(),
                                   st.weights[layer, pages, j].reshape(-1)[:n].double().cpu().numpy())
        return got if only_layer is None else got[(only_layer, only_head)]
    try:
        step([lib.StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)])
        assert [cache.held(s) for s in slots] == [90, 20, 88]
        at = 0
        for i in range(40):
            step([lib.StepEntry(s, [follow[at + j]], [0]) for j, s in enumerate(slots)])
            at += 3
        assert [cache.length(s) for s in slots] == [190, 60, 128] and all(cache.held(s) < keep.most for s in slots)
        step([lib.StepEntry(slots[0], follow[at: at + 70], [69]), lib.StepEntry(slots[1], [follow[at]], [0])])
        cache.close_sequence(slots[1])
        for key in [k for k in weights if k[0] == slots[1]]:
            del weights[key]
        assert cache.open_sequence() == slots[1]
        step([lib.StepEntry(slots[1], follow[:10], [9]), lib.StepEntry(slots[2], follow[10:12], [1])])
    finally:
        model.op_hook = None


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_over_an_evicting_cache(model_folders, dtype):
    """Decode steps as recorded graphs against steps in the open, across evictions; the cache's rows stay bounded."""
    model = get_model(model_folders, "A", dtype)
    prompts = make_prompts("A", [70, 5, 130], seed=8)
    keep = KeepRule(64, 16, slack=20)
    results = []
    for use_graph in (True, False):
        cache = model.new_cache(64 * 16, 3, kv_format="e4m3", keep=keep)
        results.append([r.tokens for r in lib.generate(model, prompts, 120, stop=[], cache=cache, use_graph=use_graph)])
        assert all(len(t) == 120 for t in results[-1]) and cache.free_pages() == [16]
    if dtype == "float32":                                 # no sum there depends on how the work is cut
        assert results[0] == results[1]
    made = lib.generate(model, prompts, 120, stop=[], kv_format="e4m3", keep=keep)
    assert [r.tokens for r in made] == results[0]
    # a batch kept over several calls, driven on the device
    cache = model.new_cache(64 * 16, 3, kv_format="e4m3", keep=keep)
    slots = [cache.open_sequence() for _ in prompts]
    lib.step(model, cache, [lib.StepEntry(s, p, []) for s, p in zip(slots, prompts)])
    batch = DecodeBatch(model, cache, slots, [0, 1, 2], lib.Sampler())
    batch.step_host([r[0] for r in results[0]], [1, 1, 1])
    batch.reserve_ahead(50)
    tokens = [batch.sampled.tolist()]
    for _ in range(60):
        batch.step_device()
        tokens.append(batch.sampled.tolist())
        assert all(cache.held(s) < keep.most for s in slots)
    if dtype == "float32":
        assert [list(t) for t in zip(*tokens)] == [r[1:62] for r in results[0]]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_an_unbounded_cache_of_8_bits_is_near_the_wide_one(model_folders, dtype):
    """Same model, same tokens: logits over 8-bit rows against logits over the compute type's.  Keys and values are off by at most
    1/16 of themselves; the two layers' logits (of a few units) then stay within a few tenths of the largest."""
    model = get_model(model_folders, "A", dtype)
    prompt = make_prompts("A", [150], seed=9)[0]
    got = []
    for kv_format in (None, "e4m3"):
        cache = model.new_cache(256, 1, kv_format=kv_format)
        slot = cache.open_sequence()
        rows = [lib.step(model, cache, [lib.StepEntry(slot, prompt[:100], [99])])]
        rows += [lib.step(model, cache, [lib.StepEntry(slot, [t], [0])]) for t in prompt[100:]]
        got.append(torch.cat(rows).double())
        if kv_format:
            cache.truncate(slot, 120)
            again = lib.step(model, cache, [lib.StepEntry(slot, [prompt[120]], [0])]).double()
            assert (again - got[-1][21:22]).abs().max() <= 0.25 * got[-1].abs().max()
    assert (got[0] - got[1]).abs().max() <= 0.25 * got[0].abs().max()
    assert (got[0] - got[1]).abs().max() > 0


def test_command_line(model_folders, capsys):
    from go_tinygrad_b200.cli.llmgen import main
    base = ["-model", model_folders["A"], "-ids", ",".join(["7"] * 90), "-tokens", "40", "-stop", "999"]
    for more in (["-kv-format", "e4m3"], ["-kv-format", "e4m3", "-keep", "32"], ["-kv-format", "e4m3", "-keep", "32", "-keep-recent", "0", "-max-len", "192"]):
        assert main(base + more) == 0
        assert "Generated tokens: 40" in capsys.readouterr().out
    assert main(base + ["-keep", "32"]) == 1 and "needs -kv-format" in capsys.readouterr().err
    assert main(base + ["-kv-format", "e4m3", "-keep", "32", "-keep-recent", "33"]) == 1
