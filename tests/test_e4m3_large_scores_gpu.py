"""Gathered weights of the 8-bit cache where scores are so large that their own rounding is more than what sets rows apart."""
import numpy as np
import pytest
import torch

import plain_e4m3 as plain
from go_tinygrad_b200.kernels import ops
from test_e4m3_gpu import BF16, DEV, F32, HALF_STEP, Pages, cut, ints

pytestmark = pytest.mark.gpu


def one_row_a_query(dtype, hd, new, held, size, key_size, heads=2, loose=False, seed=3):
    """Queries that each see one row: its score leads by 64 and more, and by more than rounding a sum of hd products twice can
    change.  That row's weight grows by one, nobody else's does, and the result is that row's values."""
    rng = np.random.default_rng(seed)
    p = Pages([held], 1, hd, seed=seed, weights=True)
    k, v = p.rows[0][0]
    k.codes, k.scales, v.codes, v.scales = np.zeros((0, hd)), [], np.zeros((0, hd)), []
    k.append(rng.standard_normal((held, hd)) * key_size)
    v.append(rng.standard_normal((held, hd)))
    p.gathered[0][0][:] = 0.0
    p.write(0)
    keys, scale = k.values(), hd ** -0.5
    q, best, spread = np.zeros((new, heads, hd)), np.zeros((new, heads), dtype=int), 0.0
    for i in range(new):
        for g in range(heads):
            while True:
                x = torch.from_numpy(rng.uniform(-1, 1, hd) * size).to(dtype).double().numpy()
                s = keys[: held - new + i + 1] @ x * scale
                most = (np.abs(keys) @ np.abs(x)).max() * scale
                top = np.sort(s)[-2:]
                if top[1] - top[0] > max(64.0, 2 * (hd + 4) * 2.0 ** -23 * most):
                    break
            q[i, g], best[i, g], spread = x, int(s.argmax()), max(spread, most)
    q_dev = torch.from_numpy(q.reshape(new, heads * hd)).to(dtype).to(DEV)
    out = torch.empty_like(q_dev)
    ops.attention_e4m3(q_dev, out, p.view(), cut([new]), ints(p.slots), ints([held - new]), new, heads, scale, max_kv_len=held // 3 if loose else held)
    got = out.double().cpu().numpy().reshape(new, heads, hd)
    for i in range(new):
        for g in range(heads):
            row = v.values()[best[i, g]]                   # (the others' share is below e^-63; codes are numbers of either type)
            assert (np.abs(got[i, g] - row) <= np.abs(row) * 2.0 ** -20 + 2.0 ** -60 * np.abs(v.values()).max()).all(), (i, g)
    want = np.bincount(best.reshape(-1), minlength=held).astype(np.float64)
    # the winning score of the attention and of the weights' own product are each off by (hd + 4) 2^-23 of the sizes' sum; from 2^20 on
    # (in powers of two) what the two may be apart is not charged
    off = 2 * (hd + 4) * 2.0 ** -23 * spread
    rel = 2.0 ** -20 + (2 * off if spread < 2.0 ** 17 else 0.0)
    added = p.read_weights(0, 0, held)
    assert (np.abs(added - want) <= want * rel + 2.0 ** -40).all(), (added.sum(), want.sum(), np.abs(added - want).max())


LARGE = [(2.0 ** 127.9, 2.0 ** -40), (2.0 ** 127.9, 2.0 ** -102), (2.0 ** 60, 2.0 ** -20), (2.0 ** 20, 2.0 ** 60), (2.0 ** 7, 1.0), (2.0 ** -90, 2.0 ** 98)]


@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("size,key_size", LARGE)
@pytest.mark.parametrize("new,held,loose", [(70, 200, False), (40, 1500, False), (70, 900, True)])
def test_prompts(hd, size, key_size, new, held, loose):
    """Scores of up to 2^90 out of queries that leave float's range when they are multiplied with codes; `loose`: rows that the plan has
    no room for."""
    one_row_a_query(BF16, hd, new, held, size, key_size, loose=loose)


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (F32, 128), (F32, 48), (F32, 20), (BF16, 20)])
@pytest.mark.parametrize("size,key_size", LARGE)
@pytest.mark.parametrize("new,held,loose", [(1, 200, False), (1, 1500, False), (70, 200, False), (40, 1500, False), (5, 900, True)])
def test_any_head_size_and_type(dtype, hd, size, key_size, new, held, loose):
    one_row_a_query(dtype, hd, new, held, size, key_size, loose=loose)


@pytest.mark.parametrize("hd", [64, 128, 48, 16])
@pytest.mark.parametrize("size,key_size", LARGE)
@pytest.mark.parametrize("new,held,loose", [(1, 200, False), (5, 900, False), (1, 900, True), (5, 900, True), (16, 2000, True)])
def test_few_queries(hd, size, key_size, new, held, loose):
    """`loose`: rows whose scores the plan has no room to keep, which are computed once more."""
    one_row_a_query(BF16, hd, new, held, size, key_size, loose=loose)


def equal_rows(dtype, hd, new, held, size, key_size, sign, heads=2, loose=False, seed=8):
    """Rows of one key among rows of another, whose scores are far below: the first share each query's probability evenly, however
    large the score they have in common is, and the result is the mean of their values."""
    rng = np.random.default_rng(seed)
    p = Pages([held], 1, hd, seed=seed, weights=True)
    k, v = p.rows[0][0]
    k.codes, k.scales, v.codes, v.scales = np.zeros((0, hd)), [], np.zeros((0, hd)), []
    low, high = np.sort(rng.uniform(1, 3, 2))
    if sign < 0:
        low, high = -high, -low                            # the larger score is the one nearer to zero
    direction = rng.choice([-1.0, 1.0], hd) * rng.choice([1.0, 0.5, 0.25], hd)
    wins = rng.random(held) < 0.7
    wins[: held - new + 1: 5] = True
    wins[0] = True
    k.append(np.where(wins[:, None], high, low) * direction * key_size)
    values = rng.standard_normal((held, hd))
    values[::64] = 3.5                                     # a block has the least scale for that, or, with a larger value, the next
    v.append(values)
    p.gathered[0][0][:] = 0.0
    p.write(0)
    scale = hd ** -0.5
    q = torch.from_numpy(np.tile(direction * size, (new, heads)) * rng.choice([1.0, 0.5], (new, 1))).to(dtype).to(DEV)
    qs = q.double().cpu().numpy().reshape(new, heads, hd)
    out = torch.empty_like(q)
    ops.attention_e4m3(q, out, p.view(), cut([new]), ints(p.slots), ints([held - new]), new, heads, scale, max_kv_len=held // 3 if loose else held)
    want, gathered = plain.attend(qs, k.values(), v.values(), held - new, scale)
    spread = (np.abs(qs.reshape(-1, hd)) @ np.abs(k.values()).T).max() * scale
    got = out.double().cpu().numpy().reshape(want.shape)
    # the tied scores come out alike, whatever their roundings are; a probability is rounded to 11 bits, a result to its type
    bound = np.abs(v.values()).max() * (2.0 ** -11 + held * 2.0 ** -24) + np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -7)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
    off = 2 * (hd + 4) * 2.0 ** -23 * spread
    rel = 2.0 ** -18 + held * 2.0 ** -22 + (2 * off if spread < 2.0 ** 17 else 0.0)
    added = p.read_weights(0, 0, held)
    assert (np.abs(added - gathered) <= gathered * rel + 2.0 ** -40).all(), (added.sum(), gathered.sum(), (np.abs(added - gathered) / (gathered + 1e-30)).max())


TIED = [(2.0 ** 127, 2.0 ** -40), (2.0 ** 60, 2.0 ** -20), (2.0 ** 20, 2.0 ** 60), (2.0 ** 20, 2.0 ** 3), (2.0 ** 20, 2.0 ** -1), (2.0 ** 9, 1.0)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hd", [64, 128, 48])
@pytest.mark.parametrize("size,key_size", TIED)
@pytest.mark.parametrize("new,held,loose", [(70, 200, False), (40, 1500, False), (300, 700, False), (70, 900, True)])
def test_prompts_share_evenly(sign, hd, size, key_size, new, held, loose):
    equal_rows(BF16, hd, new, held, size, key_size, sign, loose=loose)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,hd", [(F32, 64), (F32, 20), (BF16, 20), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("size,key_size", TIED)
@pytest.mark.parametrize("new,held,loose", [(1, 200, False), (5, 900, False), (5, 900, True), (1, 1500, False)])
def test_few_tokens_share_evenly(sign, dtype, hd, size, key_size, new, held, loose):
    equal_rows(dtype, hd, new, held, size, key_size, sign, loose=loose)
