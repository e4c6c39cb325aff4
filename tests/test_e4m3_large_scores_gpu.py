"""Gathered weights of the 8-bit cache where scores are so large that their own rounding is more than what sets rows apart."""
import numpy as np
import pytest
import torch

from go_tinygrad_b200.kernels import ops
from test_e4m3_gpu import BF16, DEV, F32, Pages, cut, ints

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
