"""Evictions of the 8-bit cache at the ends of its numbers' ranges: what stays of a block are its smallest codes, or zeros; weights that
are no numbers."""
import numpy as np
import pytest
import torch

import plain_e4m3 as plain
from go_tinygrad_b200.cache import E4M3Storage
from go_tinygrad_b200.kernels import ops
from test_e4m3_gpu import DEV, Pages, ints, same

pytestmark = pytest.mark.gpu


def loud_rows_go(hd, smallest, loud, n_kv=2, held=(330, 70, 200), budget=130, recent=0, seed=5):
    """Pages whose scale one row in 16 made, all of which go; the others' codes are whole numbers of the smallest step 2^-9, up to
    `smallest[i % len]` in page i (0: a page of ordinary numbers).  Codes, scales and weights of what stays, bit by bit."""
    p = Pages(held, n_kv, hd, seed=seed, weights=True)
    rng = np.random.default_rng(seed)
    for b, n in enumerate(held):
        for j in range(n_kv):
            for plane, r in enumerate(p.rows[b][j]):
                for lo in range(0, n, 64):
                    m, most = min(64, n - lo), smallest[lo // 64 % len(smallest)]
                    if most:
                        codes = rng.integers(-most, most + 1, (m, hd)) * 2.0 ** -9
                        codes[:, 0] = most * 2.0 ** -9
                        codes[::16] = rng.choice([-1.0, 1.0], codes[::16].shape) * loud
                    else:
                        codes = plain.nearest(rng.standard_normal((m, hd)) * 40)
                    r.codes[lo: lo + m] = codes
                    r.scales[lo // 64] = 2.0 ** int(rng.integers(-3, 4)) if len(smallest) == 1 else 2.0 ** (-8 * plane)
            w = rng.random(n).astype(np.float32) + 1
            w[::16] = 0.0
            p.gathered[b][j] = w
        p.write(b)
    s = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None])
    kept = ops.kv_evict_e4m3(s, ints(p.slots), ints(list(held)), max(held), budget, recent).cpu().numpy()
    for b, n in enumerate(held):
        for j in range(n_kv):
            rows = plain.chosen(p.gathered[b][j].tolist(), budget, recent)
            assert kept[0, b, j, : len(rows)].tolist() == rows
            if n > budget:
                assert not any(i % 16 == 0 for i in rows)
                for r in p.rows[b][j]:
                    r.keep(rows)
            for (codes, scales), r in zip(p.read(b, j, len(rows)), p.rows[b][j]):
                assert same(scales, np.asarray(r.scales)[: len(scales)]), (b, j)
                assert same(codes, r.codes), (b, j, np.abs(codes - r.codes).max())


@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 96, 112, 128, 20, 256])
@pytest.mark.parametrize("smallest", [1, 2, 3, 4])
def test_evict_of_the_row_that_made_the_scale(hd, smallest):
    """What stays is 1 to 4 smallest codes: its scale is up to 2^17 times smaller, its codes up to 2^17 times larger."""
    loud_rows_go(hd, [smallest], 448.0)


@pytest.mark.parametrize("hd", [16, 64, 128, 48, 20])
@pytest.mark.parametrize("smallest", [(1, 4), (3, 1, 2), (1, 0), (2, 0, 1, 3)])
def test_evict_of_loud_rows_beside_other_pages(hd, smallest):
    """The same among rows of other pages, whose codes grow by less or shrink."""
    loud_rows_go(hd, smallest, 256.0, held=(700, 64, 300), budget=200, recent=9)


@pytest.mark.parametrize("hd", [16, 64, 128, 20])
@pytest.mark.parametrize("large", [2.0 ** 119, 2.0 ** 20, 1.0])
def test_evict_leaves_rows_of_zeros(hd, large):
    """Zeros beside rows that go, and beside others that stay, under scales up to the largest: they are zeros under any scale."""
    p = Pages([300], 2, hd, seed=12, weights=True)
    rng = np.random.default_rng(12)
    for j in range(2):
        for r in p.rows[0][j]:
            r.codes = np.zeros((300, hd))
            r.codes[::8] = rng.choice([-448.0, 256.0], (38, hd))
            r.codes[200:] = rng.integers(-2, 3, (100, hd)) * 2.0 ** -9
            r.scales = [large] * 3 + [2.0 ** -20] * 2
        p.gathered[0][j][:] = 1.0
        p.gathered[0][j][:200:8] = 0.0
    p.write(0)
    s = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None])
    ops.kv_evict_e4m3(s, ints(p.slots), ints([300]), 300, 260, 30)
    for j in range(2):
        rows = plain.chosen(p.gathered[0][j].tolist(), 260, 30)
        for (codes, scales), r in zip(p.read(0, j, 260), p.rows[0][j]):
            r.keep(rows)
            assert same(scales, np.asarray(r.scales)) and same(codes, r.codes), j


@pytest.mark.parametrize("hd", [64, 20])
def test_evict_keeps_rows_whose_weight_is_no_number(hd):
    """A weight that is NaN, of either sign, is above all others: nobody knows what its row is worth."""
    p = Pages([300], 2, hd, seed=9, weights=True)
    for j, bad in enumerate(([7, 100, 210], [0, 64, 127])):
        p.gathered[0][j][:] = 1 + np.arange(300) % 7
    p.write(0)
    nan = torch.tensor([0x7FC00000, -0x400000, 0x7F800001], dtype=torch.int32, device=DEV).view(torch.float32)
    for j, bad in enumerate(([7, 100, 210], [0, 64, 127])):
        for row, x in zip(bad, nan):
            p.weights[p.pages[0][row // 64], j, row % 64] = x
            p.gathered[0][j][row] = np.inf
    s = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None])
    kept = ops.kv_evict_e4m3(s, ints(p.slots), ints([300]), 300, 40, 10).cpu().numpy()
    for j in range(2):
        assert kept[0, 0, j].tolist() == plain.chosen(p.gathered[0][j].tolist(), 40, 10)
