"""Calls of the 8-bit cache from two threads at once, each on a stream and a cache of its own, and the order of chained kernels."""
import threading

import pytest
import torch

from go_tinygrad_b200.cache import E4M3Storage
from go_tinygrad_b200.kernels import ops
from test_e4m3_gpu import BF16, DEV, F32, Pages, cut, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,new", [(F32, 1), (BF16, 1), (BF16, 70), (F32, 40)])
def test_two_threads(dtype, new):
    """Steps that store, attend and, at the end, evict: the bits of one thread alone."""
    held, heads, n_kv, hd, steps = 1100, 4, 2, 64, 6

    def prepare(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        p = Pages([held], n_kv, hd, seed=seed, weights=True, dropped=[0], room=steps * new)
        qkv = [torch.randn(new, (heads + 2 * n_kv) * hd, device=DEV, generator=g).to(dtype) for _ in range(steps)]
        return p, qkv, cut([new]), ints(p.slots), [ints([held + new * t]) for t in range(steps)]

    def run(state, outs, times=1):
        p, qkv, cu, slots, starts = state
        kv = p.view()
        kept = [x.clone() for x in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights, p.dropped)]
        for _ in range(times):
            for x, y in zip((p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights, p.dropped), kept):
                x.copy_(y)
            for t in range(steps):
                q, out = torch.empty(new, heads * hd, dtype=dtype, device=DEV), torch.empty(new, heads * hd, dtype=dtype, device=DEV)
                ops.kv_store_e4m3(qkv[t], None, heads, n_kv, kv, cu, slots, starts[t], new, q)
                ops.attention_e4m3(q, out, kv, cu, slots, starts[t], new, heads, 0.125, max_kv_len=held + steps * new)
                outs.append(out)
            s = E4M3Storage(p.k[None], p.v[None], p.scales[None], p.table, weights=p.weights[None], dropped=p.dropped)
            outs.append(ops.kv_evict_e4m3(s, slots, ints([held + steps * new]), held + steps * new, 700, 100))
            outs += [x.clone() for x in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales, p.weights)]
    want = []
    for seed in (1, 2):
        want.append([])
        run(prepare(seed), want[-1])
    states, got, errors = [prepare(seed) for seed in (1, 2)], [[], []], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                run(states[i], got[i], times=25)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 - shown below
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(2):
        n = len(want[i])
        assert len(got[i]) == 25 * n
        for at, x in enumerate(got[i]):
            assert torch.equal(x, want[i][at % n]), (i, at)


@pytest.mark.parametrize("weights", [False, True])
def test_a_prompt_step_of_no_tokens_keeps_the_order(weights):
    """Chained kernels: rotation of many rows that are nobody's, attention of sequences that bring nothing, and a second rotation into
    the last of those rows, which must come last."""
    heads, hd, n = 32, 128, 6000
    p = Pages([300, 70], 2, hd, seed=4, weights=weights)
    nothing = ints([0, 0, 0])
    first, second = torch.randn(n, heads * hd, device=DEV).bfloat16(), torch.randn(8, heads * hd, device=DEV).bfloat16()
    qkv = torch.cat([first, torch.zeros(n, 4 * hd, device=DEV).bfloat16()], 1)
    other = torch.cat([second, torch.zeros(8, 4 * hd, device=DEV).bfloat16()], 1)
    before = [x.clone() for x in (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales)]
    kv, slots, start, out = p.view(), ints(p.slots), ints([300, 70]), torch.full((n, heads * hd), 7.0, device=DEV).bfloat16()
    q = torch.empty(n, heads * hd, dtype=BF16, device=DEV)
    with ops.chained_launches():
        for _ in range(20):
            q.zero_()
            ops.kv_store_e4m3(qkv, None, heads, 2, kv, nothing, slots, start, 200, q)
            ops.attention_e4m3(q, out, kv, nothing, slots, start, 200, heads, 0.1, max_kv_len=300)
            ops.kv_store_e4m3(other, None, heads, 2, kv, nothing, slots, start, 200, q[n - 8:])
            assert torch.equal(q[: n - 8], first[: n - 8]) and torch.equal(q[n - 8:], second)
    assert (out == 7.0).all() and all(torch.equal(a, b) for a, b in zip(before, (p.k.view(torch.uint8), p.v.view(torch.uint8), p.scales)))
    if weights:
        assert (p.read_weights(0, 0, 300).astype("float32") == p.gathered[0][0].astype("float32")).all()
