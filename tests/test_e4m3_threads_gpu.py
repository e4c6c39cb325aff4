"""Calls of the 8-bit cache from two threads at once, each on a stream and a cache of its own."""
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
