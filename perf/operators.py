"""Measured cases of the 8-bit cache: storing a step's keys and values, attention over the cache, eviction.

Storage, per layer run: pages of 64 rows (tokens); keys [page, head, row, channel], values [page, head, channel, row], both in
float8 (e4m3) as code * scale with one power of two a (page, keys | values, head); where the cache evicts, the attention weight
each row has gathered, float32 [page, head, row].  `block_table[slot, i]` is the page of a sequence's rows 64 i .. 64 i + 63."""
import math

import torch

own = False

PAGE = 64
LEAST = -126                 # exponent of the least scale


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # a decode step of eight sequences at the size of the framework's benchmark model: latency
        dict(name="store decode 8x32x64", op="store", dtype="bfloat16", seqs=8, q_lo=1, q_hi=1, past_lo=500, past_hi=2200, heads=32, kv_heads=32,
             dim=64, rot=64, pairing="half", keep=0),
        # four prompts of unequal lengths, grouped heads of 128 channels, rows of a cache that evicts
        dict(name="store prompts 4x2048 8x128", op="store", dtype="bfloat16", seqs=4, q_lo=300, q_hi=2048, past_lo=0, past_hi=0, heads=32, kv_heads=8,
             dim=128, rot=128, pairing="half", keep=1),
        # one request behind an ordinary prompt: the smallest serving call
        dict(name="decode 1x2251 32x64", op="attend", dtype="bfloat16", seqs=1, q_lo=1, q_hi=1, past_lo=2250, past_hi=2250, heads=32, kv_heads=32,
             dim=64, window=0, keep=0),
        # the benchmark's headline decode step: eight sequences of 8,192 tokens
        dict(name="decode 8x8192 32x64", op="attend", dtype="bfloat16", seqs=8, q_lo=1, q_hi=1, past_lo=8191, past_hi=8191, heads=32, kv_heads=32,
             dim=64, window=0, keep=0),
        # a full batch of unequal lengths, four query heads on each key head of 128 channels
        dict(name="decode 64 ragged 8x128", op="attend", dtype="bfloat16", seqs=64, q_lo=1, q_hi=1, past_lo=130, past_hi=2300, heads=32, kv_heads=8,
             dim=128, window=0, keep=0),
        # decode steps that gather attention weights for the eviction, four query heads on a key head of 64
        dict(name="decode 8x4100 8x64 weights", op="attend", dtype="bfloat16", seqs=8, q_lo=1, q_hi=1, past_lo=3900, past_hi=4100, heads=32, kv_heads=8,
             dim=64, window=0, keep=1),
        # one prompt of the benchmark's length
        dict(name="prompt 2048 32x64", op="attend", dtype="bfloat16", seqs=1, q_lo=2048, q_hi=2048, past_lo=0, past_hi=0, heads=32, kv_heads=32,
             dim=64, window=0, keep=0),
        # chunks of long prompts: 512 new tokens behind thousands
        dict(name="chunk 512 of 8192 8x128", op="attend", dtype="bfloat16", seqs=2, q_lo=500, q_hi=512, past_lo=7000, past_hi=7680, heads=32, kv_heads=8,
             dim=128, window=0, keep=0),
        # prompts of unequal lengths whose attention weights are gathered
        dict(name="prompts 3x1500 8x64 weights", op="attend", dtype="bfloat16", seqs=3, q_lo=200, q_hi=1500, past_lo=0, past_hi=0, heads=32, kv_heads=8,
             dim=64, window=0, keep=1),
        # the 32-bit path: a decode step at an odd head size, three query heads on one key head, a sliding window
        dict(name="decode f32 4x700 3x48 window", op="attend", dtype="float32", seqs=4, q_lo=1, q_hi=1, past_lo=600, past_hi=700, heads=3, kv_heads=1,
             dim=48, window=450, keep=0),
        # one sequence a page over its budget, all layers of a small model
        dict(name="evict 1x576 to 512", op="evict", entries=16, seqs=1, len_lo=576, len_hi=576, budget=512, recent=128, kv_heads=8, dim=64),
        # four sequences of the benchmark model cut back in one go, one of them within its budget
        dict(name="evict 4x2112 to 2000", op="evict", entries=24, seqs=4, len_lo=1950, len_hi=2112, budget=2000, recent=500, kv_heads=32, dim=64),
    ]


def _spread(lo, hi, n):
    """n whole numbers over lo..hi, the ends among them, in no order."""
    if n == 1 or lo == hi:
        return [hi] * n
    at = sorted(range(n), key=lambda i: (i * 0.6180339887498949) % 1.0)
    return [lo + (hi - lo) * at[i] // (n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, rows before them) of each sequence."""
    return _spread(case["q_lo"], case["q_hi"], case["seqs"]), list(reversed(_spread(case["past_lo"], case["past_hi"], case["seqs"])))


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "evict"])
    dim = rng.choice([16, 32, 48, 64, 64, 80, 96, 112, 128, 128])
    if op == "evict":
        while True:
            length = _log_uniform(rng, 66, 4000)
            budget = rng.randint(max(1, length // 4), length)
            c = dict(op=op, entries=rng.randint(1, 24), seqs=_log_uniform(rng, 1, 8), len_lo=rng.randint(max(1, length // 2), length), len_hi=length,
                     budget=budget, recent=rng.randint(0, budget), kv_heads=rng.choice([1, 2, 3, 8, 16, 32]), dim=dim)
            if c["entries"] * c["seqs"] * length * c["kv_heads"] * dim <= 24 * 4 * 2112 * 32 * 64:
                return c
    dtype = rng.choice(["bfloat16"] * 4 + ["float32"])
    kv_heads = rng.choice([1, 2, 3, 5, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    heads = heads if heads <= 64 else kv_heads
    keep = rng.choice([0, 0, 1])
    while True:
        if rng.random() < 0.5:                                      # single tokens behind what is there
            seqs, q_hi, past = _log_uniform(rng, 1, 64), 1, _log_uniform(rng, 1, 16000)
        else:                                                       # prompts and chunks
            seqs, q_hi, past = _log_uniform(rng, 1, 8), _log_uniform(rng, 2, 2500), rng.choice([0, 0, _log_uniform(rng, 1, 8000)])
        c = dict(op=op, dtype=dtype, seqs=seqs, q_lo=rng.randint((q_hi + 1) // 2, q_hi), q_hi=q_hi, past_lo=past // rng.randint(1, 3), past_hi=past,
                 heads=heads, kv_heads=kv_heads, dim=dim)
        if op == "store":
            c.update(rot=rng.choice([dim, dim, dim // 2]), pairing=rng.choice(["half", "half", "interleaved"]), keep=keep)
            if work(c)["bytes"] <= 5e7 and seqs * past * kv_heads * dim <= 8 * 8192 * 32 * 64:
                return c
            continue
        c.update(window=rng.choice([0, 0, 0, rng.randint(1, 2 * (past + q_hi))]), keep=keep)
        if c["window"]:
            c["keep"] = 0                                           # layers with a window forget by themselves
        w = work(c)
        most = 2e9 if dtype == "float32" else 1.2e11
        # (the padded form of the products is what the plain side computes)
        padded = seqs * heads * q_hi * (past + q_hi)
        if w["flops"] <= most and w["bytes"] <= 2.6e8 and padded <= 6e8 and seqs * (past + q_hi) * kv_heads * dim <= 8 * 8192 * 32 * 64:
            return c


def work(case):
    if case["op"] == "evict":
        lengths = _spread(case["len_lo"], case["len_hi"], case["seqs"])
        per = case["entries"] * case["kv_heads"]
        over = [n for n in lengths if n > case["budget"]]
        # weights read; kept rows (codes, weight) read and written, a number for each of them
        return {"bytes": per * (4 * sum(over) + len(over) * case["budget"] * 2 * (2 * case["dim"] + 4) + 4 * case["seqs"] * case["budget"]),
                "flops": per * sum(over)}
    new, past = _lengths(case)
    n, size = sum(new), 2 if case["dtype"] == "bfloat16" else 4
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "store":
        blocks = sum((p + q - 1) // PAGE - p // PAGE + 1 for q, p in zip(new, past))
        return {"bytes": n * (2 * heads + 2 * kv_heads) * dim * size + n * case["rot"] * 4 + n * 2 * kv_heads * dim + blocks * 2 * kv_heads * 4
                + case["keep"] * n * kv_heads * 4, "flops": n * (heads + 2 * kv_heads) * dim * 4}
    window = case["window"] or 1 << 60
    seen = sum(sum(min(p + i + 1, window) for i in range(q)) for q, p in zip(new, past))
    rows = sum(min(p + q, window + q - 1) for q, p in zip(new, past))
    # gathered weights need every row's final maximum and sum: the products of queries and keys a second time, but for single tokens
    twice = case["keep"] * (1 if case["q_hi"] > 1 else 0)
    return {"bytes": 2 * n * heads * dim * size + rows * kv_heads * (2 * dim + 8 * case["keep"]) + rows // PAGE * 8 * kv_heads,
            "flops": (4 + 2 * twice) * heads * dim * seen}


# --------------------------------------------------------------------------- inputs
def _codes(g, shape, channel_axis):
    """Random codes: normal values, a few channels several times as large as the others."""
    x = torch.randn(shape, generator=g, device="cuda")
    n = shape[channel_axis]
    loud = torch.where(torch.rand(n, generator=g, device="cuda") < 0.06, 4.0, 1.0)
    x *= 24.0 * loud.reshape([n if a == channel_axis else 1 for a in range(len(shape))])
    return x.clamp_(-448, 448).to(torch.float8_e4m3fn)


def _pages(g, case, lengths):
    """Pages handed out in no order to len(lengths) slots, and a block table in slots that are not the sequences' order."""
    n_slots = len(lengths) + 1
    counts = [(n + PAGE - 1) // PAGE for n in lengths]
    order = torch.randperm(sum(counts) + 2, generator=g, device="cuda").to(torch.int32)
    slots = torch.randperm(n_slots, generator=g, device="cuda")[: len(lengths)].to(torch.int32)
    table = torch.zeros(n_slots, max(counts) + 1, dtype=torch.int32, device="cuda")
    host_slots, o = slots.tolist(), 0
    for slot, c in zip(host_slots, counts):
        table[slot, :c] = order[o: o + c]
        o += c
    return table, slots, sum(counts) + 2


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv_heads, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        lengths = _spread(case["len_lo"], case["len_hi"], case["seqs"])
        table, slots, n_pages = _pages(g, case, lengths)
        lead = (case["entries"], n_pages)
        k, v = _codes(g, lead + (kv_heads, PAGE, dim), 4), _codes(g, lead + (kv_heads, dim, PAGE), 3)
        # gathered weight: a few rows have most of it, many have next to none, some have the same
        w = torch.rand(lead + (kv_heads, PAGE), generator=g, device="cuda").pow_(8).mul_(40.0)
        w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.2, (w * 16).floor() / 16, w)
        return dict(case=dict(case), k=k, v=v, scales=_scales(g, lead + (2, kv_heads)), weights=w, block_table=table, slots=slots, lengths=_ints(lengths),
                    dropped=torch.zeros(table.shape[0], dtype=torch.int32, device="cuda"), max_length=max(lengths),
                    kept=torch.zeros(case["entries"], case["seqs"], kv_heads, case["budget"], dtype=torch.int32, device="cuda"))
    new, past = _lengths(case)
    dtype = getattr(torch, case["dtype"])
    heads = case["heads"]
    table, slots, n_pages = _pages(g, case, [q + p for q, p in zip(new, past)])
    k, v = _codes(g, (n_pages, kv_heads, PAGE, dim), 3), _codes(g, (n_pages, kv_heads, dim, PAGE), 2)
    s = dict(case=dict(case), block_table=table, slots=slots, k=k, v=v, scales=_scales(g, (n_pages, 2, kv_heads)), start_pos=_ints(past),
             weights=torch.rand(n_pages, kv_heads, PAGE, generator=g, device="cuda") if case["keep"] else None,
             cu_seqlens=_ints([sum(new[:i]) for i in range(len(new) + 1)]), max_q_len=max(new),
             max_kv_len=max(q + p for q, p in zip(new, past)), total_kv_len=sum(new) + sum(past))
    n = sum(new)
    filled = past if case["op"] == "store" else [q + p for q, p in zip(new, past)]
    host_slots = slots.tolist()
    for slot, rows in zip(host_slots, filled):                      # rows of a last page that nobody has written yet hold anything, NaN too
        if rows % PAGE:
            page = int(table[slot, rows // PAGE])
            k[page].view(torch.uint8)[:, rows % PAGE:] = 0x7F
            v[page].view(torch.uint8)[:, :, rows % PAGE:] = 0x7F
    if case["op"] == "store":
        width = heads + 2 * kv_heads
        qkv = torch.randn(n, width, dim, generator=g, device="cuda") * 1.3
        qkv[:, :, :: max(1, dim // 5)] *= 3.0
        s["qkv"] = qkv.reshape(n, width * dim).to(dtype)
        inv = 10000.0 ** (-2.0 * torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda") / case["rot"])
        pos = torch.cat([torch.arange(p, p + q, dtype=torch.float64, device="cuda") for q, p in zip(new, past)])
        angle = pos[:, None] * inv
        s["cos_sin"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
        s["q"] = torch.empty(n, heads * dim, dtype=dtype, device="cuda")
        return s
    s["q"] = (torch.randn(n, heads * dim, generator=g, device="cuda") * 1.5).to(dtype)
    s["out"] = torch.empty(n, heads * dim, dtype=dtype, device="cuda")
    s["scale"] = dim ** -0.5
    return s


def _scales(g, shape):
    return torch.exp2(torch.randint(-6, -3, shape, generator=g, device="cuda").float())


# --------------------------------------------------------------------------- the operators
_modules = []


def _framework():
    if not _modules:
        import go_tinygrad_b200
        _modules.append((go_tinygrad_b200.cache, go_tinygrad_b200.kernels.ops))
    return _modules[0]


def _handle(s):
    """The cache's handle, which a program has from its cache and keeps: made once a state."""
    if "handle" not in s:
        cache, _ = _framework()
        kind = cache.E4M3Storage if s["k"].dim() == 5 else cache.E4M3KVView
        s["handle"] = kind(s["k"], s["v"], s["scales"], s["block_table"], window=s["case"].get("window") or None, weights=s["weights"],
                           dropped=s.get("dropped"))
    return s["handle"]


def run(s):
    c = s["case"]
    if c["op"] == "store":
        if own:
            _, ops = _framework()
            ops.kv_store_e4m3(s["qkv"], s["cos_sin"], c["heads"], c["kv_heads"], _handle(s), s["cu_seqlens"], s["slots"], s["start_pos"],
                              s["max_q_len"], s["q"], pairing=c["pairing"], rotary_dim=c["rot"])
        else:
            _plain_store(s, c)
        return {"q": s["q"], "k": s["k"], "v": s["v"], "scales": s["scales"], "weights": s["weights"]}
    if c["op"] == "attend":
        if own:
            _, ops = _framework()
            ops.attention_e4m3(s["q"], s["out"], _handle(s), s["cu_seqlens"], s["slots"], s["start_pos"], s["max_q_len"], c["heads"], s["scale"],
                               max_kv_len=s["max_kv_len"], total_kv_len=s["total_kv_len"])
        else:
            _plain_attend(s, c)
        return {"out": s["out"], "weights": s["weights"]}
    if own:
        _, ops = _framework()
        ops.kv_evict_e4m3(_handle(s), s["slots"], s["lengths"], s["max_length"], c["budget"], c["recent"], kept=s["kept"])
    else:
        _plain_evict(s, c)
    return {"k": s["k"], "v": s["v"], "scales": s["scales"], "weights": s["weights"], "dropped": s["dropped"], "kept": s["kept"]}


def _needed(most):
    """The least power of two (from 2^-126 on) that `most` / 448 does not exceed, for finite `most` >= 0."""
    mantissa, exponent = torch.frexp(most)                          # most = mantissa * 2^exponent, mantissa in [0.5, 1)
    k = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    k = torch.where(most > 0, k, torch.full_like(k, LEAST)).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(most), k)


def _finite(x):
    return torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))


def _rotated(x, cos_sin, pairing):
    """x [N, heads, channels] in float, the first channels turned in pairs."""
    rot = 2 * cos_sin.shape[1]
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairing == "interleaved" else (x[..., : rot // 2], x[..., rot // 2: rot])
    if pairing == "interleaved":
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        y[..., : rot // 2], y[..., rot // 2: rot] = a * c - b * s, a * s + b * c
    return y


def _plain_store(s, c):
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    n = s["qkv"].shape[0]
    x = s["qkv"].float().reshape(n, heads + 2 * kv_heads, dim)
    turned = _rotated(x[:, : heads + kv_heads], s["cos_sin"], c["pairing"])
    s["q"].copy_(turned[:, :heads].reshape(n, heads * dim))
    start, cu, slots = s["start_pos"].long(), s["cu_seqlens"].long(), s["slots"].long()
    q_len = cu[1:] - cu[:-1]
    dev = start.device
    # blocks of 64 rows that the step's tokens fall into
    block = start[:, None] // PAGE + torch.arange((s["max_q_len"] + PAGE - 2) // PAGE + 1, device=dev)
    row = block[..., None] * PAGE + torch.arange(PAGE, device=dev)
    new = (row >= start[:, None, None]) & (row < (start + q_len)[:, None, None])
    b, j = new.any(-1).nonzero(as_tuple=True)
    new, row, block = new[b, j], row[b, j], block[b, j]
    page = s["block_table"].long()[slots[b], block]
    token = (cu[b][:, None] + row - start[b][:, None]).clamp(0, n - 1)
    older = row < start[b][:, None]
    fresh = ~older.any(-1)
    for plane, codes, values in ((0, s["k"], turned[:, heads:]), (1, s["v"], x[:, heads + kv_heads:])):
        got = values[token]                                         # [blocks, row, head, channel]
        need = _needed((_finite(got) * new[:, :, None, None]).amax(dim=(1, 3)))
        before = s["scales"][page, plane]
        scale = torch.where(fresh[:, None], need, torch.maximum(before, need))
        ratio = torch.where(fresh[:, None], torch.ones_like(before), before / scale)
        old = codes[page].float()
        old = old if plane == 0 else old.transpose(2, 3)            # [blocks, head, row, channel]
        kept = (old * ratio[:, :, None, None]).to(torch.float8_e4m3fn)
        put = (got.transpose(1, 2) / scale[:, :, None, None]).to(torch.float8_e4m3fn)
        as_is = old.to(torch.float8_e4m3fn).view(torch.uint8)
        out = torch.where(new[:, None, :, None], put.view(torch.uint8), torch.where(older[:, None, :, None], kept.view(torch.uint8), as_is))
        codes.view(torch.uint8)[page] = out if plane == 0 else out.transpose(2, 3)
        s["scales"][page, plane] = scale
    if s["weights"] is not None:
        s["weights"][page] = torch.where(new[:, None, :], 0.0, s["weights"][page])


def _plain_attend(s, c):
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    start, cu, slots = s["start_pos"].long(), s["cu_seqlens"].long(), s["slots"].long()
    q_len = cu[1:] - cu[:-1]
    seqs, group, dev = start.numel(), heads // kv_heads, start.device
    n_blocks = (s["max_kv_len"] + PAGE - 1) // PAGE
    length = start + q_len
    page = s["block_table"].long()[slots, :n_blocks]
    row = torch.arange(n_blocks * PAGE, device=dev)
    there = row < length[:, None]                                   # [sequence, row]
    k = s["k"][page].float() * s["scales"][page, 0][..., None, None]            # [sequence, block, head, row, channel]
    v = s["v"][page].float() * s["scales"][page, 1][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, -1, dim)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kv_heads, -1, dim)
    k = torch.where(there[:, None, :, None], k, torch.zeros_like(k))
    v = torch.where(there[:, None, :, None], v, torch.zeros_like(v))
    at = torch.arange(s["max_q_len"], device=dev)
    real = at < q_len[:, None]                                      # [sequence, query]
    token = (cu[:-1, None] + at).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][token].float().reshape(seqs, -1, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, -1, dim)
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    score = score.reshape(seqs, kv_heads, group, -1, row.numel())
    pos = start[:, None] + at
    seen = (row <= pos[..., None]) & there[:, None, :]
    if c["window"]:
        seen &= row > pos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.reshape(seqs, kv_heads, -1, row.numel()) @ v).reshape(seqs, kv_heads, group, -1, dim).permute(0, 3, 1, 2, 4)
    b, i = real.nonzero(as_tuple=True)
    s["out"][token[b, i]] = o[b, i].reshape(-1, heads * dim).to(s["out"].dtype)
    if s["weights"] is not None:
        gathered = (p * real[:, None, None, :, None]).sum(dim=(2, 3)).reshape(seqs, kv_heads, n_blocks, PAGE).transpose(1, 2)
        used = there.reshape(seqs, n_blocks, PAGE).any(-1)
        s["weights"][page[used]] += gathered[used] * there.reshape(seqs, n_blocks, 1, PAGE)[used]


def _plain_evict(s, c):
    budget, recent, kv_heads = c["budget"], c["recent"], c["kv_heads"]
    entries, seqs = c["entries"], c["seqs"]
    length, slots = s["lengths"].long(), s["slots"].long()
    dev = length.device
    n_blocks = (s["max_length"] + PAGE - 1) // PAGE
    rows = n_blocks * PAGE
    page = s["block_table"].long()[slots, :n_blocks]
    row = torch.arange(rows, device=dev)
    over = length > budget
    w = s["weights"][:, page].permute(0, 1, 3, 2, 4).reshape(entries, seqs, kv_heads, rows)
    candidate = row < (length - recent)[:, None]
    w = torch.where(candidate[None, :, None], w, torch.full_like(w, -math.inf))
    heaviest = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., : budget - recent]
    newest = (length[:, None] - recent + torch.arange(recent, device=dev))[None, :, None].expand(entries, seqs, kv_heads, recent)
    chosen = torch.cat([heaviest, newest], dim=-1).sort(dim=-1).values
    whole = torch.arange(budget, device=dev).expand(entries, seqs, kv_heads, budget)
    kept = torch.where(over[None, :, None, None], chosen, torch.where(whole < length[:, None, None], whole, -1))
    s["kept"].copy_(kept)
    s["dropped"][slots] += (length - budget).clamp(min=0).to(torch.int32)
    # blocks of the compacted rows; the last one may end before its 64th row
    new_blocks = (budget + PAGE - 1) // PAGE
    pad = new_blocks * PAGE - budget
    source = torch.nn.functional.pad(kept, (0, pad), value=-1).clamp(min=0)
    real = (torch.arange(new_blocks * PAGE, device=dev) < budget) & (over[:, None])           # [sequence, row]
    moved = ((source != torch.arange(new_blocks * PAGE, device=dev)) & real[None, :, None]).reshape(entries, seqs, kv_heads, new_blocks, PAGE).any(-1)
    to = page[:, :new_blocks]
    e = torch.arange(entries, device=dev)[:, None, None, None]
    h = torch.arange(kv_heads, device=dev)[None, None, :, None]
    from_page = torch.gather(page[None, :, None].expand(entries, seqs, kv_heads, n_blocks), 3, source // PAGE)
    real = real.reshape(1, seqs, 1, new_blocks, PAGE)
    target = to[None, :, None].expand(entries, seqs, kv_heads, new_blocks)
    shape = (entries, seqs, kv_heads, new_blocks, PAGE)
    results = []
    for plane, codes in ((0, s["k"]), (1, s["v"])):
        flat = codes if plane == 0 else codes.transpose(3, 4)
        got = flat[e, from_page, h, source % PAGE].float() * s["scales"][e, from_page, plane, h][..., None]
        got = got.reshape(shape + (c["dim"],))
        scale = _needed((_finite(got) * real[..., None]).amax(dim=(4, 5)))
        put = (got / scale[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
        was = flat.view(torch.uint8)[e, target, h]
        results.append((plane, codes, torch.where((real & moved[..., None])[..., None], put, was),
                        torch.where(moved, scale, s["scales"][e, target, plane, h])))
    weights = s["weights"][e, from_page, h, source % PAGE].reshape(shape)
    weights = torch.where(real & moved[..., None], weights, s["weights"][e, target, h])
    # (where two sequences are cut, their pages are their own: no page is written twice.  A sequence may have fewer blocks than the budget.)
    has = torch.arange(new_blocks, device=dev) * PAGE < length[:, None]
    at = has[None, :, None].expand(entries, seqs, kv_heads, new_blocks).nonzero(as_tuple=True)
    page_at = target[at]
    for plane, codes, put, scale in results:
        codes.view(torch.uint8)[at[0], page_at, at[2]] = put[at] if plane == 0 else put[at].transpose(1, 2)
        s["scales"][at[0], page_at, plane, at[2]] = scale[at]
    s["weights"][at[0], page_at, at[2]] = weights[at]


# --------------------------------------------------------------------------- from the definition, in 64 bits
def _nearest(x):
    """The nearest number with 3 bits behind the point and exponents from -6 (a fixed step of 2^-9 below), ties to even; NaN for what is not finite."""
    x = x.double()
    _, exponent = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (exponent - 1).clamp(min=-6) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, torch.full_like(x, math.nan))


def _power(most):
    """2^ceil(log2(most / 448)), not below 2^-126; the logarithm's rounding is put right."""
    k = torch.ceil(torch.log2(most.double().clamp(min=1e-300) / 448.0)).clamp(min=LEAST)
    k = torch.where(448.0 * torch.exp2(k - 1) >= most, k - 1, k)
    k = torch.where(448.0 * torch.exp2(k) < most, k + 1, k).clamp(min=LEAST)
    return torch.exp2(k)


def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s, case)


def _exact_store(s, c):
    heads, kv_heads, dim, rot = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    k, v, scales = s["k"].double(), s["v"].double(), s["scales"].double()
    weights = None if s["weights"] is None else s["weights"].double()
    x = s["qkv"].double().reshape(-1, heads + 2 * kv_heads, dim)
    # each pair as a complex number, turned by one of absolute value 1
    z = torch.complex(s["cos_sin"][..., 0].double(), s["cos_sin"][..., 1].double())[:, None]
    part = x[:, : heads + kv_heads, :rot]
    if c["pairing"] == "half":
        t = torch.complex(part[..., : rot // 2], part[..., rot // 2:]) * z
        part = torch.cat([t.real, t.imag], dim=-1)
    else:
        part = torch.view_as_real(torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * z).flatten(-2)
    turned = torch.cat([part, x[:, : heads + kv_heads, rot:]], dim=-1)
    table, slots, new, past = s["block_table"].tolist(), s["slots"].tolist(), *_lengths(c)
    first = 0
    for slot, q, p in zip(slots, new, past):
        for lo in range(p - p % PAGE, p + q, PAGE):
            page, a, e = table[slot][lo // PAGE], max(lo, p), min(lo + PAGE, p + q)
            fresh_k = turned[first + a - p: first + e - p, heads:].transpose(0, 1)             # [head, rows, channels]
            fresh_v = x[first + a - p: first + e - p, heads + kv_heads:].permute(1, 2, 0)
            for plane, codes, fresh in ((0, k[page], fresh_k), (1, v[page], fresh_v.transpose(1, 2))):
                view = codes if plane == 0 else codes.transpose(1, 2)
                most = torch.where(fresh.isfinite(), fresh.abs(), torch.zeros_like(fresh)).amax(dim=(1, 2))
                scale = _power(most)
                if a > lo:
                    scale = torch.maximum(scale, scales[page, plane])
                    view[:, : a - lo] = _nearest(view[:, : a - lo] * (scales[page, plane] / scale)[:, None, None])
                view[:, a - lo: e - lo] = _nearest(fresh / scale[:, None, None])
                scales[page, plane] = scale
            if weights is not None:
                weights[page, :, a - lo: e - lo] = 0.0
        first += q
    return {"q": turned[:, :heads].reshape(-1, heads * dim), "k": k, "v": v, "scales": scales, "weights": weights}


def _exact_attend(s, c):
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    group = heads // kv_heads
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    table, slots, new, past = s["block_table"], s["slots"].tolist(), *_lengths(c)
    first = 0
    for slot, q, p in zip(slots, new, past):
        n = p + q
        pages = table[slot, : (n + PAGE - 1) // PAGE].long()
        query = s["q"][first: first + q].double().reshape(q, kv_heads, group, dim)
        i, j = torch.arange(p, n, device="cuda")[:, None], torch.arange(n, device="cuda")
        hidden = (j > i) | (j <= i - c["window"]) if c["window"] else j > i
        for h in range(kv_heads):
            key = (s["k"][pages, h].double() * s["scales"][pages, 0, h].double()[:, None, None]).reshape(-1, dim)[:n]
            value = (s["v"][pages, h].double() * s["scales"][pages, 1, h].double()[:, None, None]).transpose(1, 2).reshape(-1, dim)[:n]
            logits = torch.einsum("qgd,kd->gqk", query[:, h], key) * s["scale"]
            p_all = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1)
            out[first: first + q, h * group * dim: (h + 1) * group * dim] = torch.einsum("gqk,kd->qgd", p_all, value).reshape(q, group * dim)
            if weights is not None:
                total = torch.zeros(pages.numel() * PAGE, dtype=torch.float64, device="cuda")
                total[:n] = p_all.sum(dim=(0, 1))
                weights[pages, h] += total.reshape(-1, PAGE)
        first += q
    return {"out": out, "weights": weights}


def _exact_evict(s, c):
    budget, recent, dim, kv_heads = c["budget"], c["recent"], c["dim"], c["kv_heads"]
    k, v, scales, weights = s["k"].float(), s["v"].float(), s["scales"].clone(), s["weights"].clone()
    kept = torch.full(s["kept"].shape, -1, dtype=torch.int32, device="cuda")
    dropped = s["dropped"].clone()
    head = torch.arange(kv_heads, device="cuda")
    blocks = [(lo, min(lo + PAGE, budget)) for lo in range(0, budget, PAGE)]
    for b, (slot, n) in enumerate(zip(s["slots"].tolist(), s["lengths"].tolist())):
        if n <= budget:
            kept[:, b, :, :n] = torch.arange(n, dtype=torch.int32, device="cuda")
            continue
        pages = s["block_table"][slot, : (n + PAGE - 1) // PAGE].long()
        dropped[slot] += n - budget
        for e in range(c["entries"]):
            mass = s["weights"][e, pages].transpose(0, 1).reshape(kv_heads, -1)
            order = (-mass[:, : n - recent].cpu().numpy()).argsort(axis=-1, kind="stable")[:, : budget - recent]
            at = torch.cat([torch.from_numpy(order).cuda().sort(dim=-1).values, torch.arange(n - recent, n, device="cuda").expand(kv_heads, recent)], dim=-1)
            kept[e, b] = at.int()
            rows = at[..., None].expand(kv_heads, budget, dim)
            key = s["k"][e, pages].double() * s["scales"][e, pages, 0].double()[..., None, None]
            value = s["v"][e, pages].double().transpose(2, 3) * s["scales"][e, pages, 1].double()[..., None, None]
            key, value = (x.transpose(0, 1).reshape(kv_heads, -1, dim).gather(1, rows) for x in (key, value))
            mass = mass.gather(1, at)
            for lo, hi in blocks:
                changed = head[(at[:, lo:hi] != torch.arange(lo, hi, device="cuda")).any(-1)]
                page = pages[lo // PAGE]
                for plane, x in ((0, key[changed, lo:hi]), (1, value[changed, lo:hi])):
                    most = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dim=(1, 2))
                    scale = _power(most)
                    scales[e, page, plane, changed] = scale.float()
                    code = _nearest(x / scale[:, None, None]).float()
                    if plane == 0:
                        k[e, page, changed, : hi - lo] = code
                    else:
                        v[e, page, changed, :, : hi - lo] = code.transpose(1, 2)
                weights[e, page, changed, : hi - lo] = mass[changed, lo:hi]
    return {"k": k, "v": v, "scales": scales, "weights": weights, "dropped": dropped, "kept": kept}
