"""What the attention over the 8-bit cache asks its library before a launch, without a GPU."""
import os
import re

import pytest
import torch

from go_tinygrad_b200.kernels import build, ops
from test_e4m3 import view


def c_arguments(source, symbol):
    with open(os.path.join(build.CSRC, source)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    arguments = re.search(r"\b%s\(([^)]*)\)" % symbol, text).group(1)
    return [re.sub(r"\s+", " ", a.strip()) for a in arguments.split(",")], text


@pytest.mark.parametrize("symbol", ["gtg_attention_e4m3_scratch_floats", "gtg_attention_e4m3", "gtg_attention_e4m3_tcgen05", "gtg_kv_store_e4m3",
                                    "gtg_kv_evict_e4m3"])
def test_every_argument_of_an_entry_is_used(symbol):
    library, types = ops._SIGNATURES[symbol]
    arguments, text = c_arguments(build.LIBRARIES[library], symbol)
    assert len(arguments) == len(types)
    body = text[re.search(r"\b%s\([^)]*\)\s*{" % symbol, text).end():]
    body = body[: body.index("\n}")]
    for a in arguments:
        name = re.search(r"(\w+)$", a).group(1)
        assert re.search(r"(?<!\(void\))\b%s\b" % name, body), name


def test_steps_that_differ_in_all_rows_only_ask_once(monkeypatch):
    """The rows of all sequences together change from step to step and decide nothing: one question for the scratch of a size."""
    asked = []

    def library(symbol):
        assert symbol == "gtg_attention_e4m3_scratch_floats"
        return lambda *numbers: asked.append(numbers) or 100
    monkeypatch.setattr(ops, "_fn", library)
    ops._e4m3_few_scratch.cache_clear()
    try:
        kv = view()
        for total in (0, 60, 61, 62, 10 ** 12):
            assert ops.attention_e4m3_scratch_floats(torch.float32, 2, 2, 1, 4, kv, 40, total) == 100
        assert len(asked) == 1 and len(asked[0]) == len(ops._SIGNATURES["gtg_attention_e4m3_scratch_floats"][1])
        ops.attention_e4m3_scratch_floats(torch.float32, 2, 2, 1, 4, kv, 41)
        assert len(asked) == 2
    finally:
        ops._e4m3_few_scratch.cache_clear()


def test_heads_that_the_attention_does_not_take():
    """A model with larger heads is refused when its cache is made, not in its first step; at the limit it is served."""
    from conftest import TINY_A
    from go_tinygrad_b200.config.registry import find_architecture
    from go_tinygrad_b200.engine.model import Model
    from go_tinygrad_b200.kernels import KernelError
    from go_tinygrad_b200.parts.base import Runtime
    arch = find_architecture(TINY_A)
    for dim in (256, 258, 320):
        model = Model(arch.plan(arch.read_config(dict(TINY_A, head_dim=dim))), Runtime(torch.device("cpu"), torch.bfloat16))
        assert all(h.kv.head_dim == dim for h in model.new_cache(128, 1).handles)
        if dim <= ops.E4M3_MAX_CHANNELS:
            assert all(h.kv.format == "e4m3" for h in model.new_cache(128, 1, kv_format="e4m3").handles)
        else:
            with pytest.raises(ValueError, match="entry 0 asks for keys and values that its mixer does not read"):
                model.new_cache(128, 1, kv_format="e4m3")
    q, one = torch.zeros(1, 4 * 272), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(KernelError, match="up to 256 channels, not 272"):
        ops.attention_e4m3(q, torch.zeros_like(q), view(dim=272), torch.tensor([0, 1], dtype=torch.int32), one, one, 1, 4, 0.1, max_kv_len=1)
