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
