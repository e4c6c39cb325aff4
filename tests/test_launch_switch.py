"""The switch of a library that lets kernels begin early is its caller's: no launch turns it."""
import os
import re

import pytest

from go_tinygrad_b200.kernels import build


def sources():
    return sorted(f for f in os.listdir(build.CSRC) if f.endswith((".cu", ".cuh", ".h")))


@pytest.mark.parametrize("name", sources())
def test_only_its_setter_turns_the_switch(name):
    """Calls come from several threads at once (ctypes lets the others run): one that turned the switch on for a launch and put
    back what it had read could put back another's."""
    with open(os.path.join(build.CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    written = re.findall(r"[^\n]*\bg_chained_launch\b\s*(?:[-+|&^]?=(?!=)|\+\+|--)[^\n]*", text)
    taken = re.findall(r"&\s*g_chained_launch\b", text)
    allowed = ["static int g_chained_launch = 0;", "GTG_API void gtg_set_chained_launch(int on) { g_chained_launch = on ? 1 : 0; }"]
    assert [w.strip() for w in written] == (allowed if name == "common.cuh" else []) and not taken


def test_a_call_reads_the_switch_once():
    """Few queries: whether the kernel reads older pages before its wait, and whether it is launched to begin early, are one answer."""
    text = "".join(open(os.path.join(build.CSRC, f)).read() for f in ("attention_e4m3.cu", "attention_e4m3_few.cuh"))
    assert len(re.findall(r"\bg_chained_launch\b", text)) == 1 and "launch_chained(few_queries_kernel" not in text
