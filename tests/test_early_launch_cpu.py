"""Kernels that start while the kernel before them ends (programmatic launches): what their source has to keep to.

Such a kernel is resident while the one before it on the stream may still write its inputs.  So every thread waits before it
touches memory, and loads that promise memory which nothing writes during the kernel's life (``__ldg``, ``ld.global.nc``,
``const __restrict__`` pointers) are closed to it, before the wait and after.  No run can show that they are absent: a stale
line is a matter of schedules."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "maxsim_b200" / "csrc"
FILES = ["kv4.cu", "kv4_attend.cu", "kv4_chunk.cu", "pages.cu", "rotary.cu"]


def _plain(text):
    """Without comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def _block(text, at):
    """From `at` to the end of the first braces after it."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError("unbalanced braces")


def _kernels(text):
    out = {}
    for found in re.finditer(r"__global__", text):
        body = _block(text, found.start())
        out[re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", body)).group(1)] = body
    return out


@pytest.mark.parametrize("name", FILES)
def test_early_kernels_wait(name):
    text = _plain((CSRC / name).read_text())
    kernels, early = _kernels(text), set(re.findall(r"launch_early\(\s*(\w+)", text))
    assert early and early <= set(kernels)
    for kernel in early:
        assert "wait_for_previous()" in kernels[kernel], kernel


@pytest.mark.parametrize("name", FILES + ["quant4.cuh", "pages.cuh", "rotary.cuh"])
def test_early_kernels_do_not_promise_constant_memory(name):
    """Outside the kernels that are only ever launched normally there is one such load, and its template argument is
    whether the instance is launched early."""
    text = _plain((CSRC / name).read_text())
    early = set(re.findall(r"launch_early\(\s*(\w+)", text))
    for kernel, body in _kernels(text).items():
        if kernel not in early:
            text = text.replace(body, "")
    if name == "quant4.cuh":
        helper = _block(text, text.index("load_input"))
        assert helper.count("__ldg(") == 1 and "if constexpr (kEarly)" in helper
        text = text.replace(helper, "")
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", text)
    assert set(re.findall(r"load_input<(\w+)>", text)) <= {"kSparse"}
