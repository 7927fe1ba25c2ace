"""Kernels that may start before the one ahead of them has ended: every thread waits for it before it can return, so that the end of a
kernel keeps implying the end of everything ahead of it (csrc/common.cuh)."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "csrc"


def kernels(text):
    """Names and bodies of the kernels of a source file, without comments."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__[^;{]*?(\w+)\s*\((?:[^(){}]|\([^(){}]*\))*\)\s*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


def returns_before_wait(body):
    """Whether a return of the kernel itself (not of a lambda in it) stands in front of its first wait."""
    wait = body.find("kb_dep_wait()")
    if wait < 0:
        return False
    head = body[:wait]
    while True:                                                  # lambdas: their returns are their own
        m = re.search(r"\[&?\]\s*(?:\([^()]*\))?\s*(?:->\s*\w+\s*)?\{", head)
        if not m:
            break
        depth, at = 1, m.end()
        while depth and at < len(head):
            depth += {"{": 1, "}": -1}.get(head[at], 0)
            at += 1
        head = head[:m.start()] + head[at:]
    return re.search(r"\breturn\b", head) is not None


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")), ids=lambda p: p.name)
def test_no_thread_returns_before_its_wait(path):
    assert [name for name, body in kernels(path.read_text()) if returns_before_wait(body)] == []


def test_the_reading_of_sources():
    text = (CSRC / "tree_attn_sm100.cu").read_text()
    assert {n for n, _ in kernels(text)} == {"tree_attn_kernel", "tree_merge_kernel"}
    assert returns_before_wait("if (n > 3) return; kb_dep_wait();") and not returns_before_wait("kb_dep_wait(); return;")
    assert not returns_before_wait("auto f = [&](int x) { return x; }; kb_dep_wait();")
    for p in CSRC.glob("*.cu"):
        text = re.sub(r"//[^\n]*", "", p.read_text())
        assert text.count("__global__") == len(list(kernels(text))), p.name
