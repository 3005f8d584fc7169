"""The order that programmatic dependent launches rely on, read from the kernels' sources: a kernel lets its
dependents start only after its own wait, so that whatever starts finds all kernels before its predecessor
finished.  A kernel that triggers without waiting must be launched without the attribute."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tfjs-core_b200", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu"))


def _kernels(text):
    """(name, body) of each __global__ function."""
    for m in re.finditer(r"__global__", text):
        open_brace = text.index("{", m.end())
        head = text[m.end():open_brace]
        if ";" in head:
            continue   # a declaration
        name = re.findall(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", head))[0]
        depth, at = 1, open_brace + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield name, text[open_brace:at]


def _read(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_the_reader_finds_the_kernels():
    assert {"embedding_sort_kernel", "embedding_sum_kernel", "embedding_join_kernel"} <= {n for n, _ in _kernels(_read("embedding.cu"))}


@pytest.mark.parametrize("source", SOURCES)
def test_waits_come_before_triggers(source):
    text = _read(source)
    for name, body in _kernels(text):
        trigger, wait = body.find("pdl_launch_dependents("), body.find("pdl_wait(")
        if trigger < 0:
            continue
        if wait >= 0:
            assert wait < trigger, name
        else:
            launches = re.findall(r"launch_(?:ex|dependent)\(ctx,\s*(\w+)", text)
            assert name not in launches, name
