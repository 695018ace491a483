"""Kernels that may start before their predecessor on the stream has ended wait for it before they
read anything: checked on the sources, since a kernel that reads too early is right most of the time."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thunderkittens-sm7x_b200", "csrc")
FILES = ["attention_masked.cuh", "attention_paged.cuh", "kvcache.cuh"]
# p.x[0] and p.x[1] are parameters themselves, not what a pointer among them leads to.
READS = re.compile(r"\bp\.\w+\s*\[(?!\s*[01]\s*\])|[=(,;{]\s*\*\s*p\.\w+|\bids\s*\[|\brequest_of\s*\(|\bmake_item\s*\(|\btma_load\w*\s*\(|\breturn\b")


def kernels():
    """(file, name, body) of each kernel that is not launched in the ordinary way."""
    for file in FILES:
        with open(os.path.join(CSRC, file)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            if m.group(1) + "<<<" in text:
                continue
            begin = text.index("{", m.end())
            depth, at = 0, begin
            while True:
                depth += {"{": 1, "}": -1}.get(text[at], 0)
                if depth == 0:
                    break
                at += 1
            yield file, m.group(1), text[begin + 1:at]


FOUND = list(kernels())


def test_kernels_are_found():
    assert {n for _, n, _ in FOUND} >= {"plan_kernel", "plan_fill_kernel", "append_kernel", "paged_kernel", "join_kernel", "runs_kernel",
                                        "zero_kernel", "masked_kernel"}


@pytest.mark.parametrize("file,name,body", FOUND, ids=[n for _, n, _ in FOUND])
def test_waits_before_it_reads(file, name, body):
    """The first wait stands in the kernel's outermost block: every thread comes by it, and nothing
    that another kernel of the stream may write is read before."""
    assert "grid_wait()" in body
    before = body[:body.index("grid_wait()")]
    depth = before.count("{") - before.count("}")
    assert depth == 0, "the wait is inside a condition"
    # Bodies of lambdas run where they are called.
    while True:
        plain = re.sub(r"\{[^{}]*\}", "", before)
        if plain == before:
            break
        before = plain
    assert not READS.search(before), READS.search(before).group(0)
