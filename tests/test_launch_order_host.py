"""The order of tensor memory and early launches in the kernels' source (no GPU).

A kernel launched early begins once every CTA of the kernel before it has called allow_dependent_launch() or
ended, takes its tensor memory and then waits for that kernel's end. A CTA that calls it before it holds its own
columns could find them taken on its SM, and the two would wait for each other."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

SOURCES = sorted((Path(__file__).resolve().parents[1] / "faquant-public_b200" / "csrc").glob("*.cu"))


def _kernels(text):
    """``(name, body)`` of the kernels of a source, comments taken out."""
    text = re.sub(r"//[^\n]*", "", text)
    for match in re.finditer(r"__global__[^;{]*?(\w+)\s*\((?:[^(){}]|\([^()]*\))*\)\s*\{", text):
        depth, end = 1, match.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield match.group(1), text[match.end() : end]


KERNELS = [(name, body) for path in SOURCES for name, body in _kernels(path.read_text())]


def test_the_kernels_are_found() -> None:
    names = [name for name, _ in KERNELS]
    assert {"sparse_tile_kernel", "paged_chunk_kernel", "kv_append_kernel"} <= set(names)
    assert len(names) == sum(len(re.findall(r"__global__", re.sub(r"//[^\n]*", "", p.read_text()))) for p in SOURCES)


@pytest.mark.parametrize("name, body", [k for k in KERNELS if "tmem_alloc" in k[1]], ids=lambda x: x if len(x) < 60 else "")
def test_tensor_memory_is_held_before_the_next_kernel_may_begin(name, body) -> None:
    at = body.find("allow_dependent_launch()")
    if at < 0:
        return  # the next kernel begins at this one's end
    taken = body.index("tmem_alloc")
    assert taken < at and "__syncthreads()" in body[taken:at], name
