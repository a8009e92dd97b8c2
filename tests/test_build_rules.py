"""What the build goes by: an object is made again when any of the repository's files that it includes has changed."""

from __future__ import annotations

import hashlib
import os
import re
import subprocess

import pytest

from pplx_kernels import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pplx-kernels_amd", "csrc")


def included(name: str, seen: set[str] | None = None) -> set[str]:
    """A source's own headers, and theirs."""
    seen = set() if seen is None else seen
    folder = next(d for d in (CSRC, os.path.join(ROOT, "include")) if os.path.exists(os.path.join(d, name)))
    with open(os.path.join(folder, name)) as f:
        for header in re.findall(r'^\s*#include "([^"]+)"', f.read(), re.M):
            if header not in seen:
                seen.add(header)
                included(header, seen)
    return seen


def prerequisites() -> dict[str, set[str]]:
    """Of every target, by the names of files: what make itself says."""
    said = subprocess.run(["make", "-C", CSRC, "-npqr"], capture_output=True, text=True).stdout
    found: dict[str, set[str]] = {}
    for line in said.splitlines():
        rule = re.match(r"^([^#\s:=][^:=]*\.o|[^#\s:=][^:=]*/bin/\w+): (.*)$", line)
        if rule:
            found.setdefault(os.path.basename(rule[1]), set()).update(os.path.basename(p) for p in rule[2].split())
    return found


RULES = prerequisites()
SOURCES = sorted(name for name in os.listdir(CSRC) if name.endswith((".hip", ".cpp")))


@pytest.mark.parametrize("source", SOURCES)
def test_objects_are_made_again_when_a_header_changes(source):
    stem = os.path.splitext(source)[0]
    target = f"{stem}.o" if f"{stem}.o" in RULES else stem
    assert included(source) - RULES[target] == set()


@pytest.mark.parametrize("made,sources", [
    ("headers_id", ["torch_common.h"]),
    ("experts_headers_id", ["torch_common.h", "torch_tensors.h"]),
])  # fmt: skip
def test_the_layer_is_built_with_the_headers_in_the_tree(made, sources):
    """Beside the ids of the sources themselves: which headers each object of the binding was compiled with."""
    h = hashlib.sha256()
    for name in sources:
        with open(os.path.join(CSRC, name), "rb") as f:
            h.update(f.read())
    assert getattr(ops._C, made)() == h.hexdigest()[:16], "pplx_kernels/_C.so is stale: run `make -C pplx-kernels_amd/csrc`"
