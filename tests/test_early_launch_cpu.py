"""Kernels that may begin before the ones ahead of them end (csrc/launch.cuh) read no memory by the non-coherent path, and wait before they
touch any (no GPU)."""
import glob
import os
import re

import pytest

from unpopped_b200 import build


def text_of(name):
    with open(os.path.join(build.CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


FILES = sorted(os.path.basename(p) for p in glob.glob(os.path.join(build.CSRC, "*.cu")) if "launch_early(" in text_of(os.path.basename(p)))


def test_there_are_such_files():
    assert {"experts.cu", "f8_matmul.cu", "f8_quantise.cu"} <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_no_read_goes_by_the_non_coherent_path(name):
    text = text_of(name)
    assert not re.search(r"\.nc\b|ld_nc\w*\s*\(|__ldg\s*\(", text)
    assert not re.search(r"\bconst\b[^,;(){}]*\*\s*(const\s+)?__restrict__", text)


@pytest.mark.parametrize("name", FILES)
def test_every_kernel_waits(name):
    """Each kernel's own body, or the function that it is made of, waits for the kernels ahead."""
    text = text_of(name)
    bodies = re.split(r"__global__", text)[1:]
    assert bodies
    for body in bodies:
        body = body[:body.index("\n}")]
        waits = "after_previous();" in body
        if not waits:
            called = re.findall(r"^\s+(\w+)<?[\w, ]*>?\(.*\);$", body, re.M)
            waits = any(re.search(r"void " + f + r"\((?:(?!\n}).)*after_previous\(\);", text, re.S) for f in called)
        assert waits, body[:120]
