"""The serving operators' revisions cover all of their sources (no GPU)."""
import glob
import os
import re

import pytest

from unpopped_b200 import build

SHARED = {"common.cuh", "tc.cuh", "up_sm100.h"}  # the library's, not an operator's


def included(name):
    """The files of csrc that `name` includes, at any depth."""
    with open(os.path.join(build.CSRC, name)) as f:
        near = {os.path.basename(p) for p in re.findall(r'#include "(.*?)"', f.read())} - SHARED
    return near.union(*(included(n) for n in near)) if near else set()


@pytest.mark.parametrize("name", sorted(build.OPERATOR_SOURCES))
def test_the_line_of_the_others_is_theirs(name):
    with open(os.path.join(build.CSRC, name)) as f:
        lines = [line for line in f if line.startswith("// FNV-1a 64 of")]
    assert lines == [build.sources_line(name)], "run python -m unpopped_b200.build --sources"


def test_no_source_is_left_out():
    units = {"rope.cu": ["rope.cu"], "kv4_append.cu": ["kv4_append.cu"],
             "kv4_attention.cu": ["kv4_attention.cu"] + [os.path.basename(p) for p in glob.glob(os.path.join(build.CSRC, "kv4_*.cu"))
                                                         if "append" not in p]}
    for name, files in units.items():
        all_of = set(files).union(*(included(f) for f in files)) - {name}
        assert tuple(sorted(all_of)) == build.OPERATOR_SOURCES[name]


def test_a_change_of_a_kernel_changes_the_line(tmp_path, monkeypatch):
    for path in glob.glob(os.path.join(build.CSRC, "*")):
        with open(path, "rb") as f:
            (tmp_path / os.path.basename(path)).write_bytes(f.read())
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    before = {n: build.revision_hash(str(tmp_path / n)) for n in build.OPERATOR_SOURCES}
    with open(tmp_path / "kv4_prompt.cu", "a") as f:
        f.write("\n")
    build.write_sources_lines()
    after = {n: build.revision_hash(str(tmp_path / n)) for n in build.OPERATOR_SOURCES}
    assert {n for n in before if before[n] != after[n]} == {"kv4_attention.cu"}
    with open(tmp_path / "divide.cuh", "a") as f:
        f.write("\n")
    build.write_sources_lines()
    assert all(build.revision_hash(str(tmp_path / n)) != after[n] for n in after)
