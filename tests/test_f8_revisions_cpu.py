"""The 8-bit and experts' operators' revisions cover all of their sources (no GPU)."""
import glob
import os

import pytest

from test_kv4_revisions_cpu import included
from unpopped_b200 import build

UNITS = ["experts.cu", "f8_matmul.cu", "f8_quantise.cu"]


@pytest.mark.parametrize("name", UNITS)
def test_no_source_is_left_out(name):
    assert tuple(sorted(included(name))) == build.OPERATOR_SOURCES[name]


@pytest.mark.parametrize("name", UNITS)
def test_the_line_of_the_others_is_theirs(name):
    with open(os.path.join(build.CSRC, name)) as f:
        assert [line for line in f if line.startswith("// FNV-1a 64 of")] == [build.sources_line(name)], \
            "run python -m unpopped_b200.build --sources"


def test_a_change_of_the_launches_changes_their_revisions(tmp_path, monkeypatch):
    for path in glob.glob(os.path.join(build.CSRC, "*")):
        with open(path, "rb") as f:
            (tmp_path / os.path.basename(path)).write_bytes(f.read())
    monkeypatch.setattr(build, "CSRC", str(tmp_path))
    before = {n: build.revision_hash(str(tmp_path / n)) for n in build.OPERATOR_SOURCES}
    with open(tmp_path / "launch.cuh", "a") as f:
        f.write("\n")
    build.write_sources_lines()
    after = {n: build.revision_hash(str(tmp_path / n)) for n in build.OPERATOR_SOURCES}
    assert {n for n in before if before[n] != after[n]} == set(UNITS)
