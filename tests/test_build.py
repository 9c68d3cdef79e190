"""kaldi_amd/csrc/Makefile: what is built again when (make on a copy with empty sources and a compiler that writes empty files)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "kaldi_amd", "csrc")


@pytest.fixture
def tree(tmp_path):
    """a tree in which everything is up to date, compiled by a stand-in that writes empty files"""
    csrc = tmp_path / "kaldi_amd" / "csrc"
    csrc.mkdir(parents=True)
    (tmp_path / "include").mkdir()
    for f in os.listdir(CSRC):
        (csrc / f).write_text("")
    (tmp_path / "include" / "kaldi_amd.h").write_text("")
    shutil.copy(os.path.join(CSRC, "Makefile"), csrc / "Makefile")
    cc = tmp_path / "cc"
    cc.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    cc.chmod(0o755)

    def make(*args):
        r = subprocess.run(["make", "-C", str(csrc), "HIPCC=" + str(cc), "CXX=" + str(cc), *args], capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return {os.path.basename(o) for o in re.findall(r" -o (\S+)", r.stdout)}
    everything = make()
    assert "libkaldi_amd.so" in everything and "decoder.o" in everything and len(everything) > 20
    assert make() == set()
    make.csrc, make.everything = csrc, everything
    return make


def objects(names):
    return {n for n in names if n.endswith(".o")}


def test_a_changed_source_builds_its_object(tree):
    os.utime(tree.csrc / "rownorm.hip", (2e9, 2e9))
    assert tree() == {"rownorm.o", "libkaldi_amd.so"}


def test_changed_flags_build_every_object(tree):
    """the flags are part of what the library computes (no contraction, no packed arithmetic): no object of the old ones stays"""
    mk = tree.csrc / "Makefile"
    mk.write_text(mk.read_text().replace("-O3", "-O3 -DOTHER"))
    assert objects(tree()) == objects(tree.everything)
    assert tree() == set()


def test_changed_settings_build_every_object(tree):
    assert objects(tree("KAMD_NT=512")) == objects(tree.everything)
    assert tree("KAMD_NT=512") == set()
    assert objects(tree()) == objects(tree.everything)
