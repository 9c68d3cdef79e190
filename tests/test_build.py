"""kaldi_amd/csrc/Makefile: what is built again when (make on a copy with empty sources and a compiler that writes empty files)."""
import os
import re
import shutil
import subprocess
import sys

import pytest
import torch          # before the library: they share one HIP runtime then

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


def test_the_torch_module_is_of_one_torch(tree, tmp_path):
    """it reads tensors through the layouts it was compiled with: another torch or Python gets a module of its own"""
    from kaldi_amd import int8
    name = os.path.basename(int8._extension_path())
    assert name in tree.everything and os.path.exists(int8._extension_path())
    other = tmp_path / "site" / "torch"
    other.mkdir(parents=True)
    (other / "__init__.py").write_text("")
    (other / "version.py").write_text("__version__ = '99.1+x'\n")
    python = tmp_path / "python"
    python.write_text('#!/bin/sh\nPYTHONPATH=%s exec %s "$@"\n' % (other.parent, sys.executable))
    python.chmod(0o755)
    made = tree("PY=" + str(python))
    assert len(made) == 1 and "torch-99.1+x" in made.pop()


def test_a_module_of_another_torch_is_not_loaded(monkeypatch):
    from kaldi_amd import int8
    from kaldi_amd._lib import KamdError
    monkeypatch.setattr(int8, "_X", None)
    monkeypatch.setattr(torch, "__version__", "99.1+x")
    with pytest.raises(KamdError, match="torch-99.1.*is missing"):
        int8.rms_norm(torch.zeros(2, 8))
