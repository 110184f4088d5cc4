"""The Makefile's dependences, with a stand-in for the compiler that only notes what it was asked to compile: objects follow
their flags, and nothing is compiled twice with the same ones."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join("t5vqvae_amd", "csrc")

COMPILER = """#!/bin/sh
echo "$@" >> "$COMPILER_LOG"
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then shift; echo built > "$1"; fi
  shift
done
"""


@pytest.fixture
def tree(tmp_path):
    """A copy of the sources without anything built, and make() -> the sources it compiled."""
    (tmp_path / CSRC).mkdir(parents=True)
    for name in os.listdir(os.path.join(ROOT, CSRC)):
        if name == "Makefile" or name.endswith((".hip", ".h", ".cpp")):
            shutil.copy(os.path.join(ROOT, CSRC, name), tmp_path / CSRC / name)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    compiler, log = tmp_path / "compiler", tmp_path / "log"
    compiler.write_text(COMPILER)
    compiler.chmod(0o755)

    def make(*variables, target=None):
        if log.exists():
            log.unlink()
        out = target or str(tmp_path / CSRC / "libt5vq.so")
        subprocess.run(["make", "-C", str(tmp_path / CSRC), f"HIPCC={compiler}", "PYTHON=true", *variables, out], check=True,
                       stdout=subprocess.DEVNULL, env=dict(os.environ, COMPILER_LOG=str(log)), timeout=120)
        lines = log.read_text().splitlines() if log.exists() else []
        return {line.split()[-1]: line for line in lines if " -c " in line}, [line for line in lines if " -shared " in line]

    make.csrc = tmp_path / CSRC
    return make


def sources(make):
    return {name for name in os.listdir(make.csrc) if name.endswith(".hip")}


def test_objects_follow_their_flags(tree):
    compiled, linked = tree()
    assert set(compiled) == sources(tree) and len(linked) == 1
    assert all("-packed-fp32-ops" in line and "-ffp-contract=off" in line for line in compiled.values())
    assert tree() == ({}, [])                                    # nothing to do a second time
    for variant in ("EXTRA=-DT5VQ_TUNING", "ARCH=gfx950:sramecc+"):
        compiled, linked = tree(variant)
        assert set(compiled) == sources(tree) and len(linked) == 1
        assert all(variant.split("=")[1] in line for line in compiled.values())
        assert tree(variant) == ({}, [])
    compiled, linked = tree()                                     # back to the default: not the variant's objects
    assert set(compiled) == sources(tree) and len(linked) == 1
    assert not any("T5VQ_TUNING" in line or "sramecc" in line for line in compiled.values())


def test_a_variant_library_in_another_place_is_made_of_its_own_objects(tree, tmp_path):
    tree()
    other = str(tmp_path / "variant.so")
    compiled, linked = tree("EXTRA=-DT5VQ_TUNING", f"OUT={other}", target=other)
    assert set(compiled) == sources(tree) and other in linked[0]
    compiled, linked = tree()
    assert set(compiled) == sources(tree) and not any("T5VQ_TUNING" in line for line in compiled.values())


def test_objects_follow_the_makefile(tree):
    tree()
    makefile = tree.csrc / "Makefile"
    makefile.write_text(makefile.read_text().replace("-O3", "-O2"))
    compiled, linked = tree()
    assert set(compiled) == sources(tree) and all("-O2" in line for line in compiled.values()) and len(linked) == 1


def test_build_compiles_also_where_a_built_library_is_there(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "run", lambda args, **kw: calls.append((args, kw)))
    entry.build()
    (args, kw), = calls
    assert args[0] == "make" and "-B" in args and "all" in args and kw == {"check": True}
