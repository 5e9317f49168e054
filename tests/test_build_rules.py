"""The library's Makefile with a compiler that only notes what it was asked for: what a change rebuilds, and the build id."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "esm_amd", "csrc")

COMPILER = """#!/bin/sh
echo "$*" >> "$NOTES"
while [ $# -gt 0 ]; do if [ "$1" = -o ]; then out=$2; fi; shift; done
: > "$out"
[ -z "$REMARK" ] || echo "$REMARK" >&2
"""


@pytest.fixture
def tree(tmp_path):
    """A copy of the sources, without anything built."""
    csrc = tmp_path / "esm_amd" / "csrc"
    csrc.mkdir(parents=True)
    for f in os.listdir(CSRC):
        if f == "Makefile" or f == "esmk.map" or (f.endswith((".hip", ".hpp")) and not f.startswith("_")):
            shutil.copy2(os.path.join(CSRC, f), csrc / f)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    cc = tmp_path / "cc"
    cc.write_text(COMPILER)
    cc.chmod(0o755)

    def make(*args, remark=""):
        """Sources compiled by one call of make, sorted.  remark: what the compiler says."""
        notes = tmp_path / "notes"
        notes.write_text("")
        subprocess.run(["make", "-C", str(csrc), f"HIPCC={cc}", *args], check=True, capture_output=True,
                       env={**os.environ, "NOTES": str(notes), "REMARK": remark})
        return sorted(re.findall(r"-c (\S+\.hip)", notes.read_text()))

    def build_id(out="obj"):
        found = [re.search(r'ESMK_BUILD_ID "([0-9a-f]{12})"', p.read_text()) for d in (csrc, csrc / out) for p in d.glob("*build_id.h")]
        assert len(found) == 1
        return found[0].group(1)
    return csrc, make, build_id


def change(path, old, new):
    text = path.read_text()
    assert text.count(old) == 1
    path.write_text(text.replace(old, new))


def test_changed_flags_rebuild_every_object_and_change_the_build_id(tree):
    csrc, make, build_id = tree
    everything = make()
    assert "attn_grad.hip" in everything and "gemm.hip" in everything and make() == []
    first = build_id()
    change(csrc / "Makefile", "CXXFLAGS += -Xclang -target-feature -Xclang -packed-fp32-ops\n", "")
    assert make() == everything
    second = build_id()
    assert second != first and make() == []
    change(csrc / "Makefile", "attn attn_grad\n", "attn\n")  # the files without the SLP vectoriser
    assert make() == everything
    assert build_id() not in (first, second)


def test_flags_on_the_command_line_count_too(tree):
    csrc, make, build_id = tree
    make()
    make("EXPERIMENTS=1")
    assert build_id("xobj") != build_id()
    one = make("VARIANT=one", "EXTRA=-DONE=1")
    assert one and make("VARIANT=one", "EXTRA=-DONE=1") == []
    before = build_id("vobj_one")
    assert make("VARIANT=one", "EXTRA=-DONE=2") == one and build_id("vobj_one") != before
    assert make() == [] and make("EXPERIMENTS=1") == []  # each kind of build keeps its own


def test_a_changed_source_rebuilds_itself_and_the_build_id(tree):
    csrc, make, build_id = tree
    make()
    first = build_id()
    change(csrc / "pref_loss.hip", "namespace {\n", "namespace {  // changed\n")
    os.utime(csrc / "pref_loss.hip", (2 ** 31, 2 ** 31))
    assert make()[:1] == ["pref_loss.hip"] and build_id() != first


@pytest.mark.parametrize("kind,source,most", [((), "attn_grad", 24), (("EXPERIMENTS=1",), "gemm4w", 0), (("EXPERIMENTS=1",), "gemm4v", 0)])
def test_scratch_beyond_what_is_stated_ends_the_build(tree, kind, source, most):
    csrc, make, _ = tree
    said = "k.hip:1:1: remark:     ScratchSize [bytes/lane]: %d [-Rpass-analysis=kernel-resource-usage]"
    out = csrc / ("xobj" if kind else "obj") / f"{source}.o"
    target = str(out.relative_to(csrc))
    with pytest.raises(subprocess.CalledProcessError):
        make(target, *kind, remark=said % (most + 1))
    assert not out.exists()
    make(target, *kind, remark=said % most)
    assert out.exists()
