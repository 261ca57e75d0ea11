"""The scripts that build other variants of the library compile what the Makefile compiles, the way it does, plus their own flags."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "taichi_3d_gaussian_splatting_amd", "csrc")
SOURCES = sorted(f[:-4] for f in os.listdir(CSRC) if f.endswith(".hip"))
NO_PACKED = "-Xclang -target-feature -Xclang -packed-fp32-ops"

pytestmark = pytest.mark.skipif(shutil.which("make") is None, reason="no make")


def _run(tmp_path, script, *args):
    """The command lines that a script gives the compiler (a stand-in that only makes its output file)."""
    log = tmp_path / "log"
    hipcc = tmp_path / "hipcc"
    hipcc.write_text(f'#!/bin/bash\necho "$PWD $@" >> {log}\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && echo x > "$2"; shift; done\n')
    hipcc.chmod(0o755)
    env = dict(os.environ, HIPCC=str(hipcc), GS_VARIANTS_DIR=str(tmp_path / "variants"))
    subprocess.run(["bash", os.path.join(ROOT, "tools", script), *args], check=True, env=env, stdout=subprocess.DEVNULL, timeout=100)
    return log.read_text().splitlines()


def test_build_variants_takes_sources_and_flags_from_the_makefile(tmp_path):
    assert "gs_adamw" in SOURCES
    lines = _run(tmp_path, "build_variants.sh", "a:-DGS_ONE=1 -DGS_TWO=2", "b:")
    compiled = [line for line in lines if " -c " in line]
    for flags in ("-DGS_ONE=1 -DGS_TWO=2", ""):
        mine = [line for line in compiled if (flags in line if flags else "-DGS_ONE" not in line)]
        assert sorted(re.search(r"-c (?:\S*/)?(\w+)\.hip", line).group(1) for line in mine) == SOURCES
        assert all(NO_PACKED in line and "-munsafe-fp-atomics" in line and "--offload-arch=gfx950" in line for line in mine)
        for line in mine:
            assert ("-fno-slp-vectorize" in line) == bool(re.search(r"-c (?:\S*/)?gs_(frontend|point_backward)\.hip", line))
    links = [line for line in lines if "-shared" in line]
    assert len(links) == 2 and all(f"{name}.o" in line for line in links for name in SOURCES)
    assert sorted(os.listdir(tmp_path / "variants")) == ["libgsplat_hip_a.so", "libgsplat_hip_b.so"]
    assert not any(line.startswith(CSRC + " ") for line in lines), "the tree's own objects were touched"


def test_build_ablations_links_every_object_and_keeps_the_flags(tmp_path):
    if shutil.which("patch") is None:
        pytest.skip("no patch")
    if not all(os.path.exists(os.path.join(CSRC, name + ".o")) for name in SOURCES):
        pytest.skip("the tree is not built")
    lines = _run(tmp_path, "build_ablations.sh")
    ablated = [line for line in lines if "-DGS_ABLATE_" in line]
    assert len(ablated) == 6 and all("gs_frontend.hip" in line and NO_PACKED in line and "-fno-slp-vectorize" in line for line in ablated)
    links = [line for line in lines if "-shared" in line and "libgsplat_hip" in line][-6:]
    assert len(links) == 6 and all(f"{name}.o" in line for line in links for name in SOURCES)


def test_no_tool_has_compiler_flags_of_its_own_for_the_librarys_sources():
    for name in os.listdir(os.path.join(ROOT, "tools")):
        if name.endswith((".sh", ".py")):
            with open(os.path.join(ROOT, "tools", name)) as fh:
                assert "munsafe-fp-atomics" not in fh.read(), name
