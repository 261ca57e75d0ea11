"""The hash by which bench.py knows whether a committed profile of the frame belongs to the tree's kernels."""
import importlib.util
import os
import shutil

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "taichi_3d_gaussian_splatting_amd", "csrc")


def _bench():
    spec = importlib.util.spec_from_file_location("bench_for_its_hash", os.path.join(ROOT, "bench.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_hash_follows_the_frames_sources_and_flags_alone(tmp_path):
    bench, copy = _bench(), tmp_path / "csrc"
    copy.mkdir()
    for name in os.listdir(CSRC):
        if name.endswith((".hip", ".h", ".cpp")) or name == "Makefile":
            shutil.copy(os.path.join(CSRC, name), copy / name)
    first = bench.kernel_source_hash(str(copy))
    assert first == bench.kernel_source_hash()
    # other operators of the library: the record stays
    for name in ("gs_adamw.hip", "gs_optim.hip", "gs_loss.hip", "gs_host.cpp"):
        assert (copy / name).exists()
        (copy / name).write_text((copy / name).read_text() + "\n// more\n")
    makefile = (copy / "Makefile").read_text()
    (copy / "Makefile").write_text(makefile + "\n# more\nother:\n\ttrue\n")
    assert bench.kernel_source_hash(str(copy)) == first
    # what the frame's kernels are made of: it does not
    seen = {first}
    for old, new in (("-O3", "-O2"), ("-packed-fp32-ops", "+packed-fp32-ops"), ("-fno-slp-vectorize", "-fslp-vectorize")):
        assert old in makefile
        (copy / "Makefile").write_text(makefile.replace(old, new, 1))
        seen.add(bench.kernel_source_hash(str(copy)))
    (copy / "Makefile").write_text(makefile)
    for name in ("gs_blend.hip", "gs_common.h", "gs_frame.hip"):
        (copy / name).write_text((copy / name).read_text() + "\n")
        seen.add(bench.kernel_source_hash(str(copy)))
    assert len(seen) == 7
