import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run through gpurun)")


def pytest_collection_modifyitems(config, items):
    """Without a HIP device the gpu-marked tests are skipped (a CPU-only run then still reports CPU-side regressions)
    -- except on a gpurun box (GRAFT_REPO_ROOT is set there), where a missing device must fail loudly."""
    if not os.path.isdir("/root/reference/taichi_3d_gaussian_splatting"):
        # an empty folder in their place is no reference sources either
        for item in items:
            if any("reference sources" in str(m.kwargs.get("reason")) for m in item.iter_markers("skipif")):
                item.add_marker(pytest.mark.skip(reason="no reference sources here"))
    import torch
    if torch.cuda.is_available() or os.environ.get("GRAFT_REPO_ROOT"):
        return
    skip = pytest.mark.skip(reason="no HIP device (gpu tests run through gpurun)")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


@pytest.fixture(scope="session", autouse=True)
def _build_native():
    """Build the checker (CPU oracle) and, if the in-tree library is missing or stale, the HIP library
    (hipcc cross-compiles gfx950 without a GPU; the same image is on the GPU box)."""
    from oracle import gs_oracle
    gs_oracle.build()
    from taichi_3d_gaussian_splatting_amd import _lib
    csrc = os.path.join(ROOT, "taichi_3d_gaussian_splatting_amd", "csrc")
    srcs = [os.path.join(csrc, f) for f in os.listdir(csrc) if f.endswith((".hip", ".h"))]
    srcs.append(os.path.join(ROOT, "include", "gsplat_hip.h"))
    if not os.path.exists(_lib.LIB_PATH) or os.path.getmtime(_lib.LIB_PATH) < max(map(os.path.getmtime, srcs)):
        _lib.build()
