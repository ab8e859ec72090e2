"""raydp_torch.so against a library of kernels that was built from other sources (no GPU needed)."""
import os
import shutil
import subprocess
import sys

import pytest

from raydp_amd.native import loader

LOAD = """
import importlib.util, torch
spec = importlib.util.spec_from_file_location("raydp_torch", "raydp_torch.so")
mod = importlib.util.module_from_spec(spec)
spec.loader.exec_module(mod)
"""


def _run(tmp_path):
    return subprocess.run([sys.executable, "-c", LOAD], cwd=tmp_path, capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("wrong", ["rx_aw_layout", "rx_expert_layout", None])
def test_the_module_loads_only_with_the_layout_it_was_built_with(wrong, tmp_path):
    """A stand-in exports what the module calls and says that it has one of the two layouts or, in the end, both."""
    ext = loader.load_torch()
    here = os.path.dirname(loader.__file__)
    shutil.copy(os.path.join(here, "raydp_torch.so"), tmp_path)
    names = subprocess.run(["nm", "-D", "--undefined-only", tmp_path / "raydp_torch.so"], capture_output=True, text=True, check=True)
    names = [line.split()[-1] for line in names.stdout.splitlines() if line.split()[-1].startswith("rx_")]
    right = {"rx_aw_layout": ext.layouts[0], "rx_expert_layout": ext.layouts[1]}
    body = [f"unsigned long long {n}(void) {{ return {right.get(n, 0) + (n == wrong)}ull; }}" for n in names]
    (tmp_path / "stand_in.c").write_text("\n".join(body) + "\n")
    subprocess.run(["gcc", "-shared", "-fPIC", "stand_in.c", "-o", "libhipkernels.so"], cwd=tmp_path, check=True)
    got = _run(tmp_path)
    if wrong is None:
        assert got.returncode == 0, got.stderr[-500:]
    else:
        assert got.returncode != 0 and "different sources" in got.stderr, got.stderr[-500:]
