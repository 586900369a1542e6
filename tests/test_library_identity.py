"""nerfhip_version() names the sources of the field's kernels: the counter summaries under profiles/ are matched by it, and stay valid
when other kernels of the library change."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nerf_amd", "csrc")


def _identity(csrc):
    """The hash that a build in this folder would record (make only prints the command)."""
    text = subprocess.check_output(["make", "-s", "-n", "-B", "-C", str(csrc), "version.o"], text=True)
    return re.search(r'NERFHIP_SRC_HASH=\\"([0-9a-f]{12})\\"', text).group(1)


@pytest.fixture
def csrc(tmp_path):
    to = tmp_path / "csrc"
    to.mkdir()
    for name in os.listdir(CSRC):
        if not name.endswith(".o"):
            shutil.copy(os.path.join(CSRC, name), to / name)
    return to


@pytest.mark.parametrize("name", ["adamw.hip", "ffn.hip", "ffn_gemm.hip.h", "ffn_gemm_inst.hip", "op_common.h"])
def test_the_operators_sources_do_not_count(csrc, name):
    before = _identity(csrc)
    (csrc / name).open("a").write("// another line\n")
    assert _identity(csrc) == before


@pytest.mark.parametrize("name", ["mlp_fwd.hip", "wgrad_bf16.hip", "common.h", "train_impl.inc", "ray_kernels.hip"])
def test_the_fields_sources_count(csrc, name):
    before = _identity(csrc)
    (csrc / name).open("a").write("// another line\n")
    assert _identity(csrc) != before


def test_the_library_records_the_identity_of_this_tree():
    from nerf_amd import _lib
    assert _lib.load().nerfhip_version().decode().endswith("src " + _identity(CSRC))
