"""What the built extension says of its kernels' registers."""

import shutil
import subprocess

import pytest

from replay_amd.ops import _load

SOURCE = """
#include <hip/hip_runtime.h>
extern "C" __global__ void plain(int* p) { p[threadIdx.x] += 1; }
extern "C" __global__ void spills(int* p, int n) {
  volatile int own[37];
  for (int i = 0; i < 37; ++i) own[i] = p[i] + n;
  p[threadIdx.x] = own[(threadIdx.x + n) % 37];
}
namespace {
__global__ void la_pass_test(int* p, int n) {
  volatile int own[9];
  for (int i = 0; i < 9; ++i) own[i] = p[i] + n;
  p[threadIdx.x] = own[(threadIdx.x + n) % 9];
}
}
void launch(int* p, int n) {
  if (n < 0) la_pass_test<<<1, 64>>>(p, n);
}
"""


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    if shutil.which("hipcc") is None:
        pytest.skip("needs hipcc")
    where = tmp_path_factory.mktemp("kernels")
    (where / "k.hip").write_text(SOURCE)
    command = ["hipcc", "-O2", "--offload-arch=gfx950", "-shared", "-fPIC", "-o", str(where / "k.so"), str(where / "k.hip")]
    subprocess.run(command, check=True, capture_output=True, timeout=300)
    return where / "k.so"


def test_scratch_is_read(library):
    used = _load.scratch_bytes(library)
    assert used["plain"] == 0 and used["spills"] >= 37 * 4
    assert any("la_pass_test" in name for name in used)


def test_scratch_is_refused(library):
    with pytest.raises(RuntimeError, match="la_pass_test"):
        _load.check_scratch(library)


def test_a_library_without_the_kernels_is_refused(tmp_path):
    (tmp_path / "empty.so").write_bytes(b"nothing")
    with pytest.raises(RuntimeError, match="no kernels"):
        _load.check_scratch(tmp_path / "empty.so")


@pytest.mark.skipif(not _load._so_path().exists(), reason="the extension is not built")
def test_the_extension_does_not_spill():
    _load.check_scratch(_load._so_path())
