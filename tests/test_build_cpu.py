"""The build places every kernel where the last one did: options under which ptxas
orders a translation unit's kernels by which thread is done first are not used
(their times then differ from build to build by up to 15 %)."""
from cudalab_b200 import build


def test_kernels_are_placed_alike_in_every_build():
    flags = " ".join(build.NVCC_FLAGS + build.ARCH_FLAGS)
    assert "split-compile" not in flags and "--threads" not in flags
