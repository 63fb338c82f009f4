"""Rules of the lean training-step operators that can be checked without a GPU."""
import re

from paper_01_anti_decoy_pnfirtau_b200 import _build


def code(path):
    """A source file without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_kernels_launched_early_read_through_the_ordinary_path():
    """A kernel that is launched while the one before still runs may read what that one writes. The read-only path
    (and a restrict pointer, from which the compiler may infer it) is for data that is constant while a kernel lives."""
    files = [f for f in sorted(_build.CSRC.glob("*.cu*")) if "wait_previous()" in code(f)]
    files += [_build.CSRC / f for f in ("skinny.cuh", "xent_math.cuh", "gemm_tc.cuh") if _build.CSRC / f not in files]
    assert len(files) >= 6
    for f in files:
        found = re.findall(r"__ldg|__restrict__|\.nc\b", code(f))
        assert not found, (f.name, found)


def test_kernels_launched_early_wait():
    """Every kernel of those files lets the next one start and waits for the one before."""
    for f in sorted(_build.CSRC.glob("*.cu*")):
        text = code(f)
        if "wait_previous()" in text:
            assert text.count("__global__") == len(re.findall(r"(?<!void )wait_previous\(\);", text)), f.name
            assert text.count("__global__") == len(re.findall(r"(?<!void )launch_next\(\);", text)), f.name
