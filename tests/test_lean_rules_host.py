"""Rules of the lean training-step operators that can be checked without a GPU."""
import re

import pytest
import torch

import paper_01_anti_decoy_pnfirtau_b200 as P
from paper_01_anti_decoy_pnfirtau_b200 import _build, _lib, lm_ops


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


def test_refreshed_copies_of_changed_parameters_count_as_changed(monkeypatch):
    """A copy's version moves when it is refreshed from a parameter that changed, and only then: autograd sees by it
    that a tensor saved for a backward holds other values now."""
    calls = []

    class Library:
        def pnft_cast_bf16(self, *args):
            calls.append(args)
            return 0

    monkeypatch.setattr(lm_ops._lib, "lib", Library)
    monkeypatch.setattr(lm_ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    a, b, head = (torch.nn.Parameter(torch.randn(6, 4)) for _ in range(3))
    casts = lm_ops.Bf16Casts([a, b, head], padded={id(head): 8})
    versions = lambda: [c._version for c in casts.copies]  # noqa: E731
    casts.refresh()
    first = versions()
    casts.refresh()
    assert versions() == first and len(calls) == 2
    with torch.no_grad():
        b.add_(1)
        head.add_(1)
    casts.refresh()
    assert [x > y for x, y in zip(versions(), first)] == [False, True, True]
    a.data = a.data.clone()  # another storage
    casts.refresh()
    assert versions()[0] > first[0]


def test_limits_of_the_few_row_calls_agree():
    """The Python calls leave rows unaligned up to the number of rows that the C entry points take so."""
    header = (_build.INCLUDE / "pnfirtau_b200.h").read_text()
    limit = lambda name: int(re.search(rf"#define {name} (\d+)", header).group(1))  # noqa: E731
    assert _lib.GATED_FEW_ROWS == limit("PNFT_GATED_FEW_ROWS")
    assert _lib.XENT_FEW_ROWS == limit("PNFT_XENT_FEW_ROWS")


def test_act8_refuses_buffers_that_do_not_hold_its_shape():
    """The kernels read what shape says: the buffer has to hold it."""
    P.Act8(torch.zeros(4, 1024, dtype=torch.uint8), torch.Size((2, 2, 1000)), torch.bfloat16)._layout()
    good = dict(data=torch.zeros(4, 1024, dtype=torch.uint8), shape=torch.Size((4, 1000)), dtype=torch.bfloat16)
    for bad in (dict(data=torch.zeros(4, 1008, dtype=torch.uint8)), dict(data=torch.zeros(3, 1024, dtype=torch.uint8)),
                dict(data=torch.zeros(4, 1024, dtype=torch.int8)), dict(data=torch.zeros(4 * 1024, dtype=torch.uint8)),
                dict(data=torch.zeros(4, 2048, dtype=torch.uint8)[:, ::2]), dict(shape=torch.Size((4, 1025))),
                dict(shape=torch.Size((5, 1000))), dict(shape=torch.Size(())), dict(shape=torch.Size((4, 0))),
                dict(dtype=torch.float64), dict(data=torch.zeros(4 * 1024 + 8, dtype=torch.uint8)[8:].view(4, 1024))):
        with pytest.raises(RuntimeError, match="Act8"):
            P.Act8(**{**good, **bad})._layout()
    with pytest.raises(RuntimeError, match="CUDA"):
        P.act8_unpack(P.Act8(**good))
