"""CPU tests of the entry points that search over continuations: argument errors are returned before any CUDA
call, so they need no GPU (addresses below are never dereferenced)."""
import ctypes

import pytest

from mockbird_b200 import _lib
from mockbird_b200.build import build

BASE = 0x10000


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.load()


def select(lib, **kw):
    a = dict(groups=2, beams=4, codes=64, dtype=_lib.MB_F32, logits=BASE, stride=64, scores=BASE, scores_out=BASE,
             finished=None, finished_out=None, end_id=-1, seen=None, penalty=1.0, parents=BASE, tokens=BASE)
    a.update(kw)
    return lib.mb_beam_select(*a.values(), None)


@pytest.mark.parametrize("kw", [
    {"groups": -1}, {"groups": 65536}, {"beams": 0}, {"beams": 17}, {"codes": 0}, {"codes": (1 << 24) + 1},
    {"dtype": 3}, {"dtype": -1}, {"stride": 63}, {"stride": 0}, {"stride": -64}, {"stride": (1 << 32) + 1},
    {"end_id": -2}, {"end_id": 64}, {"finished": BASE, "finished_out": BASE}, {"finished": BASE, "end_id": 1},
    {"finished_out": BASE, "end_id": 1}, {"seen": BASE, "codes": 63, "stride": 64}, {"seen": BASE, "penalty": 0.0},
    {"seen": BASE, "penalty": -1.0}, {"seen": BASE, "penalty": float("nan")}, {"seen": BASE, "penalty": float("inf")},
    {"logits": None}, {"scores": None}, {"scores_out": None}, {"parents": None}, {"tokens": None},
    {"logits": BASE + 2}, {"logits": BASE + 1, "dtype": _lib.MB_F16}, {"scores": BASE + 2}, {"scores_out": BASE + 1},
    {"finished": BASE + 2, "finished_out": BASE, "end_id": 1}, {"finished": BASE, "finished_out": BASE + 2, "end_id": 1},
    {"seen": BASE + 2}, {"parents": BASE + 2}, {"tokens": BASE + 3},
])
def test_beam_select_refuses_bad_arguments(lib, kw):
    assert select(lib, **kw) == 1  # MB_ERR_ARG


def test_beam_select_takes_no_groups_and_aligned_arguments(lib):
    import torch

    assert select(lib, groups=0, logits=None) == 0
    if torch.cuda.is_available():
        pytest.skip("only meaningful without a GPU (the call would otherwise run)")
    for kw in ({}, {"logits": BASE + 2, "dtype": _lib.MB_BF16}, {"finished": BASE, "finished_out": BASE, "end_id": 0},
               {"seen": BASE, "penalty": 1.2}, {"beams": 16, "stride": 1000}):
        assert select(lib, **kw) == 6  # MB_ERR_CUDA: past the checks, stopped at the launch


def test_null_contexts(lib):
    n = ctypes.c_void_p()
    assert lib.mb_tree_attend(n, 0, 1, 1, n, n, n, n, n, n) == 1
    assert lib.mb_tree_commit(n, 0, 1, 1, 1, n, n, n, n, n, n, n) == 1
    assert lib.mb_ring_reorder(n, 1, 1, n, n, n) == 1


def test_beam_select_wants_device_tensors():
    import torch

    from mockbird_b200 import beam_select

    with pytest.raises(TypeError, match="logits"):
        beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2))
