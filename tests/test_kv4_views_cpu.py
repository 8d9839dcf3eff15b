"""CPU tests of what the 4-bit cache's calls refuse because views share memory."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from llm_fa_b200 import _lib
from llm_fa_b200.build import build

HERE = Path(__file__).resolve().parent
BAD = _lib.LLMFA_ERR_INVALID_ARGUMENT


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


def test_views_meet_where_marks_do(tmp_path):
    """tests/csrc/test_kv4_views.cu compares the search with marks in an array."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc not available")
    exe = tmp_path / "test_kv4_views"
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-o",
                    str(exe), str(HERE / "csrc" / "test_kv4_views.cu")], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.startswith("ok")


# addresses that are never read: every call here is refused. A row has 256 bytes.
CACHE = _lib.Kv4Cache(1 << 20, 1 << 20, 1 << 20, 8, 2, 64, 64)
SEQS = _lib.Kv4Seqs(1 << 20, 4, 4, 1 << 20, 3)
P = ctypes.c_void_p
DENSE = (5 * 2 * 128, 2 * 128, 128)  # [3, 5, 2, 128]
ROWS = 3 * 5 * 2


def _attend(L, q, qs, o, os):
    return L.llmfa_kv4_attention(CACHE, SEQS, P(q), _lib.strides3(qs), P(o), _lib.strides3(os), None,
                                 None, None, 2, 5, 1, ctypes.c_float(0.1), ctypes.c_float(-1.0), 0, 0,
                                 P(1 << 20), 1 << 40, None)


def _expand(L, k, ks, v, vs):
    return L.llmfa_kv4_expand(CACHE, SEQS, P(k), _lib.strides3(ks), P(v), _lib.strides3(vs), None, 5, 0,
                              None)


@pytest.mark.parametrize("call", [_attend, _expand])
@pytest.mark.parametrize("shift", [0, 16, -16, 240, 256, (ROWS - 1) * 256 + 240])
def test_a_view_over_another_is_refused(L, call, shift):
    assert call(L, 1 << 24, DENSE, (1 << 24) + shift, DENSE) == BAD


@pytest.mark.parametrize("call", [_attend, _expand])
def test_slices_that_reach_into_one_another_are_refused(L, call):
    wide = tuple(2 * s for s in DENSE)
    assert call(L, 1 << 24, wide, (1 << 24) + 256 - 16, wide) == BAD
    assert call(L, 1 << 24, wide, (1 << 24) + 256 + 16, wide) == BAD


@pytest.mark.parametrize("strides", [(1280, 256, 120), (1280, 128, 128), (8, 2560, 256), (256, 256, 128)])
def test_an_output_whose_rows_meet_is_refused(L, strides):
    assert _attend(L, 1 << 24, DENSE, 1 << 26, strides) == BAD
    assert _expand(L, 1 << 24, DENSE, 1 << 26, strides) == BAD
    assert _expand(L, 1 << 26, strides, 1 << 24, DENSE) == BAD


@pytest.mark.parametrize("shift", [0, 8, -8])
def test_new_lengths_over_the_old_ones_are_refused(L, shift):
    new = (1 << 20) + shift
    assert L.llmfa_kv4_evict_select(CACHE, SEQS, None, 64, 8, P(1 << 24), P(new), P(1 << 26), 1 << 30,
                                    None) == BAD
