"""CPU tests of the 4-bit cache: its layout (host code of the kernels' own header), the C ABI's
refusals before any CUDA call, and the Python surface's refusals."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from llm_fa_b200 import KV4Cache, _lib, kv4
from llm_fa_b200.build import build

from . import kv4_plain as plain

HERE = Path(__file__).resolve().parent
BAD, UNSUP = _lib.LLMFA_ERR_INVALID_ARGUMENT, _lib.LLMFA_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


@pytest.mark.parametrize("name", ["test_kv4_layout", "test_kv4_plan"])
def test_index_arithmetic_as_host_code(tmp_path, name):
    """tests/csrc/*.cu run the kernels' index functions as host code. Layout: every block of a
    page is its own, slots outside the table and ids outside the pool have no page, offsets pass
    32 bits. Plan: every tile is in exactly one CTA's share, and a cut unit's pieces are found."""
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(nvcc).exists():
        pytest.skip("nvcc not available")
    exe = tmp_path / name
    subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a",
                    "-o", str(exe), str(HERE / "csrc" / f"{name}.cu")],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert out.stdout.startswith("ok")


@pytest.mark.parametrize("group", [32, 64, 128])
def test_plain_format_round_trip(group):
    """The plain reader finds what the plain quantiser makes, at every place of a page."""
    rng = np.random.default_rng(group)
    x = rng.standard_normal((2, 32, 128))
    row = np.zeros(plain.block_bytes(group) * 2, np.uint8)
    want = {}
    for value in (0, 1):
        val, codes, scale, zero = plain.quantise(x[value], group)
        for t in range(32):
            at, pairs = plain.row_offset(t, value, group)
            for ch in range(128):
                byte, shift = plain.code_place(ch, value)
                row[at + byte] |= int(codes[t, ch]) << shift
            word = np.stack((scale[t], zero[t]), -1).astype(np.float32).view(np.uint32) >> 16
            row[pairs:pairs + 4 * (128 // group)] = word.astype(np.uint16).reshape(-1).view(np.uint8)
        want[value] = val
    for value in (0, 1):
        got = np.stack([plain.read_token(row, t, value, group) for t in range(32)])
        assert np.array_equal(got, want[value])
        pages = row[None, None]
        assert np.array_equal(plain.read(pages, np.array([0]), 32, 32, group, 0, value), want[value])


def test_page_bytes(L):
    for group, block in ((32, 2560), (64, 2304), (128, 2176)):
        for page in kv4.PAGE_SIZES:
            assert kv4.page_bytes(page, group) == page // 16 * block
            assert page // 16 * plain.block_bytes(group) == page // 16 * block
    n = ctypes.c_uint64(0)
    for page, group in ((8, 64), (48, 64), (512, 64), (64, 16), (64, 256), (0, 64)):
        assert L.llmfa_kv4_page_bytes(page, group, ctypes.byref(n)) == BAD
    assert L.llmfa_kv4_page_bytes(64, 64, None) == BAD


# fake, never-dereferenced addresses: validation fails before any CUDA call
CACHE = dict(pages=16, positions=16, weights=16, num_pages=8, heads=2, page_size=64, group=64)
SEQS = dict(page_table=16, table_stride=4, max_pages=4, lengths=16, batch=3)


def _structs(kw):
    kw = dict(kw)
    c = _lib.Kv4Cache(**{f: kw.pop(f, d) for f, d in CACHE.items()})
    s = _lib.Kv4Seqs(**{f: kw.pop(f, d) for f, d in SEQS.items()})
    return c, s, kw


def _p(a):
    return ctypes.c_void_p(a) if a else None


ST = (1 << 20, 256, 128)


def _append(L, **kw):
    c, s, kw = _structs(kw)
    g = lambda n, d: kw.get(n, d)  # noqa: E731
    return L.llmfa_kv4_append(c, s, _p(g("k", 16)), _lib.strides3(g("ks", ST)), _p(g("v", 16)),
                              _lib.strides3(ST), _p(g("counts", 0)), _p(g("seen", 0)),
                              g("tokens", 5), g("dtype", 0), None)


def _expand(L, **kw):
    c, s, kw = _structs(kw)
    g = lambda n, d: kw.get(n, d)  # noqa: E731
    return L.llmfa_kv4_expand(c, s, _p(g("k", 16)), _lib.strides3(g("ks", ST)), _p(g("v", 16)),
                              _lib.strides3(ST), _p(g("counts", 0)), g("tokens", 5), g("dtype", 0),
                              None)


def _attend(L, **kw):
    c, s, kw = _structs(kw)
    g = lambda n, d: kw.get(n, d)  # noqa: E731
    return L.llmfa_kv4_attention(c, s, _p(g("k", 16)), _lib.strides3(g("ks", ST)), _p(g("v", 16)),
                                 _lib.strides3(ST), _p(g("lse", 0)),
                                 _lib.strides2(g("ls", (64, 8))), _p(g("counts", 0)),
                                 g("heads_q", 2), g("tokens", 5), 1,
                                 ctypes.c_float(g("scale", 0.1)), ctypes.c_float(g("decay", -1.0)),
                                 g("fill", 0), g("dtype", 0), _p(g("ws", 256)), g("ws_bytes", 1 << 30), None)


SHARED = [
    (dict(pages=0), BAD), (dict(positions=0), BAD), (dict(weights=0), BAD),
    (dict(page_table=0), BAD), (dict(num_pages=0), BAD), (dict(heads=0), BAD),
    (dict(page_size=48), BAD), (dict(page_size=8), BAD), (dict(page_size=512), BAD),
    (dict(group=16), BAD), (dict(group=0), BAD), (dict(batch=0), BAD), (dict(max_pages=0), BAD),
    (dict(table_stride=3), BAD), (dict(pages=24), UNSUP), (dict(positions=18), UNSUP),
    (dict(weights=18), UNSUP), (dict(page_table=18), UNSUP), (dict(heads=2000), UNSUP),
    (dict(num_pages=1 << 31), UNSUP), (dict(batch=5000), UNSUP),
    (dict(max_pages=1 << 24, table_stride=1 << 24), UNSUP),
]
ROWS = [
    (dict(lengths=0), BAD), (dict(lengths=18), UNSUP), (dict(k=0), BAD), (dict(v=0), BAD),
    (dict(k=24), UNSUP), (dict(ks=(1 << 20, 256, 100)), UNSUP), (dict(ks=(0, 256, 128)), UNSUP),
    (dict(ks=(1 << 20, -256, 128)), UNSUP), (dict(tokens=0), BAD), (dict(tokens=1 << 24), UNSUP),
    (dict(dtype=2), BAD), (dict(dtype=-1), BAD), (dict(counts=18), UNSUP),
]


@pytest.mark.parametrize("kw,code", SHARED + ROWS + [(dict(seen=18), UNSUP)])
def test_append_refuses_without_cuda(L, kw, code):
    assert _append(L, **kw) == code


@pytest.mark.parametrize("kw,code", SHARED + ROWS)
def test_expand_refuses_without_cuda(L, kw, code):
    assert _expand(L, **kw) == code


@pytest.mark.parametrize("kw,code", SHARED + ROWS + [
    (dict(heads_q=3), BAD), (dict(heads_q=0), BAD), (dict(scale=0.0), BAD),
    (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(decay=1.5), BAD),
    (dict(decay=float("nan")), BAD), (dict(ws=0), BAD), (dict(ws=24), BAD), (dict(ws_bytes=16), BAD),
    (dict(lse=18), BAD), (dict(lse=16, ls=(0, 8)), BAD), (dict(lse=16, ls=(64, 0)), BAD),
])
def test_attention_refuses_without_cuda(L, kw, code):
    assert _attend(L, **kw) == code


@pytest.mark.parametrize("fill", [4, -1, 8 | 1])
def test_attention_refuses_unknown_fills(L, fill):
    assert _attend(L, fill=fill) == BAD


@pytest.mark.parametrize("scale,code", [(3e38, BAD), (2.4e38, BAD), (-1.0, BAD)])
def test_attention_refuses_a_scale_that_log2_e_takes_out_of_range(L, scale, code):
    assert 2.4e38 * 1.4427 > 3.4029e38
    assert _attend(L, scale=scale) == code


def _select(L, **kw):
    c, s, kw = _structs(kw)
    g = lambda n, d: kw.get(n, d)  # noqa: E731
    return L.llmfa_kv4_evict_select(c, s, _p(g("seen", 0)), g("keep", 64), g("recent", 8),
                                    _p(g("src", 16)), _p(g("new", 16)), _p(g("ws", 256)),
                                    g("ws_bytes", 1 << 30), None)


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(lengths=0), BAD), (dict(keep=0), BAD), (dict(recent=-1), BAD), (dict(recent=65), BAD),
    (dict(src=0), BAD), (dict(new=0), BAD), (dict(src=18), UNSUP), (dict(new=18), UNSUP),
    (dict(seen=18), UNSUP), (dict(keep=1 << 31), UNSUP),
])
def test_select_refuses_without_cuda(L, kw, code):
    assert _select(L, **kw) == code


@pytest.mark.parametrize("keep", [2 ** 31 - 1, 2 ** 31 - 8191])
def test_select_refuses_a_budget_whose_last_step_passes_32_bits(L, keep):
    assert _select(L, keep=keep, ws_bytes=1 << 60) == UNSUP
    n = ctypes.c_uint64(0)
    assert L.llmfa_kv4_evict_workspace_size(1, 1, keep, ctypes.byref(n)) == UNSUP
    assert L.llmfa_kv4_evict_workspace_size(1, 1, 2 ** 31 - 8192, ctypes.byref(n)) == _lib.LLMFA_OK


@pytest.mark.parametrize("kw,code", SHARED + [
    (dict(src=0), BAD), (dict(keep=0), BAD), (dict(src=18), UNSUP), (dict(keep=1 << 31), UNSUP)])
def test_move_refuses_without_cuda(L, kw, code):
    c, s, kw = _structs(dict(kw, lengths=0))
    assert L.llmfa_kv4_evict_move(c, s, _p(kw.get("src", 16)), kw.get("keep", 64), None) == code


def test_null_structs_and_workspace_sizes(L):
    c, s, _ = _structs({})
    assert L.llmfa_kv4_evict_move(None, s, _p(16), 4, None) == BAD
    assert L.llmfa_kv4_evict_move(c, None, _p(16), 4, None) == BAD
    n = ctypes.c_uint64(0)
    size = L.llmfa_kv4_attention_workspace_size
    assert size(1, 1, 1, 1, 0, None) == BAD
    assert size(0, 1, 1, 1, 0, ctypes.byref(n)) == BAD
    assert size(1, 2, 3, 1, 0, ctypes.byref(n)) == BAD
    assert size(1, 1, 1, 1, -1, ctypes.byref(n)) == BAD
    assert size(5000, 1, 1, 1, 0, ctypes.byref(n)) == UNSUP
    assert size(4096, 8, 64, 1 << 20, 0, ctypes.byref(n)) == UNSUP
    # tracking keeps scores of up to 256 MB
    need = []
    for capacity in (0, 1 << 20, (1 << 20) + 64):
        assert size(2, 4, 32, 1, capacity, ctypes.byref(n)) == _lib.LLMFA_OK
        need.append(n.value)
    assert need[0] < need[2] < need[1] and need[1] - need[2] == 256 << 20


def test_python_surface_refuses_cpu_tensors():
    build()
    pages = torch.zeros(2, 1, kv4.page_bytes(16, 128), dtype=torch.uint8)
    ints, floats = torch.zeros(2, 1, 16, dtype=torch.int32), torch.zeros(2, 1, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        KV4Cache(pages, ints, floats, page_size=16, group=128)
    with pytest.raises(RuntimeError, match="page_size"):
        KV4Cache(pages, ints, floats, page_size=20)
    with pytest.raises(RuntimeError, match="group"):
        KV4Cache(pages, ints, floats, page_size=16, group=48)
    with pytest.raises(RuntimeError, match="bytes"):
        KV4Cache(pages, ints, floats, page_size=32, group=128)
    with pytest.raises(RuntimeError, match="positions"):
        KV4Cache(pages, floats, floats, page_size=16, group=128)
