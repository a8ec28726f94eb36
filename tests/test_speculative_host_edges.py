"""Speculative decoding, host side: what kernels and wrappers have to hold at the edges of their arguments (no GPU)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from esolearn_b200 import _native as N
from esolearn_b200 import speculative as S

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "esolearn_b200", "csrc")


@pytest.fixture(scope="module")
def pace(tmp_path_factory):
    """clocks_passed of the kernels' pacing loop, compiled for the host."""
    d = tmp_path_factory.mktemp("pace")
    src, lib = d / "pace.cpp", d / "libpace.so"
    src.write_text('#include "clock_pace.cuh"\nextern "C" int passed(uint32_t a, uint32_t b, uint32_t n) { return sb::clocks_passed(a, b, n); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, "-o", str(lib), str(src)], check=True)
    f = C.CDLL(str(lib)).passed
    f.argtypes, f.restype = [C.c_uint32] * 3, C.c_int
    return f


@pytest.mark.parametrize("start", [0, 1, 2 ** 31 - 30, 2 ** 31, 2 ** 32 - 1000, 2 ** 32 - 62, 2 ** 32 - 1])
@pytest.mark.parametrize("n", [62, 62 * 13])
def test_pacing_ends_across_the_counters_wrap(pace, start, n):
    """Read every 20 clocks from `start` on, the wait is over at the first reading n clocks later, and stays over."""
    for dt in range(0, 4 * n, 20):
        assert bool(pace(start, (start + dt) % 2 ** 32, n)) == (dt >= n)


@pytest.mark.parametrize("make", [lambda x: x[:1].expand(3, 7), lambda x: x.flatten().as_strided((3, 7), (5, 1)), lambda x: x, lambda x: x[:, :6],
                                  lambda x: x[:1, :5], lambda x: x[::2], lambda x: x[:0]])
def test_rows_of_a_matrix_stay_inside_its_storage(make):
    """Row i of what a kernel is given lies at i times the stride, within the tensor's memory, and holds row i."""
    x = make(torch.arange(21.0).view(3, 7))
    y, ld = S._matrix_rows(x)
    b, v = x.shape
    assert ld >= v
    last = y.storage_offset() + (b - 1) * ld + v
    assert b == 0 or last <= y.untyped_storage().nbytes() // 4
    assert torch.equal(torch.as_strided(y, (b, v), (ld, 1)), x)


class _On:
    """Stands for a tensor on a device."""

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


def test_tensors_of_another_device_are_refused(monkeypatch):
    """The library launches on the thread's current device: a stream of another one must not reach it."""
    monkeypatch.setattr(S, "_raw_stream", lambda i: 1000 + i)
    monkeypatch.setattr(S, "_raw_device", lambda: 1, raising=False)
    assert S._stream(_On(1)) == 1001
    for other in (0, 2):
        with pytest.raises(N.SbError, match=f"cuda:{other}"):
            S._stream(_On(other))


def test_recorded_wait_errors_are_taken_one_by_one(tmp_path):
    """The words that kernels set when a wait gives up: each is reported once and cleared."""
    src, lib = tmp_path / "w.cpp", tmp_path / "libw.so"
    src.write_text('#include "wait_errors.cuh"\nextern "C" int take(unsigned *w) { return sb::take_wait_error(w); }\n'
                   'extern "C" int words() { return sb::WAIT_ERRORS; }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I" + CSRC, "-o", str(lib), str(src)], check=True)
    l = C.CDLL(str(lib))
    n = l.words()
    w = (C.c_uint * n)()
    assert l.take(w) == -1
    for i in range(n):
        w[i] = 1
    assert [l.take(w) for _ in range(n + 1)] == list(range(n)) + [-1]
    assert list(w) == [0] * n


def test_every_entry_point_reports_a_wait_that_gave_up_before():
    """Wrappers never call sb_stream_sync: without this, outputs would be wrong in silence."""
    lib = N.lib()
    path = [l.split()[-1] for l in open("/proc/self/maps") if l.rstrip().endswith("libscryb200.so")][0]
    base = min(int(l.split("-")[0], 16) for l in open("/proc/self/maps") if l.rstrip().endswith("libscryb200.so"))
    at = [l.split()[0] for l in subprocess.run(["nm", path], capture_output=True, text=True, check=True).stdout.splitlines() if "g_wait_errors" in l and "g_wait_errors_mu" not in l]
    assert len(at) == 1
    place = C.c_void_p.from_address(base + int(at[0], 16))
    words, before = (C.c_uint * 16)(), place.value
    calls = [lambda: lib.sb_kv_append(0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0, 1.0, 0, 0), lambda: lib.sb_kv_commit(0, 1, 0, 0, 1, 0, 0),
             lambda: lib.sb_kv_read(0, 1, 0, 1, 0, 0, 0, 0), lambda: lib.sb_tree_attention(0, 0, 0, 0, 1, 1, 1, 0, 0, 0, 0, 1, 0, 0),
             lambda: lib.sb_verify_drafts(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 1, 1.0, 0, 0, 0, 0)]
    place.value = C.addressof(words)
    try:
        for call in calls:
            words[0] = 1
            with pytest.raises(N.SbError, match="timed out"):
                N.check(call())
            assert words[0] == 0
            with pytest.raises(N.SbError) as e:  # its own null pointers, from now on
                N.check(call())
            assert "timed out" not in str(e.value)
    finally:
        place.value = before


@pytest.mark.parametrize("temperature", [float("inf"), float("nan")])
def test_temperatures_that_are_none_are_refused(temperature):
    """An infinite temperature would turn a masked logit (-inf) into a NaN exponent; refused before any launch."""
    args = [256, 8, 256, 256, 0, 0, 0, 256, 256, 8, 1, 2, 8, temperature, 256, 256, 256, 0]
    with pytest.raises(N.SbError, match="temperature"):
        N.check(N.lib().sb_verify_drafts(*args))
