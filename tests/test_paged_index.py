"""The paged cache's index arithmetic (csrc/fw_paged.h, the same code the
kernels run), compiled for the host: division by the page size, what a request
asks of the plan, slots (CPU)."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("paged") / "paged_index.so")
    subprocess.run(["gcc", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "franken_whisper_amd", "csrc"), os.path.join(ROOT, "tests", "paged_index.c"),
                    "-o", out], check=True)
    L = C.CDLL(out)
    L.t_div.restype = C.c_uint32
    L.t_div.argtypes = [C.c_uint32, C.c_uint32]
    L.t_div_bad.restype = C.c_int64
    L.t_div_bad.argtypes = [C.c_uint32] * 4
    L.t_slot.restype = C.c_int64
    L.t_slot.argtypes = [C.c_int32, C.c_uint32, C.c_uint32]
    return L


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 16, 24, 31, 32, 33, 100, 127, 128, 255, 256, 641, 4096, 65537,
                               (1 << 24) - 1, 1 << 24])
def test_division_by_the_page_size_is_exact(lib, d):
    top = (1 << 31) - 1
    assert lib.t_div_bad(d, 0, 300000, 1) == 0
    assert lib.t_div_bad(d, top - 300000, top + 1, 1) == 0
    assert lib.t_div_bad(d, 0, top, 9973) == 0
    for q in range(1, min(top // d, 50000)):  # around multiples
        for n in (q * d - 1, q * d, q * d + 1):
            assert lib.t_div(n, d) == n // d


def _req(lib, *a):
    rows, need, status = C.c_int64(), C.c_int64(), C.c_int()
    lib.t_req(*a, C.byref(rows), C.byref(need), C.byref(status))
    return rows.value, need.value, status.value


def test_what_a_request_asks_for(lib):
    big = (1 << 31) - 1
    assert _req(lib, 0, 0, 0, 4, 16) == (0, 0, 0)
    assert _req(lib, 0, 1, 0, 4, 16) == (1, 1, 0)
    assert _req(lib, 15, 1, 1, 4, 16) == (1, 0, 0)
    assert _req(lib, 16, 1, 1, 4, 16) == (1, 1, 0)
    assert _req(lib, 60, 5, 4, 4, 16) == (5, 0, 1)     # the table row is full
    assert _req(lib, 3, 64, 1, 5, 16) == (64, 4, 0)
    assert _req(lib, 3, 4, 3, 5, 16) == (4, 0, 0)      # pages of tokens taken back are still held
    assert _req(lib, -1, 4, 0, 5, 16) == (4, 0, 2)
    assert _req(lib, 1, -4, 0, 5, 16) == (0, 0, 2)
    assert _req(lib, 1, 4, -1, 5, 16) == (4, 0, 2)
    assert _req(lib, 1, 4, 6, 5, 16) == (4, 0, 2)
    assert _req(lib, big, big, 0, 5, 16) == (big, 0, 2)
    assert _req(lib, big - 40, 8, 0, 5, 16) == (8, 0, 1)
    assert _req(lib, big, 0, 0, 5, 1) == (0, 0, 2)     # no token index of 2^31 - 1


def test_requests_against_plain_arithmetic(lib):
    rng = random.Random(3)
    for _ in range(5000):
        page = rng.choice((1, 2, 3, 16, 24, 64, 1000))
        ln, new, width = rng.randint(0, 5000), rng.randint(0, 300), rng.randint(0, 400)
        held = rng.randint(0, width)
        want = max(0, -(-(ln + new) // page) - held)
        fits = want <= width - held
        assert _req(lib, ln, new, held, width, page) == (new, want if fits else 0, 0 if fits else 1)


def test_slots(lib):
    assert lib.t_slot(-1, 5, 16) == -1
    assert lib.t_slot(0, 0, 16) == 0
    assert lib.t_slot(7, 37, 16) == 7 * 16 + 5
    assert lib.t_slot((1 << 31) - 1, 37, 16) == ((1 << 31) - 1) * 16 + 5
