"""Shared memory of the one-kernel int8 expert layer: the sizes that its launch is made with (csrc/moe_i8_sizes.h, compiled here by itself), and
that no stage of the ring is read beyond its end.  A read out of range cannot be shown by running it."""
import ctypes as C
import os
import random
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-scaler_b200", "csrc")
FIELDS = ("grid", "pitch", "row_cap", "xr", "front", "up_piece", "down_piece", "down_rows", "stages", "stage_bytes", "smem")


class Sizes(C.Structure):
    _fields_ = [(n, C.c_int) for n in FIELDS]


@pytest.fixture(scope="module")
def sizes(tmp_path_factory):
    d = tmp_path_factory.mktemp("sizes")
    src, lib = str(d / "sizes.cpp"), str(d / "sizes.so")
    with open(src, "w") as f:
        f.write('#include "moe_i8_sizes.h"\n'
                'extern "C" int fields() { return sizeof(b2q::mi8::Sizes) / sizeof(int); }\n'
                'extern "C" int limit() { return b2q::mi8::SMEM_MAX - b2q::mi8::STATIC_BYTES; }\n'
                'extern "C" void sizes(int T, int k, int H, int I, int pitch, int sms, b2q::mi8::Sizes* s) { *s = b2q::mi8::sizes_of(T, k, H, I, pitch, sms); }\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, src, "-o", lib], check=True)
    so = C.CDLL(lib)
    assert so.fields() == len(FIELDS)

    def get(T, k, H, I, sms=148):
        s = Sizes()
        so.sizes(T, k, H, I, (H + 127) // 128 * 128 + 64, sms, C.byref(s))
        return s
    get.limit = so.limit()
    return get


def _source():
    with open(os.path.join(CSRC, "moe_i8.cu")) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _second_rows_are_bounded():
    """Whether multiply16() loads a lane's second weight row only where the stage has one."""
    text = _source()
    body = text.split("void multiply16(")[1].split("\n}\n")[0]
    name = re.search(r"bool (\w+), int len", body.split("{")[0]).group(1)
    call = re.search(r"multiply16\(acc, ([^;]*)\);", text).group(1)
    return bool(re.search(r"if \(in && %s\) c = lds\(v \+ k\);" % name, body)) and name != "has" and "g + 8 < min(sr, left)" in call


def _preferred(T, k, H, I, row_cap):
    return T <= 16 and T * (4 * k * I + H) <= 40960 and T * k * row_cap * 4 <= 24 * 1024


def _check(s, T, k, H, I, limit):
    assert s.smem <= limit and s.stages >= 5, (T, k, H, I)      # six, but for the rounding of a stage to 128 bytes
    assert s.stage_bytes % 128 == 0 and (s.up_piece == H or s.up_piece % 64 == 0) and (s.down_piece == I or s.down_piece % 64 == 0)
    # weights, from the start of a stage: eight rows at a time, or the rows that a multiplication of sixteen reads
    rows = 8 if s.down_rows <= 8 else (s.down_rows if _second_rows_are_bounded() else 16)
    assert 8 * s.up_piece <= s.stage_bytes, (T, k, H, I)
    assert rows * s.down_piece <= s.stage_bytes, (T, k, H, I, rows, s.down_piece, s.stage_bytes)
    # codes of h, behind the weights
    assert s.down_rows * s.down_piece + s.xr * (s.down_piece + 16) <= s.stage_bytes, (T, k, H, I)


@pytest.mark.parametrize("T,k,H,I", [(1, 2, 1280, 2048), (1, 4, 1408, 2048), (1, 8, 2048, 768), (2, 2, 1344, 1024), (3, 1, 1504, 1024), (1, 1, 2400, 2048)])
def test_down_stages_of_nine_to_fifteen_rows(sizes, T, k, H, I):
    s = sizes(T, k, H, I)
    assert 9 <= s.row_cap and _preferred(T, k, H, I, s.row_cap)
    _check(s, T, k, H, I, sizes.limit)


@pytest.mark.parametrize("sms", [148, 132, 74, 16])
def test_no_stage_is_read_beyond_its_end(sizes, sms):
    rng = random.Random(sms)
    seen = 0
    for H in range(1024, 4097, 16):
        for _ in range(20):
            T, k, I = rng.randint(1, 16), rng.randint(1, 8), 16 * rng.randint(1, 256)
            T = min(T, max(1, 40960 // (4 * k * I + H)))
            s = sizes(T, k, H, I, sms)
            if _preferred(T, k, H, I, s.row_cap):
                seen += 1
                _check(s, T, k, H, I, sizes.limit)
    for _ in range(4000):                                    # and everything else that one kernel serves
        T, k, H, I = rng.randint(1, 16), rng.randint(1, 32), 16 * rng.randint(1, 2048), 16 * rng.randint(1, 640)
        s = sizes(T, k, H, I, sms)
        if _preferred(T, k, H, I, s.row_cap):
            seen += 1
            _check(s, T, k, H, I, sizes.limit)
    assert seen > 1000
