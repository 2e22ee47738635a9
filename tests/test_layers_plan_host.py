"""The layer norm's plans, from the header that makes them, compiled here: every plan has a kernel, fits the GPU, and finds in
the workspace that a caller is told to bring the room that it writes to."""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest

from serron_b200 import _lib

PACKAGE = os.path.dirname(os.path.abspath(_lib.__file__))
FIELDS = ("ok", "rows", "V", "NV", "R", "shifted", "full", "tx", "ty", "clusters", "tiles", "blocks", "floats")
SOURCE = """
#include "layer_plan.h"
extern "C" void plan(const int64_t* in, int64_t* out) {
    const serron::NormPlan p = serron::norm_plan(in[0], in[1], in[2], in[3], in[4], in[5]);
    const int64_t v[] = {p.ok, p.rows, p.V, p.NV, p.R, p.shifted, p.full, p.tx, p.ty, p.clusters, p.tiles, p.blocks,
                         p.ok ? serron::plan_shared_floats(p, in[5]) : 0};
    for (int i = 0; i < 13; ++i) out[i] = v[i];
}
extern "C" int width(int rows, int size, int k) { return serron::plan_widths(rows, size)[k]; }
"""


@pytest.fixture(scope="module")
def planner(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs a C++ compiler")
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", f"-I{os.path.join(PACKAGE, 'csrc')}", "-o",
                    str(at / "plan.so"), str(at / "plan.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "plan.so"))

    def plan(rows, length, inner, v, size, backward):
        out = (ctypes.c_int64 * len(FIELDS))()
        lib.plan((ctypes.c_int64 * 6)(rows, length, inner, v, size, backward), out)
        return dict(zip(FIELDS, out))

    def chosen(outer, length, inner, width, size, backward):
        """The plan of a call whose pointers allow vectors of ``width``, or None."""
        k = 0
        while (v := lib.width(int(inner == 1), size, k)) != 0:
            if v <= width:
                p = plan(outer * inner, length, inner, v, size, int(backward))
                if p["ok"]:
                    return p
            k += 1
        return None

    return chosen


def _sizes(count):
    rng = random.Random(5)

    def log(low, high):
        return min(high, int(low * (high / low) ** rng.random()))

    yield from [(1, 1, 1), (8192, 1024, 1), (64, 32, 65536), (33, 50001, 1), (150000, 16, 1), (5, 67, 5917), (1, 131072, 1),
                (1, 131073, 1), (64, 256, 65536), (1, 2048, 4), (1, 2049, 4), (3, 1, 7), (1 << 20, 7, 1), (2, 16, 1 << 26)]
    for _ in range(count):
        length = log(1, 300000)
        if rng.random() < 0.5:
            yield log(1, max(1, (1 << 31) // length)), length, 1
        else:
            inner = log(2, max(2, min(1 << 20, (1 << 31) // length)))
            yield log(1, max(1, (1 << 31) // (length * inner))), length, inner


def test_plans_have_kernels_and_fit(planner):
    for outer, length, inner in _sizes(4000):
        for size in (2, 4):
            wide = 16 // size
            for backward in (False, True):
                for width in (1, 2, 4, 8):
                    p = planner(outer, length, inner, width, size, backward)
                    if p is None:
                        continue
                    at = (outer, length, inner, size, backward, p)
                    shape = (p["V"], p["NV"], p["R"])
                    if p["rows"]:
                        assert shape in {(wide, 1, 4), (wide, 1, 1), (wide, 2, 2), (wide, 2, 1), (wide, 4, 1)} and p["V"] > 1 or (
                            shape in {(1, 4, 4), (1, 4, 1), (1, 16, 1)} and not p["shifted"]), at
                        assert not backward or p["NV"] * p["V"] <= 16, at
                        assert p["tx"] % 32 == 0 or 32 % p["tx"] == 0 and p["tx"] * p["ty"] >= 32, at
                        assert p["tx"] <= 512 and (p["tx"] <= 32 or p["ty"] == 1) and (p["clusters"] == 1 or p["ty"] == 1), at
                        vectors = -(-(length + (p["V"] - 1 if p["shifted"] else 0)) // p["V"])
                        assert p["tx"] * p["clusters"] * p["NV"] >= vectors, at  # every vector has its thread
                        # blocks that walk over the tiles of shifted rows keep their shift
                        assert not p["shifted"] or p["blocks"] == p["tiles"] or p["blocks"] % p["V"] == 0, at
                    else:
                        assert (p["V"], p["NV"]) in {(4, 4), (4, 8), (1, 8), (1, 16)} | ({(4, 16)} if size == 2 else set()), at
                        assert not (p["full"] and p["V"] == 1) and inner % p["V"] == 0, at
                        assert not backward or p["NV"] * p["V"] * size <= 64, at
                        assert p["tx"] % 32 == 0 and p["NV"] * p["ty"] * p["clusters"] >= length, at
                        assert not p["full"] or p["NV"] * p["ty"] * p["clusters"] == length, at
                        assert length * inner < 1 << 31, at
                    assert 32 <= p["tx"] * p["ty"] <= 512 and p["clusters"] in (1, 2, 4, 8), at
                    assert 1 <= p["blocks"] <= p["tiles"] and p["blocks"] < (1 << 31) - 1, at
                    assert 4 * p["floats"] <= 48 * 1024, at


def test_workspace_holds_what_the_plans_write(planner):
    size_of = _lib.load().serron_layer_norm_workspace_bytes
    for outer, length, inner in _sizes(3000):
        for dtype, size in ((0, 4), (1, 8), (2, 2), (3, 2)):
            for backward in (False, True):
                got = size_of(outer, length, inner, dtype, int(backward))
                acc, rows = (8 if dtype == 1 else 4), outer * inner
                plans = [planner(outer, length, inner, w, size, backward) if dtype != 1 else None for w in (1, 2, 4, 8)]
                need = [0]
                for p in plans:
                    if p is not None:  # two sums of every element of a row for each block
                        need.append(p["blocks"] * 2 * length * 4 if backward else 0)
                    else:  # two numbers a chunk of a row; statistics, or the parameters' first sums of 128 rows or 8192 columns
                        chunk = max(8192 if inner == 1 else 1024, -(-length // 65535))
                        sums = -(-rows // (128 if inner == 1 else 8192)) * 2 * length * acc
                        need.append(rows * -(-length // chunk) * 2 * acc + (sums if backward else rows * 2 * acc))
                assert max(need) <= got <= max(need) + 3 * 256, (outer, length, inner, dtype, backward, got, need)
