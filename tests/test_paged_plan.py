"""How the paged attention cuts a call into workgroups (csrc/attn_paged_plan.hpp, compiled here as host code) against
the workspace that the library asks for: what a plan writes has to fit, for the same numbers and for larger ones."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = 0, 3  # jas_dtype
ROUNDS, LEAST = {16: 8, 64: 4, 128: 2}, {16: 128, 64: 256, 128: 256}

SHIM = """
#include "jasmine_amd/csrc/attn_paged_plan.hpp"
extern "C" void plan(int n, int B, int H, int n_kv, int D, int max_q, int max_len, int dtype, long cus, long *out)
{
    const jas::PagedPlan p = jas::paged_plan(n, B, H, n_kv, max_q, max_len, dtype, cus);
    out[0] = p.rows, out[1] = p.tiles, out[2] = p.nsplit, out[3] = p.chunk, out[4] = (long)jas::paged_need(p, n_kv, D);
}
extern "C" size_t bytes(int n, int B, int H, int n_kv, int D, int max_q, int max_len, double cus)
{
    return jas::paged_workspace(n, B, H, n_kv, D, max_q, max_len, cus);
}
"""


@pytest.fixture(scope="module")
def shim(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-I", ROOT, str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.plan.argtypes, lib.plan.restype = [C.c_int] * 8 + [C.c_long, C.POINTER(C.c_long)], None
    lib.bytes.argtypes, lib.bytes.restype = [C.c_int] * 7 + [C.c_double], C.c_size_t
    return lib


def plan(shim, n, B, H, n_kv, D, max_q, max_len, dtype, cus=256):
    out = (C.c_long * 5)()
    shim.plan(n, B, H, n_kv, D, max_q, max_len, dtype, cus, out)
    return dict(zip(("rows", "tiles", "nsplit", "chunk", "need"), out))


def fits(shim, call, within=None, dtypes=(F32, BF16), cus=256):
    """call: n, B, H, n_kv, D, max_q, max_len; within: the numbers that the workspace is asked for."""
    size = shim.bytes(*(within or call), cus)
    for dtype in dtypes:
        p = plan(shim, *call, dtype, cus)
        assert p["need"] <= size, (call, within, dtype, p, size)
        assert p["tiles"] > 0 and 1 <= p["nsplit"] <= 63 and (p["nsplit"] % 2) and p["chunk"] > 0
        if size == 0:
            assert p["nsplit"] == 1


# shares of the keys just above a multiple of 128: tiles of 16, 64 and 128 rows, max_q below the real one too
TIGHT = [
    (393, 9, 3, 1, 64, 156, 14619), (145, 9, 8, 1, 128, 145, 14610), (145, 9, 8, 1, 128, 32, 14610), (193, 3, 6, 3, 128, 128, 14610),
    (83, 36, 7, 1, 128, 2, 7297), (412, 412, 16, 1, 128, 1, 641), (229, 229, 16, 1, 128, 1, 1153), (294, 294, 16, 1, 64, 1, 897),
    (206, 206, 32, 2, 128, 1, 641),
]


@pytest.mark.parametrize("call", TIGHT)
def test_plan_fits_its_workspace(shim, call):
    fits(shim, call)


def test_plans_around_every_share(shim):
    """Draws whose keys are an odd number of splits and a few more, at shares around the splits' multiple of 128: one split
    more than the share gives would be two with the odd number that is launched."""
    rng = np.random.default_rng(1)
    for _ in range(20000):
        rows, n_kv, G = int(rng.choice([16, 64, 128])), int(rng.choice([1, 1, 2, 3, 4])), int(rng.choice([1, 2, 3, 4, 7, 8, 16]))
        chunk = 128 * int(rng.integers(LEAST[rows] // 128, 6))
        max_len = chunk * int(rng.choice([1, 3, 5, 7, 9, 15, 31, 57])) + int(rng.integers(0, 12))
        full = ROUNDS[rows] * 256 * (chunk + rng.uniform(-1, 2)) / max_len
        B = max(1, round(full / n_kv))
        n = max(1, min(B * rows // G + int(rng.integers(0, max(2, rows // G))), 1 << 20))
        if rng.random() < .2:
            B = int(rng.integers(1, B + 1))
        most = {16: 16 // G, 64: 64 // G, 128: n}[rows]
        for max_q in {max(1, most), max(1, 16 // G)}:
            fits(shim, (n, B, G * n_kv, n_kv, int(rng.choice([32, 64, 128])), max_q, max_len))


def test_plans_within_a_larger_workspace(shim):
    """Any smaller call fits the workspace of larger numbers; other chips' numbers of units too."""
    rng = np.random.default_rng(2)
    upto = lambda hi: int(np.exp(rng.uniform(0, np.log(hi)))) if hi > 1 else 1  # noqa: E731
    for _ in range(20000):
        n, B, max_q, max_len = upto(20000), upto(3000), upto(2000), upto(2 ** 31 - 1)
        g, kv, D = int(rng.choice([1, 2, 4, 7, 16])), int(rng.choice([1, 2, 8, 12, 32])), int(rng.choice([32, 64, 128]))
        less = [upto(v) for v in (n, B, max_q, max_len)]
        fits(shim, (less[0], less[1], g * kv, kv, D, less[2], less[3]), (n, B, g * kv, kv, D, max_q, max_len), cus=int(rng.choice([256, 256, 256, 304, 80, 1])))


def test_library_asks_for_the_same(shim):
    if not os.path.exists(os.path.join(ROOT, "jasmine_amd", "libjasmine_hip.so")):
        pytest.skip("library not built")
    from jasmine_amd.capi import lib
    for call in TIGHT:
        sizes = {shim.bytes(*call, cus) for cus in (256, 304)}  # (256 where there is no device)
        assert lib.jas_attn_paged_workspace(*call) in sizes
