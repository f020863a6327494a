"""How the one-launch MXFP4 product is cut (comp_b200/csrc/mx_plan.h), compiled for the host: what its CTAs take of an SM."""

import ctypes
import os
import subprocess

import pytest

from tests.conftest import ROOT

SOURCE = r"""
#include "mx_plan.h"
extern "C" int plan(int64_t rows, int64_t used, int64_t row_tiles, int64_t stages, int sms, int64_t* out) {
  b2q::GemvPlan p;
  if (!b2q::plan_gemv(rows, used, row_tiles, stages, sms, &p)) return 0;
  out[0] = p.ranks, out[1] = p.nk, out[2] = p.ring, out[3] = p.columns, out[4] = (int64_t)p.smem;
  return 1;
}
extern "C" unsigned under_way(unsigned issued, unsigned ring) { return b2q::first_under_way(issued, ring); }
"""

SM_SMEM, RESERVED, COLUMNS, STAGE = 228 * 1024, 1024, 512, 17408


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(ROOT, "comp_b200", "csrc"), str(at / "plan.cpp"),
                    "-o", str(at / "plan.so")], check=True)
    lib = ctypes.CDLL(str(at / "plan.so"))
    lib.plan.argtypes = [ctypes.c_int64] * 4 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int64)]

    def call(rows, used, row_tiles, stages, sms=148):
        out = (ctypes.c_int64 * 5)()
        return dict(zip(("ranks", "nk", "ring", "columns", "smem"), out)) if lib.plan(rows, used, row_tiles, stages, sms, out) else None

    call.under_way = lib.under_way
    return call


@pytest.fixture(scope="module")
def every(plan):
    """The plans of all numbers of stages, from one tile to more than there are SMs."""
    cases = [(1, t, s) for t in (1, 8, 9, 18, 19, 32, 37, 38, 64, 74, 75, 149) for s in range(1, 940)]
    cases += [(u, t, s) for u in (2, 8, 32) for t in (1, 2, 16) for s in range(1, 130)]
    return [p for c in cases for p in [plan(4, *c)] if p]


def test_shared_and_tensor_memory_of_a_cta(every):
    for p in every:
        assert p["ranks"] in (1, 2, 4, 8) and 2 <= p["ring"] <= 8
        # the ring (aligned to 1024), the rows' codes with a gap after the last stage, their scales
        assert p["smem"] == p["ring"] * STAGE + (p["nk"] + 1) * 1024 + p["nk"] * 512 + 1024 <= 214 * 1024
        # two accumulators, two sets of weight scales, four columns a stage of x: the least power of two that leaves four free
        need = 48 + 4 * p["nk"] + 4
        assert p["columns"] in (64, 128, 256, 512) and need <= p["columns"] and (p["columns"] == 64 or 2 * need > p["columns"])


def test_no_mix_of_calls_is_short_of_tensor_memory(every):
    """Calls on several streams, of any sizes: the CTAs that an SM has shared memory for take no more than its 512 columns."""
    kinds = {(p["smem"] + RESERVED, p["columns"]) for p in every}
    step = 512  # bytes, rounded down for each CTA: more of them fit than in truth
    most = [0] * (SM_SMEM // step + 1)
    for b in range(len(most)):
        most[b] = max([0] + [most[b - s // step] + c for s, c in kinds if s // step <= b])
    assert most[-1] <= COLUMNS


def test_few_tiles_share_k(plan):
    assert plan(1, 1, 32, 8)["ranks"] == 4 and plan(1, 1, 8, 8)["ranks"] == 8 and plan(1, 1, 64, 32)["ranks"] == 2
    assert plan(1, 1, 75, 32)["ranks"] == 1 and plan(1, 8, 16, 16)["ranks"] == 1 and plan(1, 1, 1, 1)["ranks"] == 1


def test_refused(plan):
    assert plan(0, 1, 1, 1) is None and plan(5, 1, 1, 1) is None and plan(1, 1, 148, 116) is None and plan(1, 1, 1 << 30, 1) is None


@pytest.mark.parametrize("ring", [2, 3, 5, 8])
def test_copies_waited_for_at_the_end(plan, ring):
    """Barriers as the hardware keeps them (a wait for a parity ends when the phase of that parity has ended), stages asked for in
    turn while the last ones have not been seen by anyone: the waits cover every stage that may be under way, and end."""
    for issued in range(0, 4 * ring + 2):
        waits = {(i % ring, i // ring & 1) for i in range(plan.under_way(issued, ring), issued)}
        assert len(waits) == min(issued, ring)
        ended = [0] * ring  # phases that have ended, a slot: all but the last stage's of it are known to have
        for i in range(issued):
            ended[i % ring] += i + ring < issued
        for slot in range(min(issued, ring)):
            running = ended[slot] & 1  # the parity of the phase under way: what the slot's wait has to be for
            assert (slot, running) in waits and (slot, running ^ 1) not in waits
