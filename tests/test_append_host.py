"""The C entry of appends and how rows find their sequences, on the CPU: the search
ends at the right place for every number of lanes that the plan of a call gives a row."""
import os
import shutil
import subprocess

import pytest

from mtpx import capi, ops
from test_head_norm_rows_gpu import WORKGROUP_ROWS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not available")
    exe = str(tmp_path_factory.mktemp("calls") / "append_calls")
    subprocess.run([hipcc, "-O1", "-std=c++17", "-w", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "imr-mlp_amd", "csrc"),
                    os.path.join(ROOT, "tests", "append_calls.cpp"), "-o", exe], check=True)

    def run(*args):
        out = subprocess.run([exe, *map(str, args)], check=True, capture_output=True, text=True, timeout=60).stdout
        return [line.split() for line in out.splitlines()]

    return run


def test_a_search_ends_where_it_should(calls):
    looked, wrong = (int(v) for v in calls("search")[0])
    assert looked > 300000 and wrong == 0


@pytest.mark.parametrize("dtype,dim,rotated,interleaved,heads", [
    (1, 16, 16, 0, 1), (1, 8, 8, 1, 1), (0, 8, 8, 0, 2), (0, 2, 2, 0, 1), (1, 8, 0, 0, 1), (2, 64, 64, 0, 8), (0, 255, 2, 1, 3)])
def test_lanes_of_a_row(calls, dtype, dim, rotated, interleaved, heads):
    """A row's lanes are a power of two from a vector's up to a workgroup, one among
    them where vectors are short and rows many.  A launch's threads, whole workgroups
    of them, are a 32-bit number up to the most rows, and more are refused."""
    seen = set()
    for rows, *line in calls("lanes", dtype, dim, rotated, interleaved, heads):
        rows = int(rows)
        assert (line[0] == "refused") == (rows > 2 ** 26 - 4), rows
        if line[0] == "refused":
            assert int(line[1]) == capi.ERRORS_BY_NAME["MTPX_E_CAPACITY"]
            continue
        group, lanes = (int(v) for v in line)
        assert -(-rows * lanes // 256) * 256 < 2 ** 32
        assert lanes & (lanes - 1) == 0 and group <= lanes <= 256
        seen.add((group, lanes))
    assert ((1, 1) in seen) == (min(g for g, _ in seen) == 1)


@pytest.mark.parametrize("rows,heads,maps,dim,rotated,dtype,interleaved", WORKGROUP_ROWS)
def test_a_workgroup_has_rows_one_after_the_other(calls, rows, heads, maps, dim, rotated, dtype, interleaved):
    """The shapes that the device's test of such rows takes have a workgroup a row, and fewer workgroups than rows."""
    lanes, parts = (int(v) for v in calls("backward", rows, heads, maps, dim, rotated, int(interleaved), ops.DTYPES[dtype])[0])
    assert lanes == 256 and parts < rows


def test_weights_without_a_norm(calls):
    """Keys go into their pages as they are: a weight is refused, nothing is queued."""
    for kind, given, code, queued in ([int(v) for v in line] for line in calls("weights")):
        wrong = kind == ops.APPEND_NORMS["none"] and given > 0
        assert (code, queued) == ((capi.ERRORS_BY_NAME["MTPX_E_INVALID"], 0) if wrong else (0, 1)), (kind, given)
