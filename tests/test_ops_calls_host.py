"""The operators' C entry points over a recorded HIP runtime (tests/ops_calls.cpp)."""
import os
import shutil
import subprocess

import pytest

from mtpx import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc is not available")
    exe = str(tmp_path_factory.mktemp("calls") / "ops_calls")
    subprocess.run([hipcc, "-O1", "-std=c++17", "-w", "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "imr-mlp_amd", "csrc"),
                    os.path.join(ROOT, "tests", "ops_calls.cpp"), "-o", exe], check=True)

    def run(*args):
        out = subprocess.run([exe, *map(str, args)], check=True, capture_output=True, text=True, timeout=60).stdout
        return [line.split() for line in out.splitlines()]

    return run


def test_the_callers_device_stays_current(calls):
    """A program (torch) with several GPUs keeps its own current device."""
    seen = calls("device")
    assert [s[0] for s in seen] == ["sequences_create", "rotary", "diff_attention", "diff_attention_backward",
                                    "diff_attention_cache", "norm_block", "norm_block_backward", "sequences_destroy"]
    for name, code, queued, after in seen:
        assert code == "0" and after == "1", (name, code, after)
        assert queued in ("0", "-1") and (queued == "0" or name == "sequences_destroy"), name


@pytest.mark.parametrize("n,rows", [(1, 2 ** 30), (60, 2 ** 30), (2, 300_000_000)])
def test_too_many_rows_are_refused_before_tables_are_built(calls, n, rows):
    """A row of a table is 32 bytes per 64 rows and side: 60 sequences of 2^30
    rows would take 97 GB of the host before they were found too many."""
    assert calls("sequences", n, rows, 100) == [[str(capi.ERRORS_BY_NAME["MTPX_E_CAPACITY"])]]


def test_many_rows_are_taken(calls):
    assert calls("sequences", 200, 1_000_000, 2000) == [["0"]]
