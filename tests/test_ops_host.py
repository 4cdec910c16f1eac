"""Operators on device tensors, what needs no GPU: the binding's structures
against the header's, refusals before any device work, and the oracle's own
gradients against differences."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

import ops_oracle as OO
from mtpx import capi, ops

PAIRS = {"mtpx_rows": ops.Rows, "mtpx_rotary_request": ops.RotaryRequest,
         "mtpx_diff_attention_request": ops.AttentionRequest,
         "mtpx_diff_attention_cache_request": ops.CacheRequest,
         "mtpx_norm_block_request": ops.NormRequest}


def test_structures_match_the_header(workdir):
    """Offsets and sizes as the C compiler lays the header's structures out."""
    src, exe = os.path.join(workdir, "layout.c"), os.path.join(workdir, "layout")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mtpx.h"', "int main(void) {"]
    for name, cls in PAIRS.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        for f, _ in cls._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, f.rstrip("_")))
    open(src, "w").write("\n".join(lines + ["return 0; }"]))
    subprocess.run([os.environ.get("CC", "gcc"), "-I", os.path.dirname(capi.HEADER), src, "-o", exe],
                   check=True)
    got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True).stdout.split()]
    want = []
    for cls in PAIRS.values():
        want.append(C.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_null_arguments_are_refused():
    L = ops._ops()
    n, h = C.c_size_t(), C.c_void_p()
    assert L.mtpx_rotary(None, None) == -1
    assert L.mtpx_rotary(None, C.byref(ops.RotaryRequest())) == -1
    for f, r in (("diff_attention", ops.AttentionRequest), ("diff_attention_cache", ops.CacheRequest),
                 ("norm_block", ops.NormRequest)):
        assert getattr(L, "mtpx_" + f)(None, C.byref(r())) == -1
        assert getattr(L, "mtpx_%s_workspace" % f)(None, C.byref(r()), C.byref(n)) == -1
    assert L.mtpx_sequences_create(None, 0, None, None, C.byref(h)) == -1 and not h.value
    L.mtpx_sequences_destroy(None)


def test_torch_comes_before_the_library():
    """In a process of its own: the library used first, then mtpx.ops."""
    code = "import sys; sys.path.insert(0, %r); from mtpx import capi; capi.lib(); from mtpx import ops"
    code = code % os.path.join(capi.ROOT, "imr-mlp_amd")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode != 0 and "before the first call of mtpx.capi" in r.stderr
    ok = subprocess.run([sys.executable, "-c", code.replace("import sys;", "import sys, torch;")], capture_output=True)
    assert ok.returncode == 0


class _Ctx:
    device, h = 0, None


def test_host_tensors_are_refused():
    x = torch.zeros(2, 1, 4)
    with pytest.raises(capi.MtpxError):
        ops.rotary(_Ctx, x, torch.zeros(2, 3), torch.ones(2), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(capi.MtpxError):
        ops.norm_block(_Ctx, None, torch.zeros(2, 4))


@pytest.mark.parametrize("causal", [False, True])
def test_oracle_gradients_against_differences(causal):
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(s, generator=g).double() for s in ((7, 4, 2, 3), (9, 2, 2, 3), (9, 2, 6)))
    lam = torch.rand(4, generator=g).double()
    dout = torch.randn(7, 4, 6, generator=g).double()
    mask = torch.rand(9, generator=g) > 0.3
    at = ([0, 3, 7], [0, 2, 9])

    def loss(*t):
        return float((OO.attention(*t, 0.7, *at, causal, mask)["out"] * dout).sum())

    r = OO.attention(q, k, v, lam, 0.7, *at, causal, mask, dout)
    for i, name in enumerate(("dq", "dk", "dv", "dlam")):
        d = torch.randn([q, k, v, lam][i].shape, generator=g).double()
        h = 1e-5
        up, down = ([t + s * d if j == i else t for j, t in enumerate((q, k, v, lam))] for s in (h, -h))
        # central differences: h^2 third derivatives (about 1e-9), cancellation 1e-16 / h
        assert abs((loss(*up) - loss(*down)) / (2 * h) - float((r[name] * d).sum())) < 1e-7
    assert torch.equal(r["out"][r["lse"][0].T == -math.inf],
                       torch.zeros_like(r["out"][r["lse"][0].T == -math.inf]))


def test_the_rows_score_depends_on_differences_of_positions_only():
    """What the rotation is for: q and k turned by their positions give scores
    that a common shift does not change."""
    g = torch.Generator().manual_seed(6)
    q, k = torch.randn(5, 1, 12, generator=g).double(), torch.randn(5, 1, 12, generator=g).double()
    pos = torch.rand(5, 3, generator=g).double()
    axis = torch.arange(6) % 3
    freq = 2 * math.pi * (1 + torch.arange(6) // 3).double()

    def scores(shift):
        t = (pos + shift)[:, axis] * freq
        return OO.turned(q, t, False)[0][:, 0] @ OO.turned(k, t, False)[0][:, 0].T

    assert (scores(torch.zeros(3)) - scores(torch.tensor([0.3, -1.7, 4.0]))).abs().max() < 1e-12
