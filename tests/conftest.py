import os
import sys

import pytest
import torch  # noqa: F401 -- before libmtpx.so, so that both use torch's HIP runtime (mtpx.ops)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
for p in (os.path.join(ROOT, "imr-mlp_amd"), os.path.join(ROOT, "oracle"), ROOT):
    if p not in sys.path:
        sys.path.insert(0, p)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs the HIP library)")


@pytest.fixture(scope="session")
def workdir(tmp_path_factory):
    return str(tmp_path_factory.mktemp("mtpx"))


@pytest.fixture(scope="session")
def ctx():
    from mtpx import capi
    c = capi.Context(0)
    yield c
    c.close()
