import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

GOLDEN = os.path.join(ROOT, "tests", "golden")

# rtol=1e-3 / atol=1e-4 in fp32
RTOL, ATOL = 1e-3, 1e-4


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")


def pytest_collection_modifyitems(items):
    """An empty /root/reference is as good as none: the test that imports a module of the reference's says so itself only where the folder is missing.
    And a test of refusals that hands the residual norm's forward made-up addresses which nothing refuses is kept from machines that would read them."""
    if os.path.isdir("/root/reference") and not os.listdir("/root/reference"):
        for item in items:
            if item.name == "test_vendored_class_schedule_tables_and_helpers_match_the_reference":
                item.add_marker(pytest.mark.skip(reason="reference not present"))
    if torch.cuda.device_count() > 0:
        for item in items:
            if item.nodeid.endswith("test_gpu_residual_norm.py::test_library_refuses_what_its_kernels_do_not_take"):
                item.add_marker(pytest.mark.skip(reason="launches a kernel on made-up addresses where a GPU is there"))


sys.path.insert(0, GOLDEN)
import compact  # noqa: E402  (tests/golden/compact.py: which arrays are stored whole, which as samples, the shared DeltaBlock weights)


def load_golden(name):
    """name -> tensor, or a `compact.Sampled` comparison target (assert_close / err_stats compare its stored positions)."""
    return compact.load(os.path.join(GOLDEN, name))


def assert_close(got, want, rtol=RTOL, atol=ATOL, what=""):
    if isinstance(want, compact.Sampled):     # a reference tensor of which one element in 16 is stored: compare those positions
        got, want, what = want.take(got.detach().float().cpu()), want.values, what + " [1/16 sample]"
    got, want = got.detach().float().cpu(), want.detach().float().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} vs {tuple(want.shape)}"
    err = (got - want).abs()
    bad = err > (atol + rtol * want.abs())
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{bad.numel()} outside rtol={rtol} atol={atol}; "
                           f"max abs err {float(err.max()):.3e}, mean {float(err.mean()):.3e}, "
                           f"ref absmax {float(want.abs().max()):.3e}")


@pytest.fixture(scope="session")
def golden_small():
    return load_golden("ddpm_small.npz")


@pytest.fixture(scope="session")
def golden_celeba():
    return load_golden("ddpm_celeba.npz")
