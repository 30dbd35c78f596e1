"""No entry point makes a launch of 2^32 work-items or more: the runtime would start what is left of the number, without an
error, and bounds would be missing.  The calls are refused on the host; no device call is made."""

import pytest
import torch

from boundflow_amd import _lib


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built (run python -m boundflow_amd.build)")
    return _lib.load()


N = (1 << 32) - 255     # elements: 2^24 workgroups of 256


@pytest.mark.parametrize("name,call", [
    ("interval_relu", lambda lib, p: lib.bf_interval_relu(p, p, N, p, p, None)),
    ("interval_add", lambda lib, p: lib.bf_interval_add(p, p, p, p, N, p, p, None)),
    ("interval_mul", lambda lib, p: lib.bf_interval_mul(p, p, p, p, N, p, p, None)),
    ("center_radius", lambda lib, p: lib.bf_interval_center_radius(p, p, N, 0, p, p, None)),
    ("scale_rows", lambda lib, p: lib.bf_scale_rows(p, 1 << 20, 1 << 12, p, None)),
    ("rows_add", lambda lib, p: lib.bf_rows_add(p, p, 1 << 20, 1 << 12, 1, None, None, 0, p, None)),
    ("masked_copy_rows", lambda lib, p: lib.bf_masked_copy_rows(p, p, 1 << 20, 1 << 12, p, None))])
def test_too_large_a_launch_is_refused(lib, name, call):
    some = torch.zeros(64)
    assert call(lib, some.data_ptr()) == 3, lib.bf_last_error()
    assert b"2^32 work-items" in lib.bf_last_error()
