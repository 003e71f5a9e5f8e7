"""What the FP8 entry points promise beside their results (CPU only)."""

from __future__ import annotations

import pytest
import torch

from lightreason_b200 import build, fp8, native

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def so():
    build.build()
    return native.lib()


def test_wait_limit_is_two_seconds_and_settable(so):
    assert so.moe_fp8_wait_limit(5) == 2_000_000_000
    assert so.moe_fp8_wait_limit(2_000_000_000) == 5
