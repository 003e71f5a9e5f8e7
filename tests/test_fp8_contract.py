"""What the FP8 entry points promise beside their results (CPU only)."""

from __future__ import annotations

from types import SimpleNamespace

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


def fake_layer():
    module = SimpleNamespace(num_experts=2, hidden_dim=64, intermediate_dim=128)
    return SimpleNamespace(module=module, residency="b200-fp8", gate_up=torch.zeros(2, 256, 64, dtype=torch.bfloat16),
                           down=torch.zeros(2, 64, 128, dtype=torch.bfloat16))


def test_captured_calls_go_with_the_banks_they_read(monkeypatch):
    """A graph captured on banks that are gone must not be replayed: clear()
    drops the captured calls, and so does making banks anew under their key."""
    from lightreason_b200 import expert_stream

    def banks(gate_up, down, device, **_):
        return SimpleNamespace(experts=2, hidden=64, inner=128, nbytes=lambda: 5, release=lambda: None,
                               holds=lambda *sources: True)

    monkeypatch.setattr(fp8, "ExpertBanks", banks)
    pool, layer = expert_stream.ExpertPool("cuda:0"), fake_layer()
    key, other = (id(layer.module), "b200-fp8", 1, 8), (id(layer.module), "b200", 1, 8)
    first = pool._fp8_banks(layer)
    pool.replay_graphs = {key: "captured", other: "captured"}
    assert pool._fp8_banks(layer) is first and set(pool.replay_graphs) == {key, other}
    pool._layers.clear()
    assert pool._fp8_banks(layer) is not first and set(pool.replay_graphs) == {other}
    pool.replay_graphs[key] = "captured"
    pool.clear()
    assert pool.replay_graphs == {} and pool.stats.resident_bytes == 0
