"""What the FP8 entry points promise beside their results (CPU only)."""

from __future__ import annotations

import ctypes
import re
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


@pytest.fixture
def quantised(monkeypatch):
    """quantize_blocks on the CPU (values alone); the list of its calls' shapes, and one to fail at."""
    calls = SimpleNamespace(shapes=[], fail_at=None)

    def fake(w, out):
        if len(calls.shapes) == calls.fail_at:
            raise RuntimeError("out of memory")
        calls.shapes.append(tuple(w.shape))
        out[0].copy_(w.to(E4M3))
        out[1].fill_(float(w.flatten()[0]))

    monkeypatch.setattr(fp8, "quantize_blocks", fake)
    return calls


def bank_weights(value=1.0):
    """Experts' gate_up and down, a shared expert, a router."""
    full = lambda *s: torch.full(s, value, dtype=torch.bfloat16)  # noqa: E731
    return full(20, 256, 64), full(20, 64, 128), [full(128, 64), full(128, 64), full(64, 128)], full(20, 64)


def test_banks_half_loaded_hold_nothing(quantised):
    """A load that fails on its way leaves banks that hold no weights, those
    of before the call neither."""
    gu, dn, shared, router = bank_weights()
    banks = fp8.ExpertBanks(gu, dn, "cpu", shared=shared, extra=(router,))
    assert banks.holds(gu, dn, *shared, router)
    other = bank_weights(2.0)
    for at in range(6):
        quantised.shapes.clear()
        quantised.fail_at = at
        with pytest.raises(RuntimeError, match="out of memory"):
            banks.load(*other[:2], shared=other[2], extra=(other[3],))
        assert not banks.holds(gu, dn, *shared, router) and not banks.holds(*other[:2], *other[2], other[3])
        quantised.fail_at = None
        banks.load(gu, dn, shared=shared, extra=(router,))
        assert banks.holds(gu, dn, *shared, router)


def test_banks_check_every_shape_before_they_write(quantised):
    gu, dn, shared, router = bank_weights()
    banks = fp8.ExpertBanks(gu, dn, "cpu", shared=shared, extra=(router,))
    quantised.shapes.clear()
    gu2, dn2, shared2, router2 = bank_weights(2.0)
    for wrong in ([shared2[0], shared2[1][:64], shared2[2]], [*shared2[:2], shared2[2][:, :64]], shared2[:2]):
        with pytest.raises(ValueError, match="widths"):
            banks.load(gu2, dn2, shared=wrong, extra=(router2,))
    for extra in ((router2[:1],), (router2, router2), ()):
        with pytest.raises(ValueError, match="shapes"):
            banks.load(gu2, dn2, shared=shared2, extra=extra)
    assert quantised.shapes == [] and banks.extra[0].eq(1).all() and banks.holds(gu, dn, *shared, router)


@pytest.mark.parametrize("first,then", [(torch.inference_mode, torch.no_grad), (torch.no_grad, torch.inference_mode)])
def test_banks_made_and_loaded_in_either_mode(quantised, first, then):
    """Banks made in inference mode are loaded again outside it, and the other way round."""
    gu, dn, shared, router = bank_weights()
    with first():
        banks = fp8.ExpertBanks(gu, dn, "cpu", shared=shared, extra=(router,))
    router.mul_(3)
    with then():
        assert not banks.holds(gu, dn, *shared, router)
        banks.load(gu, dn, shared=shared, extra=(router,))
        assert banks.holds(gu, dn, *shared, router) and banks.extra[0].eq(3).all()


@pytest.mark.parametrize("experts,top_k,hidden,inner", [(256, 8, 2048, 512), (256, 1, 2048, 512), (8, 2, 16, 16384),
                                                        (64, 12, 272, 128), (1024, 32, 4096, 1024), (3, 5, 65536, 128)])
def test_experts_workspace_does_for_fewer_tokens(so, experts, top_k, hidden, inner):
    """A caller that sizes the workspace once, for its largest batch, has enough
    for every smaller one: across 12 and 13 routes, 2048 and 2049."""
    need = lambda t: so.moe_experts_fp8_workspace_bytes(t, experts, top_k, hidden, inner)  # noqa: E731
    edges = {r // top_k + d for r in (12, 2048) for d in (-1, 0, 1, 2)}
    counts = sorted({t for t in (*range(1, 30), *range(30, 5000, 61), *edges) if t > 0})
    sizes = [need(t) for t in counts]
    assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))
    P = ctypes.c_void_p(1 << 20)
    for t in counts:  # what each call itself asks for (none gets past that: the pointers are not memory)
        rc = so.moe_experts_fp8(P, P, P, P, P, P, P, P, t, experts, top_k, hidden, inner, P, P, 0, None, None)
        asked = re.search(rb"workspace of (\d+) bytes", so.moe_last_error())
        assert rc == native.MOE_EINVAL and 0 < int(asked[1]) <= need(t) <= sizes[-1], t


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    x = torch.ones(4)
    with fwd.dual_level():
        dual = fwd.make_dual(x, x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
            fp8._no_grad(None, x, dual)
        fp8._no_grad(None, x, fwd.unpack_dual(dual).primal)


def test_banks_of_another_kind_under_the_same_key_are_made_anew(quantised):
    """A key is a module's id, which a later module may get: experts alone where
    a block was, a block where experts were, another number of experts."""
    from lightreason_b200 import expert_stream

    pool = expert_stream.ExpertPool("cuda:0")
    pool.device = torch.device("cpu")
    gu, dn, shared, router = bank_weights()
    module = SimpleNamespace(num_experts=20, hidden_dim=64, intermediate_dim=128)
    layer = lambda a, b: SimpleNamespace(module=module, residency="b200-fp8", gate_up=a, down=b)  # noqa: E731
    alone = pool._fp8_banks(layer(gu, dn))
    assert pool._fp8_banks(layer(gu, dn)) is alone and pool.stats.resident_bytes == alone.nbytes()
    pool.replay_graphs = {(id(module), "b200-fp8", 1, 8): "captured"}
    block = pool._fp8_banks(layer(gu, dn), shared=tuple(shared), extra=(router,))
    assert block is not alone and block.holds(gu, dn, *shared, router) and pool.replay_graphs == {}
    assert pool._fp8_banks(layer(gu * 2, dn), shared=tuple(shared), extra=(router,)) is block
    module.num_experts = 8
    fewer = pool._fp8_banks(layer(gu[:8].clone(), dn[:8].clone()))
    assert fewer.experts == 8 and pool.stats.resident_bytes == fewer.nbytes()


def test_block_patch_refuses_more_routes_than_the_experts_take():
    """The shared expert is one route more: 32 routes a token are refused when
    the block is patched, not at each call."""
    from lightreason_b200 import expert_stream, moe_block
    from transformers.models.qwen3_5_moe.configuration_qwen3_5_moe import Qwen3_5MoeTextConfig
    from transformers.models.qwen3_5_moe.modeling_qwen3_5_moe import Qwen3_5MoeSparseMoeBlock

    def block(top_k):
        config = Qwen3_5MoeTextConfig(hidden_size=64, moe_intermediate_size=128, shared_expert_intermediate_size=128,
                                      num_experts=40, num_experts_per_tok=top_k)
        config._experts_implementation = "eager"
        return Qwen3_5MoeSparseMoeBlock(config).to(torch.bfloat16).eval().requires_grad_(False)

    pool = expert_stream.ExpertPool("cuda:0")
    assert moe_block._Block("b", block(31), pool, "b200-fp8").top_k == 31
    with pytest.raises(ValueError, match="31 routes a token"):
        moe_block._Block("b", block(32), pool, "b200-fp8")
    assert moe_block._Block("b", block(32), pool, "b200").top_k == 32


def test_resident_bytes_when_new_banks_fail(quantised):
    """Banks that had to go are counted out once, however often making the new ones fails."""
    from lightreason_b200 import expert_stream

    pool = expert_stream.ExpertPool("cuda:0")
    pool.device = torch.device("cpu")
    gu, dn, shared, router = bank_weights()
    module = SimpleNamespace(num_experts=20, hidden_dim=64, intermediate_dim=128)
    layer = SimpleNamespace(module=module, residency="b200-fp8", gate_up=gu, down=dn)
    pool._fp8_banks(layer)
    quantised.fail_at = len(quantised.shapes)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="out of memory"):
            pool._fp8_banks(layer, shared=tuple(shared), extra=(router,))
        assert pool.stats.resident_bytes == 0
    quantised.fail_at = None
    assert pool._fp8_banks(layer).nbytes() == pool.stats.resident_bytes


def test_pointers_off_their_elements_are_refused(so):
    """An address that the kernels' loads and stores cannot take is an argument
    error, not a fault on the device."""
    P = ctypes.c_void_p
    ok, odd, half, four = P(1 << 20), P((1 << 20) + 1), P((1 << 20) + 2), P((1 << 20) + 4)

    def refused(rc):
        assert rc == native.MOE_EINVAL and b"aligned" in so.moe_last_error(), so.moe_last_error()

    rows = dict(x=ok, res=ok, w=ok, q=ok, s=ok, normed=ok, total=ok)
    for name, bad in (("x", odd), ("res", odd), ("w", odd), ("s", half), ("normed", odd), ("total", odd)):
        a = {**rows, name: bad}
        refused(so.moe_rmsnorm_fp8(a["x"], 64, a["res"], 64, a["w"], 1.0, 1e-6, 2, 64, a["q"], a["s"], a["normed"],
                                   a["total"], None))
    refused(so.moe_quantize_fp8_blocks(odd, 1, 4, 4, ok, ok, None))
    refused(so.moe_quantize_fp8_blocks(ok, 1, 4, 4, ok, half, None))
    for bad in (dict(xs=half), dict(ws=half), dict(status=half)):
        a = {"xs": ok, "ws": ok, "status": None, **bad}
        refused(so.moe_linear_fp8(ok, a["xs"], ok, a["ws"], 2, 64, 64, ok, 0, a["status"], None))
    for bad in (dict(xs=half), dict(gus=half), dict(dns=half), dict(idx=four), dict(wt=odd), dict(status=half)):
        a = {"xs": ok, "gus": ok, "dns": ok, "idx": ok, "wt": ok, "status": None, **bad}
        refused(so.moe_experts_fp8(ok, a["xs"], ok, a["gus"], ok, a["dns"], a["idx"], a["wt"], 2, 4, 2, 64, 128, ok, ok,
                                   1 << 24, a["status"], None))


# ---------------------------------------------------------------- the build ---

@pytest.fixture
def scratch(monkeypatch, tmp_path):
    """A build of one source file into a folder of its own."""
    monkeypatch.setattr(build, "OUT_DIR", tmp_path)
    monkeypatch.setattr(build, "LIB", tmp_path / build.LIB.name)
    monkeypatch.setattr(build, "BIND", tmp_path / build.BIND.name)
    monkeypatch.setattr(build, "SOURCES", ["host.cu"])
    return tmp_path


@pytest.mark.parametrize("compiler", ["false", "/nowhere/c++"])
def test_the_library_is_built_where_the_python_module_cannot_be(scratch, monkeypatch, capfd, compiler):
    """Without a host compiler (or headers), the C library is there and the FP8
    entry points of Python say what is missing."""
    monkeypatch.setenv("CXX", compiler)
    assert build.build() == scratch / "libmoe_b200.so" and build.LIB.exists() and not build.BIND.exists()
    assert "not built" in capfd.readouterr().err
    ctypes.CDLL(str(build.LIB)).moe_version()
    with pytest.raises(RuntimeError, match="missing: build it"):
        fp8._bind.__wrapped__()


def test_the_python_module_belongs_to_one_torch(scratch):
    """A module built against another torch is not this one's."""
    assert torch.__version__ in build.BIND.name
    build.LIB.touch()
    other = scratch / build.BIND.name.replace(torch.__version__, "1.0.0")
    other.touch()
    assert build._bind_stale() and not build._lib_stale()
    build.BIND.touch()
    assert not build._bind_stale()
