"""Refusals of the FP8 entry points before any device use (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from lightreason_b200 import build, fp8, native

E4M3 = torch.float8_e4m3fn
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def so():
    build.build()
    return native.lib()


def refused(so, rc, text):
    assert rc == native.MOE_EINVAL
    assert text.encode() in so.moe_last_error(), so.moe_last_error()


def test_rows_refusals(so):
    ok = P(1 << 20)

    def call(x=ok, xs=256, res=None, rs=256, w=ok, eps=1e-6, tokens=4, hidden=256, q=ok, s=ok, normed=None, r=None):
        return so.moe_rmsnorm_fp8(x, xs, res, rs, w, 1.0, eps, tokens, hidden, q, s, normed, r, None)

    refused(so, call(hidden=0), "bad tokens")
    refused(so, call(tokens=-1), "bad tokens")
    refused(so, call(tokens=2**31 - 1), "bad tokens")
    refused(so, call(hidden=(1 << 20) + 1), "bad tokens")
    refused(so, call(xs=255), "row strides")
    refused(so, call(res=ok, rs=8), "row strides")
    refused(so, call(r=ok), "residual_out without residual")
    refused(so, call(w=None, res=ok), "without a norm weight")
    refused(so, call(w=None, normed=ok), "without a norm weight")
    refused(so, call(q=None), "null tensor")
    refused(so, call(eps=-1.0), "eps")
    refused(so, call(eps=float("nan")), "eps")
    assert call(tokens=0, x=None, q=None, s=None) == native.MOE_OK


def test_blocks_refusals(so):
    ok = P(1 << 20)
    refused(so, so.moe_quantize_fp8_blocks(ok, 1, 0, 4, ok, ok, None), "bad shape")
    refused(so, so.moe_quantize_fp8_blocks(ok, -1, 4, 4, ok, ok, None), "bad shape")
    refused(so, so.moe_quantize_fp8_blocks(ok, 1, 2**31 - 1, 4, ok, ok, None), "bad shape")
    refused(so, so.moe_quantize_fp8_blocks(ok, 1, 4, 2**31 - 1, ok, ok, None), "bad shape")
    refused(so, so.moe_quantize_fp8_blocks(None, 1, 4, 4, ok, ok, None), "null tensor")
    refused(so, so.moe_quantize_fp8_blocks(ok, 1 << 30, 1024, 1024, ok, ok, None), "too many blocks")
    assert so.moe_quantize_fp8_blocks(None, 0, 4, 4, None, None, None) == native.MOE_OK


def test_linear_refusals(so):
    ok, bad = P(1 << 20), P((1 << 20) + 8)

    def call(x=ok, w=ok, tokens=3, rows=64, cols=256, out=ok, f32=0):
        return so.moe_linear_fp8(x, ok, w, ok, tokens, rows, cols, out, f32, None, None)

    refused(so, call(cols=24), "multiple of 16")
    refused(so, call(cols=0), "multiple of 16")
    refused(so, call(rows=0), "bad tokens")
    refused(so, call(tokens=-1), "bad tokens")
    refused(so, call(f32=2), "out_f32")
    refused(so, call(x=None), "null tensor")
    for k in ("x", "w", "out"):
        refused(so, call(**{k: bad}), "16-byte aligned")
    # past 2^30, where a size rounded up to a tile no longer fits 32 bits
    refused(so, call(tokens=2**31 - 1), "bad tokens")
    refused(so, call(rows=2**31 - 1), "bad tokens")
    refused(so, call(cols=2**31 - 16), "multiple of 16")
    assert call(tokens=0, x=None, out=None) == native.MOE_OK


def test_experts_refusals(so):
    ok, bad = P(1 << 20), P((1 << 20) + 8)
    need = so.moe_experts_fp8_workspace_bytes(3, 8, 2, 256, 128)
    assert need > 0

    def call(x=ok, gu=ok, dn=ok, idx=ok, tokens=3, experts=8, top_k=2, hidden=256, inner=128, out=ok, work=ok,
             nbytes=need):
        return so.moe_experts_fp8(x, ok, gu, ok, dn, ok, idx, ok, tokens, experts, top_k, hidden, inner, out, work,
                                  nbytes, None, None)

    refused(so, call(hidden=250), "hidden")
    refused(so, call(inner=192), "inner")
    refused(so, call(top_k=0), "top_k")
    refused(so, call(top_k=33), "top_k")
    refused(so, call(experts=0), "experts")
    refused(so, call(experts=1025), "experts")
    refused(so, call(tokens=-1), "tokens")
    refused(so, call(tokens=1 << 29, top_k=8), "too many routes")
    refused(so, call(idx=None), "null tensor")
    for k in ("x", "gu", "dn", "out"):
        refused(so, call(**{k: bad}), "16-byte aligned")
    refused(so, call(nbytes=need - 1), "workspace")
    refused(so, call(work=None), "workspace")
    refused(so, call(work=bad), "workspace")
    assert call(tokens=0, x=None, idx=None, out=None, work=None, nbytes=0) == native.MOE_OK
    assert so.moe_experts_fp8_workspace_bytes(3, 8, 2, 250, 128) == 0


def test_python_refuses_cpu_tensors_and_wrong_types():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 256).to(E4M3), torch.zeros(4, 2)
    w, ws = torch.zeros(128, 256).to(E4M3), torch.zeros(1, 2)
    for call in (lambda: fp8.quantize_rows(x), lambda: fp8.rmsnorm_quantize(x, x[0]), lambda: fp8.quantize_blocks(x),
                 lambda: fp8.linear(q, s, w, ws),
                 lambda: fp8.experts(q, s, w[None], ws[None], w[None], ws[None], torch.zeros(4, 1).long(),
                                     torch.zeros(4, 1).bfloat16())):
        with pytest.raises(ValueError):
            call()


def test_patch_refuses_widths_without_kernels():
    """A model whose widths the FP8 kernels do not take is refused when it is
    patched, not when it runs."""
    from lightreason_b200 import expert_stream
    from transformers.models.qwen3_5_moe.configuration_qwen3_5_moe import Qwen3_5MoeTextConfig
    from transformers.models.qwen3_5_moe.modeling_qwen3_5_moe import Qwen3_5MoeExperts

    config = Qwen3_5MoeTextConfig(hidden_size=256, moe_intermediate_size=192, num_experts=4, num_experts_per_tok=2)
    config._experts_implementation = "eager"
    experts = Qwen3_5MoeExperts(config).to(torch.bfloat16).eval().requires_grad_(False)
    pool = expert_stream.ExpertPool("cuda:0")
    with pytest.raises(ValueError, match="inner of 128"):
        expert_stream._Layer("e", experts, pool, "b200-fp8")
    with pytest.raises(ValueError, match="inner of 128"):
        fp8.check_widths(256, 192)


def test_widths_and_numbers_of_experts():
    fp8.check_widths(16, 128)
    fp8.check_widths(65536, 16384, 1024)
    for bad in ((65552, 128, 4), (256, 16512, 4), (256, 128, 1025), (0, 128, 4)):
        with pytest.raises(ValueError, match="1024 experts"):
            fp8.check_widths(*bad)


def test_banks_follow_their_sources(monkeypatch):
    """ExpertBanks.holds: the tensors last loaded, unchanged; load writes into
    the memory that the banks already have."""
    quantised = []

    def fake(w, out):
        quantised.append(tuple(w.shape))
        out[0].copy_(w.to(E4M3))
        out[1].fill_(float(w.flatten()[0]))

    monkeypatch.setattr(fp8, "quantize_blocks", fake)
    gu, dn = (torch.full(s, 1.0, dtype=torch.bfloat16) for s in ((20, 256, 64), (20, 64, 128)))
    shared = [torch.full(s, 2.0, dtype=torch.bfloat16) for s in ((128, 64), (128, 64), (64, 128))]
    router = torch.full((20, 64), 3.0, dtype=torch.bfloat16)
    banks = fp8.ExpertBanks(gu, dn, "cpu", shared=shared, extra=(router,))
    assert quantised == [(16, 256, 64), (4, 256, 64), (16, 64, 128), (4, 64, 128), (1, 256, 64), (1, 64, 128)]
    assert banks.gate_up.shape == (21, 256, 64) and banks.down_scales.shape == (21, 1, 1)
    sources = [gu, dn, *shared, router]
    assert banks.holds(*sources) and not banks.holds(gu, dn) and not banks.holds(gu.clone(), dn, *shared, router)
    places = [t.data_ptr() for t in (banks.gate_up, banks.down_scales, banks.extra[0])]
    for t in sources:
        t.mul_(2)
        assert not banks.holds(*sources)
        banks.load(gu, dn, shared=shared, extra=(router,))
        assert banks.holds(*sources)
    assert places == [t.data_ptr() for t in (banks.gate_up, banks.down_scales, banks.extra[0])]
    assert banks.extra[0].eq(6).all() and banks.down_scales[:20].eq(2).all() and banks.down_scales[20:].eq(4).all()
    with pytest.raises(ValueError, match="banks' shapes"):
        banks.load(gu, dn)
    with pytest.raises(ValueError, match="1024 experts"):
        fp8.ExpertBanks(torch.zeros(1024, 256, 16, dtype=torch.bfloat16), torch.zeros(1024, 16, 128,
                        dtype=torch.bfloat16), "cpu", shared=[torch.zeros(1)] * 3)
