"""The FP8 operators on the GPU against 64-bit forms (tests/fp8_reference.py),
elementwise, at the sizes, strides, routes and values where they can go wrong."""

from __future__ import annotations

import pytest
import torch

from lightreason_b200 import build, fp8, native
from tests import fp8_reference as R

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def dev():
    build.build()
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    native.device_check(0)
    return torch.device("cuda", 0)


def gen(seed, dev):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=g.device)


def same_e4m3(q, want, what):
    """Equal as values (+0 and -0 alike)."""
    bad = q.double() != want
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} e4m3 values differ"


def within(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), f"{what}: non-finite values"
    bad = err > bound
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside their bound; worst "
                           f"{float((err / bound.clamp(min=1e-300)).max()):.2f} x")


# -------------------------------------------------------------------- rows ---

ROW_SHAPES = [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (1, 2048), (4, 2048), (333, 1000), (2, 1001), (300, 256),
              (700, 512), (200, 4096), (3, 8192), (2, 16384), (2, 16392), (1, 40000)]


@pytest.mark.parametrize("tokens,hidden", ROW_SHAPES)
def test_quantize_rows_is_the_exact_rounding(dev, tokens, hidden):
    """For BF16 input every e4m3 value is the nearest one with ties to even,
    and the scale is the FP32 value nearest to the quotient."""
    g = gen(tokens * 7919 + hidden, dev)
    x = (randn(g, tokens, hidden) * torch.exp(2 * randn(g, hidden))).to(torch.bfloat16)
    q, s = fp8.quantize_rows(x)
    _, want, scale = R.rows(x.double())
    same_e4m3(q, want, "q")
    assert torch.equal(s, scale.float()) and s.shape == (tokens, R.groups(hidden))


def test_quantize_rows_ties_zeros_and_extremes(dev):
    """Every BF16 magnitude against maxima of several exponents and mantissas:
    zero rows, subnormals, the largest finite values, ties."""
    every = torch.arange(0, 0x7F80, dtype=torch.int32, device=dev).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(0x7F80 // 64 + 1, 128, dtype=torch.bfloat16, device=dev)
    n = every.numel() // 64 * 64
    x[:n // 64, :64] = every[:n].view(-1, 64)
    x[:n // 64, 64:] = -every[:n].view(-1, 64)
    # and against fixed maxima: all mantissas of one binade
    top = torch.arange(0x3F80, 0x4000, dtype=torch.int32, device=dev).to(torch.int16).view(torch.bfloat16)
    y = every[0x3000:0x3F80].view(-1, 31).repeat_interleave(8, 0)[:, :31]
    z = torch.zeros(y.shape[0] * 4, 128, dtype=torch.bfloat16, device=dev)
    z[:, :31] = y.repeat(4, 1)
    z[:, 127] = top[torch.arange(z.shape[0], device=dev) % 128]
    for v in (x, z):
        q, s = fp8.quantize_rows(v)
        _, want, scale = R.rows(v.double())
        same_e4m3(q, want, "q")
        assert torch.equal(s, scale.float())


def test_quantize_rows_strided_and_unaligned(dev):
    """Rows of a wider tensor, starting anywhere: vector and scalar paths."""
    g = gen(3, dev)
    wide = randn(g, 40, 700).to(torch.bfloat16)
    for first, hidden in ((0, 512), (8, 512), (3, 512), (1, 300), (16, 320)):
        x = wide[:, first:first + hidden]
        q, s = fp8.quantize_rows(x)
        qc, sc = fp8.quantize_rows(x.contiguous())
        assert torch.equal(q.view(torch.uint8), qc.view(torch.uint8)) and torch.equal(s, sc)
    x = wide[::3, :512]
    assert torch.equal(fp8.quantize_rows(x)[0].view(torch.uint8),
                       fp8.quantize_rows(x.contiguous())[0].view(torch.uint8))


def norm_reference(x, weight, residual, eps, offset):
    r = (x.double() + residual.double()).to(torch.bfloat16) if residual is not None else x
    rd = r.double()
    y = rd * torch.rsqrt(rd.square().mean(-1, keepdim=True) + eps) * (offset + weight.double())
    return r, y


# FP32 relative error of y: the sum of squares adds at most 8 + 5 + 64 positive
# terms in sequence (a vector's, the warp's, the blocks of a row of 16384; the
# scalar kernel's longest chain is 40000 / 32 / 8 + 13 = 170), halved by the
# square root, plus eight roundings: below 128 of 2^-24; 256 allows twice that
NORM_REL = 256 * R.F32


def check_norm(got, x, weight, residual, eps=1e-6, offset=1.0):
    q, s, normed, total = got
    r, y = norm_reference(x, weight, residual, eps, offset)
    if residual is not None:
        assert torch.equal(total.view(torch.int16), r.view(torch.int16)), "residual_out"
    within(normed, y, (R.BF + NORM_REL) * y.abs() + 2.0 ** -134, "normed")
    a = R.tops(y)
    within(s, a / R.TOP, 2 * NORM_REL * a / R.TOP, "scales")
    v, _, _ = R.rows(y)
    within(q, v, 0.5 * R.step(v) * (1 + 4 * NORM_REL) + 4 * NORM_REL * v.abs(), "q")


@pytest.mark.parametrize("tokens,hidden", ROW_SHAPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_rmsnorm_quantize(dev, tokens, hidden, with_residual):
    g = gen(tokens * 31 + hidden, dev)
    x = (3 * randn(g, tokens, hidden)).to(torch.bfloat16)
    w = (0.5 * randn(g, hidden)).to(torch.bfloat16)
    res = randn(g, tokens, hidden).to(torch.bfloat16) if with_residual else None
    check_norm(fp8.rmsnorm_quantize(x, w, res), x, w, res)
    got = fp8.rmsnorm_quantize(x, w, res, eps=1e-3, weight_offset=0.0)
    check_norm(got, x, w, res, eps=1e-3, offset=0.0)


def test_rmsnorm_quantize_in_place_strided_and_optional(dev):
    """residual_out over residual and normed over x, as a model's residual
    stream does; strided inputs; without the BF16 output."""
    g = gen(11, dev)
    for hidden in (2048, 1001):
        wide = randn(g, 9, 2 * hidden + 16).to(torch.bfloat16)
        x, res = wide[:, 8:8 + hidden], wide[:, hidden + 16:2 * hidden + 16]
        w = randn(g, hidden).to(torch.bfloat16)
        want = fp8.rmsnorm_quantize(x.contiguous(), w, res.contiguous())
        got = fp8.rmsnorm_quantize(x, w, res)
        xc, rc = x.contiguous(), res.contiguous()
        q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
        placed = fp8.rmsnorm_quantize(xc, w, rc, out=(q, s, xc, rc))
        bare = fp8.rmsnorm_quantize(x, w, res, normed=False)
        assert bare[2] is None
        for a in (got, placed):
            for u, v in zip(a, want):
                assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
        assert torch.equal(bare[0].view(torch.uint8), want[0].view(torch.uint8))


def test_rows_with_nan_or_infinity_keep_to_themselves(dev):
    """A group with a NaN or an infinity reads back as NaN; with the norm its
    whole row does; other groups and rows are as without it."""
    g = gen(12, dev)
    for hidden in (512, 515):
        x = randn(g, 6, hidden).to(torch.bfloat16)
        w = randn(g, hidden).to(torch.bfloat16)
        bad = x.clone()
        bad[1, 130], bad[4, 3] = float("nan"), float("inf")
        q0, s0 = fp8.quantize_rows(x)
        q, s = fp8.quantize_rows(bad)
        back, clean = R.widen_rows(q, s), R.widen_rows(q0, s0)
        assert back[1, 128:256].isnan().all() and back[4, :128].isnan().all()
        back[1, 128:256], back[4, :128] = clean[1, 128:256], clean[4, :128]
        assert torch.equal(back, clean)
        q0, s0, y0, _ = fp8.rmsnorm_quantize(x, w)
        q, s, y, _ = fp8.rmsnorm_quantize(bad, w)
        assert R.widen_rows(q, s)[1].isnan().all() and y[1].isnan().all()
        # r / inf is 0 for the finite values of a row with an infinity, NaN at it
        assert y[4, 3].isnan() and R.widen_rows(q, s)[4, :128].isnan().all()
        keep = [0, 2, 3, 5]
        assert torch.equal(y[keep], y0[keep]) and torch.equal(s[keep], s0[keep])
        assert torch.equal(q[keep].view(torch.uint8), q0[keep].view(torch.uint8))


def test_rows_past_32_bit_offsets(dev):
    """More than 2^31 values: the last rows come out as they do alone."""
    tokens, hidden = (1 << 31) // 2048 + 5, 2048
    x = torch.zeros(tokens, hidden, dtype=torch.bfloat16, device=dev)
    x[-3:] = randn(gen(5, dev), 3, hidden).to(torch.bfloat16)
    w = torch.zeros(hidden, dtype=torch.bfloat16, device=dev)
    q, s = fp8.quantize_rows(x)
    qa, sa = fp8.quantize_rows(x[-3:].clone())
    assert torch.equal(q[-3:].view(torch.uint8), qa.view(torch.uint8)) and torch.equal(s[-3:], sa)
    q, s, y, _ = fp8.rmsnorm_quantize(x, w)
    qa, sa, ya, _ = fp8.rmsnorm_quantize(x[-3:].clone(), w)
    assert torch.equal(q[-3:].float(), qa.float()) and torch.equal(y[-3:], ya)
    del x, q, s, y
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ blocks ---

@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (1000, 2000), (64, 72), (3, 260, 392), (2, 257, 100),
                                   (5, 1, 3), (4, 256, 512)])
def test_quantize_blocks_is_the_exact_rounding(dev, shape):
    g = gen(sum(shape), dev)
    w = (0.02 * randn(g, *shape)).to(torch.bfloat16)
    q, s = fp8.quantize_blocks(w)
    want, scale = R.blocks(w.double())
    same_e4m3(q, want, "q")
    assert s.shape == scale.shape and torch.equal(s, scale.float())


def test_quantize_blocks_past_32_bit_offsets(dev):
    w = torch.zeros(1025, 1024, 2048, dtype=torch.bfloat16, device=dev)
    w[-1] = randn(gen(6, dev), 1024, 2048).to(torch.bfloat16)
    q, s = fp8.quantize_blocks(w)
    qa, sa = fp8.quantize_blocks(w[-1].clone())
    assert torch.equal(q[-1].view(torch.uint8), qa.view(torch.uint8)) and torch.equal(s[-1], sa)
    del w, q, s
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ linear ---

def linear_case(dev, tokens, rows, cols, seed=0):
    g = gen(seed + tokens * 131 + rows * 17 + cols, dev)
    x, xs = fp8.quantize_rows(randn(g, tokens, cols).to(torch.bfloat16))
    w, ws = fp8.quantize_blocks((0.05 * randn(g, rows, cols)).to(torch.bfloat16))
    return x, xs, w, ws


LINEAR_SHAPES = [(1, 1, 16), (1, 1024, 2048), (2, 100, 144), (3, 130, 2064), (4, 128, 128), (5, 257, 272),
                 (7, 1000, 1040), (16, 512, 512), (17, 2048, 512), (33, 129, 4096), (64, 1024, 2048), (77, 1000, 1040),
                 (127, 384, 640), (128, 256, 128), (129, 640, 256), (200, 2050, 336), (256, 8192, 256),
                 (300, 72, 1024), (513, 1024, 1168), (1000, 511, 2048), (2048, 2048, 512), (1, 8200, 16),
                 (300, 3, 48), (6, 20000, 128)]

# every row tile with every split over the columns, and widths that end inside a 16-byte unit
LINEAR_SHAPES += [(5, 2500, 7488), (5, 17000, 2064), (50, 2048, 3552), (129, 1000, 2096), (257, 2048, 6192),
                  (65, 2048, 10720), (200, 4097, 2240), (400, 4097, 1056), (257, 4097, 2560), (65, 4097, 3280),
                  (257, 2052, 5120), (3000, 1001, 256), (2500, 2052, 272), (2, 8192, 8192), (4, 512, 8192)]

# CTA pairs: the second CTA of the last pair with all its rows, some, one and none
LINEAR_SHAPES += [(2048, 4096, 1024), (2300, 2304, 400), (2177, 2500, 144), (2100, 4104, 272), (130, 40000, 128),
                  (4500, 257, 2064)]


@pytest.mark.parametrize("tokens,rows,cols", LINEAR_SHAPES)
def test_linear(dev, tokens, rows, cols):
    x, xs, w, ws = linear_case(dev, tokens, rows, cols)
    want, bound = R.linear(x, xs, w, ws)
    within(fp8.linear(x, xs, w, ws, out_dtype=torch.float32), want, bound + R.F32 * want.abs(), "f32")
    within(fp8.linear(x, xs, w, ws), want, bound + R.BF * (want.abs() + bound), "bf16")


@pytest.mark.parametrize("tokens", [1, 4, 40, 300])
def test_linear_rows_and_outside_are_left_alone(dev, tokens):
    """Rows around the output stay as they were; a row with NaN stays alone."""
    x, xs, w, ws = linear_case(dev, tokens, 264, 400)
    store = torch.full((tokens + 2, 264), 7.0, dtype=torch.bfloat16, device=dev)
    fp8.linear(x, xs, w, ws, out=store[1:-1])
    want = fp8.linear(x, xs, w, ws)
    assert torch.equal(store[1:-1], want) and (store[0] == 7).all() and (store[-1] == 7).all()
    xs = xs.clone()
    xs[tokens // 2, 1] = float("nan")
    got = fp8.linear(x, xs, w, ws)
    assert got[tokens // 2].isnan().all()
    keep = torch.arange(tokens, device=dev) != tokens // 2
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,rows", [(2100, 4104), (2100, 4100), (2177, 2501)])
def test_linear_pairs_leave_the_outside_alone(dev, tokens, rows, dtype):
    """CTA pairs whose last rows fill part of one CTA: nothing beyond the output,
    a row with NaN by itself, and the same values call after call."""
    x, xs, w, ws = linear_case(dev, tokens, rows, 400)
    pad = 16  # elements, so that the output stays on a 16-byte boundary
    store = torch.full((tokens * rows + 2 * pad,), 7.0, dtype=dtype, device=dev)
    out = store[pad:-pad].view(tokens, rows)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    fp8.linear(x, xs, w, ws, out=out, status=status)
    want, bound = R.linear(x, xs, w, ws)
    within(out, want, bound + (R.F32 * want.abs() if dtype is torch.float32 else R.BF * (want.abs() + bound)), "out")
    assert store[:pad].eq(7).all() and store[-pad:].eq(7).all() and status.item() == 0
    xs2 = xs.clone()
    xs2[tokens - 1, 1] = float("nan")
    got = fp8.linear(x, xs2, w, ws, out_dtype=dtype)
    assert got[-1].isnan().all() and torch.equal(got[:-1], out[:-1])


def test_linear_is_deterministic(dev):
    for shape in ((64, 1024, 2048), (9, 512, 4096), (700, 1024, 1024)):
        x, xs, w, ws = linear_case(dev, *shape)
        first = fp8.linear(x, xs, w, ws, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(fp8.linear(x, xs, w, ws, out_dtype=torch.float32), first)


# ----------------------------------------------------------------- experts ---

def experts_case(dev, tokens, count, top_k, hidden, inner, seed=0, routes="random"):
    g = gen(seed + tokens * 3 + count * 5 + hidden, dev)
    x, xs = fp8.quantize_rows(randn(g, tokens, hidden).to(torch.bfloat16))
    gu, gus = fp8.quantize_blocks((0.05 * randn(g, count, 2 * inner, hidden)).to(torch.bfloat16))
    dn, dns = fp8.quantize_blocks((0.05 * randn(g, count, hidden, inner)).to(torch.bfloat16))
    if routes == "random":
        idx = torch.rand(tokens, count, generator=g, device=dev).topk(top_k, -1)[1]
    elif routes == "same":        # every route of every token: one expert
        idx = torch.full((tokens, top_k), count - 1, device=dev)
    else:                         # "dropped": ids on every side of the range, whole tokens without a route
        idx = torch.randint(-2, count + 2, (tokens, top_k), generator=g, device=dev)
        idx[::3] = torch.tensor([-1, count, 1 << 40, -(1 << 40)], device=dev)[torch.arange(top_k, device=dev) % 4]
    weights = torch.softmax(randn(g, tokens, top_k), -1).to(torch.bfloat16)
    return x, xs, gu, gus, dn, dns, idx.contiguous(), weights


EXPERT_SHAPES = [(1, 8, 2, 256, 128), (1, 32, 8, 2048, 512), (2, 4, 4, 144, 128), (3, 16, 5, 400, 256),
                 (5, 64, 8, 2048, 512), (16, 32, 8, 1024, 256), (17, 16, 8, 2048, 512), (33, 4, 2, 16, 128),
                 (64, 1, 1, 128, 128), (65, 3, 3, 2064, 384), (130, 8, 2, 272, 256), (300, 6, 4, 1104, 128),
                 (700, 5, 2, 512, 640), (1500, 12, 8, 512, 256), (12, 40, 12, 640, 128), (1, 40, 32, 256, 256),
                 # two passes over the routes of one token; as many experts as there may be; the cluster plan
                 (1, 40, 12, 640, 128), (20, 1024, 8, 128, 128), (260, 64, 8, 256, 256), (1100, 300, 2, 144, 128),
                 # 9 to 25 rows an expert
                 (300, 128, 4, 272, 256), (290, 30, 1, 1040, 128), (100, 32, 8, 512, 384), (1900, 1024, 8, 144, 128)]


@pytest.mark.parametrize("tokens,count,top_k,hidden,inner", EXPERT_SHAPES)
def test_experts(dev, tokens, count, top_k, hidden, inner):
    c = experts_case(dev, tokens, count, top_k, hidden, inner)
    want, bound = R.experts(*c)
    within(fp8.experts(*c), want, bound, "out")


@pytest.mark.parametrize("tokens,count,top_k,hidden,inner", [(1, 4, 8, 256, 128), (7, 4, 6, 272, 256),
                                                             (40, 8, 8, 512, 128), (400, 20, 8, 528, 256)])
@pytest.mark.parametrize("routes", ["same", "dropped"])
def test_experts_skewed_and_dropped_routes(dev, tokens, count, top_k, hidden, inner, routes):
    """All routes on one expert (the same id several times in a token), and
    ids outside the bank, tokens with none left among them: those are zero."""
    c = experts_case(dev, tokens, count, top_k, hidden, inner, routes=routes)
    want, bound = R.experts(*c)
    got = fp8.experts(*c)
    within(got, want, bound, "out")
    if routes == "dropped":
        assert (got[::3] == 0).all()
        nothing = torch.full_like(c[6], -1)
        assert (fp8.experts(*c[:6], nothing, c[7]) == 0).all()


@pytest.mark.parametrize("tokens", [1, 6, 90, 600])
def test_experts_nan_row_keeps_to_itself(dev, tokens):
    c = list(experts_case(dev, tokens, 8, 3, 512, 256))
    store = torch.full((tokens + 2, 512), 7.0, dtype=torch.bfloat16, device=dev)
    want = fp8.experts(*c)
    fp8.experts(*c, out=store[1:-1])
    assert torch.equal(store[1:-1], want) and (store[0] == 7).all() and (store[-1] == 7).all()
    xs = c[1].clone()
    xs[tokens // 2, 0] = float("inf")
    got = fp8.experts(c[0], xs, *c[2:])
    assert not torch.isfinite(got[tokens // 2]).any()
    keep = torch.arange(tokens, device=dev) != tokens // 2
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("tokens", [1, 5, 60, 400])
def test_experts_weights_of_dropped_routes_do_not_matter(dev, tokens):
    """A dropped route's weight may hold anything, NaN too."""
    c = list(experts_case(dev, tokens, 8, 4, 256, 128))
    idx, weights = c[6].clone(), c[7].clone()
    idx[:, 1], idx[:, 3] = -1, 8
    weights[:, 1::2] = 0
    want = fp8.experts(*c[:6], idx, weights)
    weights[:, 1], weights[:, 3] = float("nan"), float("inf")
    assert torch.equal(fp8.experts(*c[:6], idx, weights), want)


def test_experts_and_linear_past_32_bit_rows(dev):
    """Route rows and outputs of more than 2^32 bytes: the last rows against 64 bits."""
    tokens, hidden, inner = 140_000, 2048, 128
    c = experts_case(dev, 64, 8, 8, hidden, inner)
    x, xs = (t.repeat(tokens // 64 + 1, 1)[:tokens].contiguous() for t in c[:2])
    idx, weights = (t.repeat(tokens // 64 + 1, 1)[:tokens].contiguous() for t in c[6:])
    got = fp8.experts(x, xs, *c[2:6], idx, weights)
    want, bound = R.experts(*c)
    last = slice(tokens - 96, tokens)
    at = torch.arange(tokens, device=dev)[last] % 64
    within(got[last], want[at], bound[at], "experts")
    within(got[:64], want, bound, "experts, first")
    del got, x, xs
    rows, cols = 1_100_000, 128
    x, xs, w, ws = linear_case(dev, 64, 2056, cols)
    xl, xsl = (t.repeat(rows // 64 + 1, 1)[:rows].contiguous() for t in (x, xs))
    got = fp8.linear(xl, xsl, w, ws)
    want, bound = R.linear(x, xs, w, ws)
    bound = bound + R.BF * (want.abs() + bound)
    at = torch.arange(rows, device=dev)[rows - 96:] % 64
    within(got[rows - 96:], want[at], bound[at], "linear")
    del got, xl, xsl
    torch.cuda.empty_cache()


def test_experts_bank_past_32_bit_offsets(dev):
    """Banks of more than 2^32 bytes: the last experts as in banks of their own."""
    count, inner, hidden = 700, 1536, 2048
    c = experts_case(dev, 24, 2, 2, hidden, inner)
    gu = torch.zeros(count, 2 * inner, hidden, dtype=torch.uint8, device=dev).view(E4M3)
    dn = torch.zeros(count, hidden, inner, dtype=torch.uint8, device=dev).view(E4M3)
    gus, dns = (torch.zeros(count, *s.shape[1:], device=dev) for s in (c[3], c[5]))
    for big, small in ((gu.view(torch.uint8), c[2].view(torch.uint8)), (gus, c[3]),
                       (dn.view(torch.uint8), c[4].view(torch.uint8)), (dns, c[5])):
        big[-2:] = small
    for tokens in (1, 24):
        x, xs, idx, wt = c[0][:tokens], c[1][:tokens], c[6][:tokens], c[7][:tokens]
        want = fp8.experts(x, xs, c[2], c[3], c[4], c[5], idx, wt)
        got = fp8.experts(x, xs, gu, gus, dn, dns, idx + count - 2, wt)
        assert torch.equal(got, want)
    del gu, dn
    torch.cuda.empty_cache()


# ------------------------------------------------------------ how it is run ---

def test_empty_batch(dev):
    x = torch.empty(0, 256, dtype=torch.bfloat16, device=dev)
    q, s = fp8.quantize_rows(x)
    assert q.shape == (0, 256) and s.shape == (0, 2)
    assert fp8.rmsnorm_quantize(x, torch.zeros(256, dtype=torch.bfloat16, device=dev), x)[3].shape == (0, 256)
    c = experts_case(dev, 2, 4, 2, 256, 128)
    assert fp8.linear(q, s, c[2][0], c[3][0]).shape == (0, 256)
    assert fp8.experts(q, s, *c[2:6], c[6][:0], c[7][:0]).shape == (0, 256)


def chain_of_calls(x, res, w, c):
    """Norm, router-independent linear and experts as a layer would use them."""
    q, s, y, r = fp8.rmsnorm_quantize(x, w, res)
    lin = fp8.linear(q, s, c[2][0], c[3][0])
    return q, s, y, r, lin, fp8.experts(q, s, *c[2:])


@pytest.mark.parametrize("tokens", [1, 48, 400])
def test_streams_and_graphs(dev, tokens):
    """The chain on a side stream, and in two captured graphs that live (and
    replay) together on changing inputs, equals the eager calls."""
    c = experts_case(dev, tokens, 8, 4, 512, 256)
    g = gen(tokens, dev)
    w = randn(g, 512).to(torch.bfloat16)
    ins = [(randn(g, tokens, 512).to(torch.bfloat16), randn(g, tokens, 512).to(torch.bfloat16)) for _ in range(4)]
    want = [chain_of_calls(*i, w, c) for i in ins]
    same = lambda a, b: all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))  # noqa: E731
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        got = [chain_of_calls(*i, w, c) for i in ins]
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(got, want))
    graphs = []
    for k in range(2):
        x, r = ins[k][0].clone(), ins[k][1].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain_of_calls(x, r, w, c)
        graphs.append((graph, x, r, out))
    for first in (0, 2):
        for k, (graph, x, r, _) in enumerate(graphs):
            x.copy_(ins[first + k][0])
            r.copy_(ins[first + k][1])
        s1, s2 = torch.cuda.Stream(dev), torch.cuda.Stream(dev)
        for s, (graph, *_) in zip((s1, s2), graphs):
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for k, (_, _, _, out) in enumerate(graphs):
            assert same(out, want[first + k])


def test_back_to_back_calls_with_new_weights(dev):
    """A product right behind the kernel that writes its weights, again and
    again into the same memory: each sees its own weights."""
    g = gen(77, dev)
    ws = [(0.05 * randn(g, 512, 1024)).to(torch.bfloat16) for _ in range(6)]
    x, xs = fp8.quantize_rows(randn(g, 1, 1024).to(torch.bfloat16))
    want = []
    for w in ws:
        q, s = fp8.quantize_blocks(w)
        torch.cuda.synchronize()
        want.append(fp8.linear(x, xs, q, s))
        torch.cuda.synchronize()
    out = fp8.quantize_blocks(ws[0])
    got = []
    for w in ws:
        fp8.quantize_blocks(w, out=out)
        got.append(fp8.linear(x, xs, *out))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_python_names_the_argument_it_refuses(dev):
    """What the C++ module does not take is named by the Python behind it."""
    c = experts_case(dev, 3, 4, 2, 256, 128)
    x, xs, gu, gus, dn, dns, idx, wt = c
    b = torch.zeros(3, 256, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(256, dtype=torch.bfloat16, device=dev)
    grad = b.clone().requires_grad_()
    cases = [
        (lambda: fp8.quantize_rows(b.float()), ValueError, "x must be a CUDA BF16"),
        (lambda: fp8.quantize_rows(b[:, ::2]), ValueError, "dense rows"),
        (lambda: fp8.quantize_rows(b[:1].expand(3, 256)), ValueError, "dense rows"),
        (lambda: fp8.quantize_rows(b, out=(x, xs[:2])), ValueError, r"out\[1\]"),
        (lambda: fp8.quantize_rows(b, out=(b, xs)), ValueError, r"out\[0\]"),
        (lambda: fp8.quantize_rows(grad), RuntimeError, "no gradient"),
        (lambda: fp8.rmsnorm_quantize(b, w[:128]), ValueError, "weight"),
        (lambda: fp8.rmsnorm_quantize(b, w, b[:2]), ValueError, "residual"),
        (lambda: fp8.rmsnorm_quantize(b, w.cpu()), ValueError, "weight"),
        (lambda: fp8.rmsnorm_quantize(b, w, out=(x, xs, None, b.clone())), ValueError, "without a residual"),
        (lambda: fp8.rmsnorm_quantize(b, w, eps=2.0), ValueError, "eps"),
        (lambda: fp8.rmsnorm_quantize(grad, w), RuntimeError, "no gradient"),
        (lambda: fp8.quantize_blocks(b.t()), ValueError, "w must be"),
        (lambda: fp8.quantize_blocks(grad), RuntimeError, "no gradient"),
        (lambda: fp8.quantize_blocks(b, out=(x, xs)), ValueError, r"out\[1\]"),
        (lambda: fp8.linear(x, xs[:, :1], gu[0], gus[0]), ValueError, "x_scales"),
        (lambda: fp8.linear(x, xs, gu[0], gus[0][:1]), ValueError, "w_scales"),
        (lambda: fp8.linear(x, xs, gu[0], gus[0], out_dtype=torch.float16), ValueError, "out_dtype"),
        (lambda: fp8.linear(x, xs, gu[0], gus[0], out=b[:2]), ValueError, "out"),
        (lambda: fp8.linear(x, xs, gu[0], gus[0], status=idx), ValueError, "status"),
        (lambda: fp8.linear(x, xs.clone().requires_grad_(), gu[0], gus[0]), RuntimeError, "no gradient"),
        (lambda: fp8.experts(x, xs, gu, gus, dn, dns, idx.int(), wt), ValueError, "idx"),
        (lambda: fp8.experts(x, xs, gu, gus, dn, dns, idx, wt.float()), ValueError, "weights"),
        (lambda: fp8.experts(x, xs, gu, gus, dn[:3], dns, idx, wt), ValueError, "down"),
        (lambda: fp8.experts(x, xs, gu, gus, dn, dns[:, :1], idx, wt), ValueError, "down_scales"),
        (lambda: fp8.experts(x, xs, gu, gus, dn, dns, idx, wt, out=b.float()), ValueError, "out"),
        (lambda: fp8.experts(x, xs, gu, gus, dn, dns, idx, wt.clone().requires_grad_()), RuntimeError, "no gradient"),
    ]
    for call, error, text in cases:
        with pytest.raises(error, match=text):
            call()
    with torch.no_grad():  # nothing to be tracked here
        assert fp8.quantize_rows(grad)[0].shape == (3, 256)


def test_tensors_without_memory_raise(dev):
    """A tensor with no data pointer is an exception, and the device and the
    interpreter are as they were."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        fake = torch.empty(4, 256, dtype=torch.bfloat16, device=dev)
    out = (torch.empty(4, 256, dtype=torch.float8_e4m3fn, device=dev), torch.empty(4, 2, device=dev))
    for _ in range(3):
        with pytest.raises(Exception, match="(?i)fake|data pointer|storage"):
            fp8.quantize_rows(fake, out=out)
    assert torch.cuda.current_device() == torch.device(dev).index
    assert fp8.quantize_rows(torch.ones(4, 256, dtype=torch.bfloat16, device=dev), out=out)[1].shape == (4, 2)


@pytest.mark.parametrize("tokens", [1, 48, 400])
def test_calls_from_two_threads_at_once(dev, tokens):
    """The chain from two threads on streams of their own equals the calls one
    after another, and no wait gives up."""
    import threading

    c = experts_case(dev, tokens, 8, 4, 512, 256)
    g = gen(tokens + 1, dev)
    w = randn(g, 512).to(torch.bfloat16)
    ins = [(randn(g, tokens, 512).to(torch.bfloat16), randn(g, tokens, 512).to(torch.bfloat16)) for _ in range(2)]
    want = [chain_of_calls(*i, w, c) for i in ins]
    status = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream(dev)):
                for _ in range(20):
                    got[k] = chain_of_calls(*ins[k], w, c)
                    fp8.experts(*got[k][:2], *c[2:], status=status[k])
                torch.cuda.current_stream(dev).synchronize()
        except Exception as error:  # noqa: BLE001 - shown by the main thread
            errors.append(error)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and status.sum() == 0
    for a, b in zip(got, want):
        assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))


# ------------------------------------------------------------ in a model ---

EXPERTS = 32


@pytest.fixture(scope="module")
def model():
    from tests.dropin_model import make_model

    return make_model(experts=EXPERTS, layers=2)[0]


def states(tokens, dev, seed=0):
    g = gen(seed + tokens, dev)
    x = randn(g, tokens, 2048).to(torch.bfloat16)
    idx = torch.rand(tokens, EXPERTS, generator=g, device=dev).topk(8, -1)[1]
    return x, idx, torch.softmax(randn(g, tokens, 8), -1).to(torch.bfloat16)


def rms_ratio(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# e4m3 rounds a value by 2^-4 of itself at most, uniformly within its step and
# so by 2^-4 / sqrt(3) rms at the worst place of a binade; rows and weights of
# both products are four such independent roundings of the terms that a result
# sums, and SwiGLU multiplies two of the first sums: sqrt(2 + 2 + 2) of them
MODEL_RMS = 6 ** 0.5 * 2.0 ** -4 / 3 ** 0.5


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_patched_experts_fp8(dev, model, tokens):
    """patch_experts(mode="b200-fp8") is the operators on the module's
    quantised banks, and near the BF16 experts."""
    from lightreason_b200 import expert_stream

    pool = expert_stream.ExpertPool(dev)
    args = states(tokens, dev)
    with torch.inference_mode(), expert_stream.patch_experts(model, mode="b200-fp8", pool=pool):
        got = [layer.experts(*args) for layer in model.layers]
        again = model.layers[0].experts(*args)
    assert pool.stats.fp8_layer_calls == 3 and pool.stats.resident_bytes > 0
    assert torch.equal(again, got[0])
    bf16 = expert_stream.ExpertPool(dev)
    with torch.inference_mode(), expert_stream.patch_experts(model, mode="b200", pool=bf16):
        want = [layer.experts(*args) for layer in model.layers]
    for layer, g, w in zip(model.layers, got, want):
        m = layer.experts
        q, s = fp8.quantize_rows(args[0])
        gu, dn = (fp8.quantize_blocks(t.detach().to(dev)) for t in (m.gate_up_proj, m.down_proj))
        assert torch.equal(g, fp8.experts(q, s, *gu, *dn, args[1], args[2]))
        assert rms_ratio(g, w) < MODEL_RMS
    pool.clear()


@pytest.mark.parametrize("tokens", [1, 33])
def test_patched_blocks_fp8(dev, model, tokens):
    """The whole block on FP8 banks against its BF16 chain: same routes, the
    shared expert weighted by its gate."""
    from lightreason_b200 import expert_stream, moe_block

    x = states(tokens, dev, seed=9)[0].reshape(1, tokens, 2048)
    outs = {}
    for mode in ("b200", "b200-fp8"):
        pool = expert_stream.ExpertPool(dev)
        with torch.inference_mode(), moe_block.patch_moe_blocks(model, mode=mode, pool=pool):
            outs[mode] = [b(x) for b in model.layers]
            assert model.layers[0](x[:, :0]).shape == (1, 0, 2048)
        pool.clear()
    for got, want in zip(outs["b200-fp8"], outs["b200"]):
        assert got.shape == want.shape and rms_ratio(got, want) < MODEL_RMS


def test_patched_experts_fp8_replayed(dev, model):
    """Captured graphs per layer and width give the eager calls' values."""
    from lightreason_b200 import expert_stream, scheduled_graph

    pool = expert_stream.ExpertPool(dev)
    with torch.inference_mode(), expert_stream.patch_experts(model, mode="b200-fp8", pool=pool):
        cases = [states(t, dev, seed=s) for t in (1, 5) for s in range(2)]
        want = [[layer.experts(*c) for layer in model.layers] for c in cases]
        with scheduled_graph.replay_experts(pool):
            got = [[layer.experts(*c).clone() for layer in model.layers] for c in cases]
        scheduled_graph.release_graphs(pool)
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    pool.clear()


def test_patched_experts_and_blocks_follow_changed_weights(dev):
    """Weights changed in place between calls: the next call, eager or replayed,
    is that of banks made from the new ones."""
    from lightreason_b200 import expert_stream, moe_block, scheduled_graph
    from tests.dropin_model import make_model

    model = make_model(experts=16, layers=1, seed=41)[0]
    layer = model.layers[0]
    g = gen(3, dev)
    x, weights = randn(g, 3, 2048).to(torch.bfloat16), torch.softmax(randn(g, 3, 8), -1).to(torch.bfloat16)
    idx = torch.rand(3, 16, generator=g, device=dev).topk(8, -1)[1]

    def change():
        with torch.no_grad():
            layer.experts.gate_up_proj[5].mul_(-1.5)
            layer.experts.down_proj.mul_(0.7)
            layer.gate.weight.copy_(layer.gate.weight.flip(0).clone())
            layer.shared_expert.up_proj.weight.mul_(3)

    def fresh(block):
        pool = expert_stream.ExpertPool(dev)
        with (moe_block.patch_moe_blocks if block else expert_stream.patch_experts)(model, mode="b200-fp8", pool=pool):
            return layer(x[None]) if block else layer.experts(x, idx, weights)

    with torch.no_grad():
        pool = expert_stream.ExpertPool(dev)
        with expert_stream.patch_experts(model, mode="b200-fp8", pool=pool), scheduled_graph.replay_experts(pool):
            first = layer.experts(x, idx, weights).clone()
            resident = pool.stats.resident_bytes
            change()
            second = layer.experts(x, idx, weights).clone()
            assert pool.stats.resident_bytes == resident
        scheduled_graph.release_graphs(pool)
        assert not torch.equal(first, second) and torch.equal(second, fresh(False))
        pool = expert_stream.ExpertPool(dev)
        with moe_block.patch_moe_blocks(model, mode="b200-fp8", pool=pool):
            first = layer(x[None])
            change()
            second = layer(x[None])
        assert not torch.equal(first, second) and torch.equal(second, fresh(True))


def test_banks_are_not_made_in_a_capture(dev):
    """Where the first call would be recorded instead of run, it is refused."""
    c = torch.zeros(2, 256, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 64, 128, dtype=torch.bfloat16,
                                                                              device=dev)
    with pytest.raises(ValueError, match="graph capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fp8.ExpertBanks(*c, dev)
    torch.cuda.synchronize()
    assert fp8.ExpertBanks(*c, dev).experts == 2


def test_layer_as_a_decoder_would_run_it(dev):
    """Residual and norm, router, experts and a projection together, against
    the same chain of 64-bit forms on the operators' own intermediate values."""
    g = gen(21, dev)
    tokens, hidden, inner, count, top_k = 19, 1024, 256, 16, 4
    x, res = (randn(g, tokens, hidden).to(torch.bfloat16) for _ in range(2))
    w = (0.1 * randn(g, hidden)).to(torch.bfloat16)
    router = (0.05 * randn(g, count, hidden)).to(torch.bfloat16)
    gu, gus = fp8.quantize_blocks((0.05 * randn(g, count, 2 * inner, hidden)).to(torch.bfloat16))
    dn, dns = fp8.quantize_blocks((0.05 * randn(g, count, hidden, inner)).to(torch.bfloat16))
    proj, ps = fp8.quantize_blocks((0.05 * randn(g, 384, hidden)).to(torch.bfloat16))
    q, s, normed, total = fp8.rmsnorm_quantize(x, w, res)
    check_norm((q, s, normed, total), x, w, res)
    idx, _, scores, _, _ = native.router_topk(normed, router, top_k=top_k)
    out = fp8.experts(q, s, gu, gus, dn, dns, idx, scores)
    want, bound = R.experts(q, s, gu, gus, dn, dns, idx, scores)
    within(out, want, bound, "experts")
    q2, s2, _, total2 = fp8.rmsnorm_quantize(out, w, total)
    check_norm((q2, s2, _, total2), out, w, total)
    y = fp8.linear(q2, s2, proj, ps, out_dtype=torch.float32)
    want, bound = R.linear(q2, s2, proj, ps)
    within(y, want, bound + R.F32 * want.abs(), "projection")
