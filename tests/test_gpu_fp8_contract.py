"""What the FP8 operators promise at their edges, on the GPU: waits that run
out, weights that change under a model, values across the borders where a
product changes its kernel."""

from __future__ import annotations

import pytest
import torch

from lightreason_b200 import fp8, native
from tests import fp8_reference as R
from tests.test_gpu_fp8 import dev, experts_case, gen, linear_case, randn, within  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ bounded waits ---

@pytest.fixture
def no_patience(dev):  # noqa: F811
    """No product is made: every wait for one runs out."""
    before = native.lib().moe_fp8_wait_limit(0)
    yield
    native.lib().moe_fp8_wait_limit(before)


# a tile of each kind, in one piece and split over the columns
GIVE_UP_LINEAR = [(5, 257, 272), (200, 2050, 336), (5, 2500, 7488), (33, 129, 4096), (513, 1024, 1168), (65, 4097, 3280),
                  (129, 1000, 2096), (64, 1024, 2048), (400, 4097, 1056), (200, 4097, 2240), (1000, 511, 2048),
                  (50, 2048, 3552), (2048, 2048, 512), (3000, 1001, 256), (257, 4097, 2560), (257, 2048, 6192),
                  (65, 2048, 10720)]


# CTA pairs (at least 64 groups of columns a CTA): the second CTA of the last pair with all
# its rows, some, one and none; widths on and off 16-byte units
PAIR_SHAPES = [(1024, 5001, 4000), (2560, 1000, 8128), (2198, 2052, 3984), (385, 5001, 8176), (1153, 4104, 4000),
               (2049, 2052, 4000), (1025, 4104, 3984), (1044, 4097, 4016)]


def give_up_linear(dev, tokens, rows, cols, dtype):  # noqa: F811
    """A product whose waits run out: NaN throughout, status 1, nothing beyond
    the output; then the same call with patience."""
    x, xs, w, ws = linear_case(dev, tokens, rows, cols)
    pad = 16  # elements, so that the output stays on a 16-byte boundary
    store = torch.full((tokens * rows + 2 * pad,), 7.0, dtype=dtype, device=dev)
    out = store[pad:-pad].view(tokens, rows)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    fp8.linear(x, xs, w, ws, out=out, status=status)
    torch.cuda.synchronize()
    assert status.item() == 1 and out.isnan().all()
    assert store[:pad].eq(7).all() and store[-pad:].eq(7).all()
    limit = native.lib().moe_fp8_wait_limit(2_000_000_000)
    status.zero_()
    fp8.linear(x, xs, w, ws, out=out, status=status)
    native.lib().moe_fp8_wait_limit(limit)
    want, bound = R.linear(x, xs, w, ws)
    within(out, want, bound + (R.F32 * want.abs() if dtype is torch.float32 else R.BF * (want.abs() + bound)), "out")
    assert status.item() == 0


@pytest.mark.parametrize("tokens,rows,cols", GIVE_UP_LINEAR)
def test_linear_that_gives_up_holds_nan(dev, no_patience, tokens, rows, cols):  # noqa: F811
    give_up_linear(dev, tokens, rows, cols, torch.bfloat16 if rows % 2 else torch.float32)


@pytest.mark.parametrize("tokens,rows,cols", PAIR_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_pairs_that_give_up_hold_nan_in_both_halves(dev, no_patience, tokens, rows, cols, dtype):  # noqa: F811
    give_up_linear(dev, tokens, rows, cols, dtype)


@pytest.mark.parametrize("tokens,count,top_k,hidden,inner", [(17, 16, 2, 272, 128), (40, 16, 8, 512, 256),
                                                             (300, 6, 4, 1104, 128), (600, 40, 8, 256, 128)])
def test_experts_that_give_up_hold_nan(dev, no_patience, tokens, count, top_k, hidden, inner):  # noqa: F811
    """Tiles of 16, 32 and 128 rows, route rows in FP32 and BF16."""
    c = experts_case(dev, tokens, count, top_k, hidden, inner)
    store = torch.full((tokens + 2, hidden), 7.0, dtype=torch.bfloat16, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    fp8.experts(*c, out=store[1:-1], status=status)
    torch.cuda.synchronize()
    assert status.item() == 1 and store[1:-1].isnan().all()
    assert store[0].eq(7).all() and store[-1].eq(7).all()
    native.lib().moe_fp8_wait_limit(2_000_000_000)
    status.zero_()
    got = fp8.experts(*c, status=status)
    want, bound = R.experts(*c)
    within(got, want, bound, "out")
    assert status.item() == 0


@pytest.mark.parametrize("tokens,count,top_k,hidden,inner", [(40, 64, 8, 1024, 512), (600, 40, 8, 1024, 512)])
def test_experts_that_give_up_half_way(dev, tokens, count, top_k, hidden, inner):  # noqa: F811
    """With a limit of a nanosecond the down items give up where their rows are
    not there yet: NaN throughout and status 1, or, if none had to wait, the values."""
    c = experts_case(dev, tokens, count, top_k, hidden, inner)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    want, bound = R.experts(*c)
    before = native.lib().moe_fp8_wait_limit(1)
    try:
        outs = []
        for _ in range(5):
            status.zero_()
            outs.append((fp8.experts(*c, status=status), status.clone()))
        torch.cuda.synchronize()
    finally:
        native.lib().moe_fp8_wait_limit(before)
    for out, status in outs:
        if status.item():
            assert out.isnan().all()
        else:
            within(out, want, bound, "out")
    within(fp8.experts(*c), want, bound, "afterwards")


@pytest.mark.parametrize("tokens,rows,cols", PAIR_SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_pairs(dev, tokens, rows, cols, dtype):  # noqa: F811
    """Values of CTA pairs; nothing beyond the output; a row with NaN by itself."""
    x, xs, w, ws = linear_case(dev, tokens, rows, cols)
    pad = 16
    store = torch.full((tokens * rows + 2 * pad,), 7.0, dtype=dtype, device=dev)
    out = store[pad:-pad].view(tokens, rows)
    fp8.linear(x, xs, w, ws, out=out)
    want, bound = R.linear(x, xs, w, ws)
    within(out, want, bound + (R.F32 * want.abs() if dtype is torch.float32 else R.BF * (want.abs() + bound)), "out")
    assert store[:pad].eq(7).all() and store[-pad:].eq(7).all()
    xs2 = xs.clone()
    xs2[tokens - 1, 1] = float("nan")
    got = fp8.linear(x, xs2, w, ws, out_dtype=dtype)
    assert got[-1].isnan().all() and torch.equal(got[:-1], out[:-1])


def time_of(call, calls=10):
    """Least device time of a call in microseconds, over replays of a graph of ten."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    times = []
    for _ in range(25):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    return min(times)


def test_linear_pairs_cost_no_round(dev):  # noqa: F811
    """Nine tiles of 128 rows take as long as eight where both fit one round
    of the SMs; as pairs the nine would need two (1.7 times as long)."""
    times = []
    for tokens in (1024, 1152):
        c = linear_case(dev, tokens, 4096, 4096)
        out = torch.empty(tokens, 4096, dtype=torch.bfloat16, device=dev)
        times.append(time_of(lambda: fp8.linear(*c, out=out)))  # noqa: B023
    assert times[1] < 1.35 * times[0], times


def test_linear_pairs_back_to_back(dev):  # noqa: F811
    """Pairs right behind other pairs and single CTAs on the same SMs, on both
    dtypes: the same values every time, no wait gives up."""
    shapes = [(1025, 4104, 3984, torch.bfloat16), (2198, 2052, 3984, torch.float32), (5, 2500, 7488, torch.bfloat16),
              (1044, 4097, 4016, torch.bfloat16)]
    cases = [(linear_case(dev, *s[:3]), s[3]) for s in shapes]
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    first = [fp8.linear(*c, out_dtype=d) for c, d in cases]
    torch.cuda.synchronize()
    again = [[fp8.linear(*c, out_dtype=d, status=status) for c, d in cases] for _ in range(8)]
    assert all(torch.equal(a, b) for outs in again for a, b in zip(outs, first)) and status.item() == 0


# ------------------------------------------------------------ in a model ---

def small_model(seed):
    from tests.dropin_model import make_model

    return make_model(experts=16, layers=1, seed=seed)[0]


def model_inputs(dev, tokens, seed):  # noqa: F811
    g = gen(seed, dev)
    idx = torch.rand(tokens, 16, generator=g, device=dev).topk(8, -1)[1]
    return randn(g, tokens, 2048).to(torch.bfloat16), idx, torch.softmax(randn(g, tokens, 8), -1).to(torch.bfloat16)


@pytest.mark.parametrize("mode", ["b200-fp8", "b200"])
def test_clear_between_replayed_calls(dev, mode):  # noqa: F811
    """After pool.clear() a replayed call is captured on new banks, with the
    values of weights changed where nothing sees it."""
    from lightreason_b200 import expert_stream, scheduled_graph

    model = small_model(43)
    layer, args = model.layers[0], model_inputs(dev, 3, 5)
    pool = expert_stream.ExpertPool(dev)
    with torch.no_grad(), expert_stream.patch_experts(model, mode=mode, pool=pool):
        with scheduled_graph.replay_experts(pool):
            first = layer.experts(*args).clone()
            layer.experts.down_proj.data.mul_(2)
            pool.clear()
            taken = [torch.full((64 << 20,), 0x7f, dtype=torch.uint8, device=dev) for _ in range(4)]  # the banks' old memory
            second = layer.experts(*args).clone()
            third = layer.experts(*args).clone()
            del taken
        eager = layer.experts(*args)
    assert torch.equal(second, 2 * first) and torch.equal(third, second) and torch.equal(eager, second)
    pool.clear()


def test_block_made_in_inference_mode_and_called_outside_it(dev):  # noqa: F811
    """Router, shared expert and experts changed between a call in inference
    mode and one under no_grad: the second has the new values."""
    from lightreason_b200 import expert_stream, moe_block

    model = small_model(44)
    layer, x = model.layers[0], model_inputs(dev, 3, 6)[0][None]

    def fresh():
        with torch.no_grad(), moe_block.patch_moe_blocks(model, mode="b200-fp8", pool=expert_stream.ExpertPool(dev)):
            return layer(x)

    pool = expert_stream.ExpertPool(dev)
    with moe_block.patch_moe_blocks(model, mode="b200-fp8", pool=pool):
        with torch.inference_mode():
            first = layer(x)
        with torch.no_grad():
            layer.gate.weight.copy_(layer.gate.weight.flip(0).clone())
            layer.experts.down_proj.mul_(0.5)
            second = layer(x)
        with torch.inference_mode():
            third = layer(x)
    assert not torch.equal(first, second) and torch.equal(second, fresh()) and torch.equal(third, second)


# ----------------------------------------------------- forward-mode tangents ---

def test_forward_mode_tangents_are_refused(dev):  # noqa: F811
    """A tensor that carries a tangent is refused instead of losing it."""
    import torch.autograd.forward_ad as fwd

    x, xs, gu, gus, dn, dns, idx, wt = experts_case(dev, 3, 4, 2, 256, 128)
    b, w = torch.ones(3, 256, dtype=torch.bfloat16, device=dev), torch.ones(256, dtype=torch.bfloat16, device=dev)
    with torch.no_grad(), fwd.dual_level():
        dual = lambda t: fwd.make_dual(t.clone(), torch.ones_like(t))  # noqa: E731
        for call in (lambda: fp8.quantize_rows(dual(b)), lambda: fp8.quantize_blocks(dual(b)),
                     lambda: fp8.rmsnorm_quantize(dual(b), w), lambda: fp8.rmsnorm_quantize(b, dual(w)),
                     lambda: fp8.rmsnorm_quantize(b, w, dual(b)), lambda: fp8.linear(x, dual(xs), gu[0], gus[0]),
                     lambda: fp8.linear(x, xs, gu[0], dual(gus[0])),
                     lambda: fp8.experts(x, xs, gu, gus, dn, dns, idx, dual(wt)),
                     lambda: fp8.experts(x, dual(xs), gu, gus, dn, dns, idx, wt)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        q, s = fp8.quantize_rows(fwd.unpack_dual(dual(b)).primal)  # the values alone are taken
    assert q.shape == (3, 256) and torch.equal(s, fp8.quantize_rows(b)[1])


# --------------------------------------------------- kernels that overlap ---

@pytest.mark.parametrize("tokens", [2, 5, 64, 300])
def test_each_kernel_reads_what_the_one_before_wrote(dev, tokens):  # noqa: F811
    """Rows and weights quantised into the same memory again and again, right
    before the products that read them, and route ids written right before the
    experts: every call sees its own inputs."""
    g = gen(tokens, dev)
    rows = [randn(g, tokens, 1024).to(torch.bfloat16) for _ in range(5)]
    mats = [(0.05 * randn(g, 512, 1024)).to(torch.bfloat16) for _ in range(5)]
    norms = [randn(g, 1024).to(torch.bfloat16) for _ in range(5)]
    banks = [((0.05 * randn(g, 4, 256, 1024)).to(torch.bfloat16), (0.05 * randn(g, 4, 1024, 128)).to(torch.bfloat16))
             for _ in range(5)]
    routers = [randn(g, 4, 1024).to(torch.bfloat16) for _ in range(5)]

    def step(k, q, s, w, gu, dn, norm, wait):
        pause = torch.cuda.synchronize if wait else (lambda: None)
        norm.copy_(norms[k])
        pause()
        fp8.rmsnorm_quantize(rows[k], norm, out=(q, s, None, None))
        pause()
        fp8.quantize_blocks(mats[k], out=w)
        pause()
        a = fp8.linear(q, s, *w)
        pause()
        idx, _, scores, _, _ = native.router_topk(rows[k], routers[k], top_k=2)
        pause()
        fp8.quantize_blocks(banks[k][0], out=gu)
        pause()
        fp8.quantize_blocks(banks[k][1], out=dn)
        pause()
        return a, fp8.experts(q, s, *gu, *dn, idx, scores), fp8.quantize_rows(a)[0]

    memory = (*fp8.quantize_rows(rows[0]), fp8.quantize_blocks(mats[0]), *map(fp8.quantize_blocks, banks[0]),
              norms[0].clone())
    want = [step(k, *memory, True) for k in range(5)]
    got = [step(k % 5, *memory, False) for k in range(20)]
    torch.cuda.synchronize()
    for k, outs in enumerate(got):
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs, want[k % 5])), k


# ------------------------------------------------ across a product's borders ---

def whole_experts_case(dev, tokens, count, top_k, seed=0):  # noqa: F811
    """Values whose gate and up sums are whole numbers below 2^13 times 2^-5, so
    that FP32 (and any tensor core's sum) has them exactly; H 256, I 128."""
    g = gen(seed + tokens, dev)
    ints = lambda top, *s: torch.randint(-top, top + 1, s, generator=g, device=dev).float()  # noqa: E731
    x, gu, dn = (v.to(torch.float8_e4m3fn) for v in (ints(2, tokens, 256), ints(3, count, 256, 256), ints(7, count, 256, 128)))
    xs, gus, dns = (torch.full(s, v, device=dev) for s, v in (((tokens, 2), 1.0), ((count, 2, 2), 2.0 ** -5), ((count, 2, 1), 0.5)))
    idx = torch.rand(tokens, count, generator=g, device=dev).topk(top_k, -1)[1]
    return x, xs, gu, gus, dn, dns, idx.contiguous(), torch.softmax(randn(g, tokens, top_k), -1).to(torch.bfloat16)


def whole_experts(x, xs, gu, gus, dn, dns, idx, weights):
    """(exact, bound, sum over the routes of weight times |row|) for such values.
    gate and up are exact; SiLU is off by 2^-23 (4.5 + 1.2 |gate|) of itself (the
    documented errors of the fast exponential and quotient, and a rounding), the
    product and the scale by two more roundings; a value of h that this may carry
    over a border moves by a step.  The down sums as in fp8_reference, the
    weighted sum k roundings, BF16 at the end."""
    out = torch.zeros(x.shape[0], dn.shape[1], dtype=torch.float64, device=x.device)
    bound, size = torch.zeros_like(out), torch.zeros_like(out)
    xd = R.widen_rows(x, xs)
    for e in range(gu.shape[0]):
        token, slot = torch.nonzero(idx == e, as_tuple=True)
        p = xd[token] @ R.widen_blocks(gu[e], gus[e]).T
        gate, up = p[:, :128], p[:, 128:]
        h = gate * torch.sigmoid(gate) * up
        off = 2 * R.F32 * (4.5 + 1.2 * gate.abs()) + 2 * R.F32
        v, q, s = R.rows(h)
        far = 2 * off.amax(-1, keepdim=True) + 4 * R.F32       # of v: its own error and its group's maximum's
        near = ((v / R.step(v) - torch.floor(v / R.step(v)) - 0.5).abs() * R.step(v)) <= far * v.abs()
        qb = torch.where(near, R.step(v), torch.zeros_like(v))
        wd = R.widen_blocks(dn[e], dns[e])
        y = (q * s) @ wd.T
        yb = (qb * s) @ wd.abs().T + (R.chain(128) * R.F32 + far) * ((q * s).abs() @ wd.abs().T)
        wt = weights[token, slot].double()[:, None]
        out.index_add_(0, token, y * wt)
        bound.index_add_(0, token, (yb + idx.shape[1] * R.F32 * y.abs()) * wt)
        size.index_add_(0, token, y.abs() * wt)
    return out, bound + R.BF * (out.abs() + bound), size


@pytest.mark.parametrize("tokens,count,top_k", [(1, 8, 8), (3, 6, 4), (2, 9, 7), (20, 8, 8), (100, 64, 8), (256, 8, 8), (128, 20, 16)])
def test_experts_up_to_2048_routes_keep_rows_in_fp32(dev, tokens, count, top_k):  # noqa: F811
    """GEMV and tiles of every kind up to 2048 routes: one rounding to BF16, at
    the end (rounding each route's row too would leave the bound)."""
    c = whole_experts_case(dev, tokens, count, top_k)
    want, bound, _ = whole_experts(*c)
    within(fp8.experts(*c), want, bound, "out")


def test_experts_above_2048_routes_round_their_rows(dev):  # noqa: F811
    """The 2049th route brings the rounding of each route's row to BF16, for
    every token of the batch; without it the values of 2048 routes."""
    c = whole_experts_case(dev, 257, 8, 8)
    want, bound, size = whole_experts(*c)
    within(fp8.experts(*c), want, bound + 1.01 * R.BF * size, "out")
    first = [t[:256] if t.shape[0] == 257 else t for t in c]
    within(fp8.experts(*first), want[:256], bound[:256], "256 tokens")


def test_linear_rows_in_batches_of_every_size(dev):  # noqa: F811
    """One row in batches that take other kernels, tiles and splits: its bits may
    differ, each is within the bound of a sum in FP32."""
    for rows, cols in ((1024, 2048), (300, 4112), (9216, 512)):
        x, xs, w, ws = linear_case(dev, 600, rows, cols)
        want, bound = R.linear(x, xs, w, ws)
        for tokens in (1, 2, 4, 5, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257, 600):
            got = fp8.linear(x[:tokens], xs[:tokens], w, ws, out_dtype=torch.float32)
            within(got, want[:tokens], (bound + R.F32 * want.abs())[:tokens], f"{tokens} rows of {cols}")


# ----------------------------------------------------------- largest widths ---

@pytest.mark.parametrize("tokens,count,top_k,hidden,inner", [(1, 2, 2, 16, 16384), (40, 2, 1, 16, 16384), (300, 2, 1, 16, 16384),
                                                             (2, 2, 2, 65536, 128), (40, 2, 1, 65536, 128),
                                                             (300, 2, 1, 65536, 128)])
def test_experts_at_the_widest(dev, tokens, count, top_k, hidden, inner):  # noqa: F811
    c = experts_case(dev, tokens, count, top_k, hidden, inner)
    want, bound = R.experts(*c)
    within(fp8.experts(*c), want, bound, "out")


@pytest.mark.parametrize("tokens,rows,cols", [(1, 3, 1 << 20), (4, 130, 1 << 19), (5, 3, 1 << 20), (40, 130, 1 << 18),
                                              (300, 257, 1 << 17)])
def test_linear_at_long_rows(dev, tokens, rows, cols):  # noqa: F811
    x, xs, w, ws = linear_case(dev, tokens, rows, cols)
    want, bound = R.linear(x, xs, w, ws)
    within(fp8.linear(x, xs, w, ws, out_dtype=torch.float32), want, bound + R.F32 * want.abs(), "f32")


@pytest.mark.parametrize("tokens", [1, 3])
def test_rows_at_the_widest(dev, tokens):  # noqa: F811
    """2^20 values a row: e4m3 exact; the norm within the longest chain of its
    sum (2^20 / 256 terms a thread, halved by the root, and eight roundings)."""
    g = gen(tokens, dev)
    x = randn(g, tokens, 1 << 20).to(torch.bfloat16)
    q, s = fp8.quantize_rows(x)
    _, want, scale = R.rows(x.double())
    assert torch.equal(q.double(), want) and torch.equal(s, scale.float())
    w = (0.5 * randn(g, 1 << 20)).to(torch.bfloat16)
    _, s, normed, _ = fp8.rmsnorm_quantize(x, w)
    xd = x.double()
    y = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
    rel = (4096 + 16) * R.F32
    within(normed, y, (R.BF + rel) * y.abs() + 2.0 ** -134, "normed")
    within(s, R.tops(y) / R.TOP, rel * R.tops(y) / R.TOP, "scales")
