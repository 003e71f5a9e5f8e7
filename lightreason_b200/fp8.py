"""The MoE layer's operators on FP8 (e4m3) values with FP32 scales.

Activations carry one scale per row and 128 columns, weights one per 128 x 128
block: a group of values v is held as q = e4m3(v * 448 / a) and a / 448, with a
the group's largest magnitude (at least 1e-10), and read back as q * scale.

  quantize_rows      BF16 rows -> q, scales
  rmsnorm_quantize   residual addition, RMS norm, then q, scales (and the BF16
                     rows a router reads)
  quantize_blocks    BF16 weights -> q, block scales
  linear             rows . weight^T
  experts            the routed SwiGLU experts (Qwen3_5MoeExperts.forward) on
                     FP8 banks, routes given

`patch_experts(model, mode="b200-fp8", pool=...)` and `patch_moe_blocks` run a
model's experts on them (ExpertBanks).  Like the rest of the package they are inference operators: no gradients.
Work is enqueued on the tensors' device's current stream without a host
synchronisation and can be captured in a CUDA graph; `out=` takes outputs that
the caller keeps.
"""

from __future__ import annotations

import ctypes
import importlib.util
import weakref
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from lightreason_b200 import build, native
from lightreason_b200.native import _require

GROUP = 128
MAX_ROUTES = 32  # of a token, in experts
E4M3 = torch.float8_e4m3fn
_BF16, _F32 = torch.bfloat16, torch.float32

# These calls sit in decode loops that may run uncaptured, where the checks of a
# call's tensors in Python would take longer than its launch.  Each goes to its
# namesake in _fp8_bind (csrc/fp8_bind.cpp), which makes the same checks and the
# call.  What it does not take comes back as None: the Python below then goes
# through the checks one by one and raises at the first that fails.


@lru_cache(maxsize=1)
def _bind():
    """The module, with the C ABI's addresses in the loaded library."""
    path = str(build.BIND)
    if not build.BIND.exists():
        raise RuntimeError(f"{path} is missing: build it with `python -m lightreason_b200.build` (it needs a host "
                           "C++ compiler and the headers of Python and of this torch)")
    spec = importlib.util.spec_from_file_location("_fp8_bind", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    so = native.lib()
    module.bind(*(ctypes.cast(getattr(so, name), ctypes.c_void_p).value for name in (
        "moe_rmsnorm_fp8", "moe_quantize_fp8_blocks", "moe_linear_fp8", "moe_experts_fp8",
        "moe_experts_fp8_workspace_bytes")))
    return module


def _groups(n: int) -> int:
    return -(-n // GROUP)


def _check(t, name: str, dtype: torch.dtype, shape: tuple, index: int) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == index
            and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on cuda:{index}")


def _refused(name: str, status) -> None:
    """The end of a call that _fp8_bind did not answer with a result."""
    if status is None:
        raise ValueError(f"{name}: arguments out of range")
    native.check(status, name)


def _no_grad(*tensors) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the FP8 operators have no forward-mode derivative: a tensor carries a tangent")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the FP8 operators have no gradient: call them under torch.no_grad() or "
                           "torch.inference_mode()")


def _rows(t: torch.Tensor, name: str) -> int:
    """The row stride of a [T, H] BF16 CUDA tensor with dense rows."""
    if not (t.is_cuda and t.dtype is _BF16 and t.dim() == 2):
        raise ValueError(f"{name} must be a CUDA BF16 [T, H] tensor")
    tokens, hidden = t.shape
    step, unit = t.stride()
    _require(hidden >= 1, f"{name} has no columns")
    _require((hidden == 1 or unit == 1) and (tokens <= 1 or step >= hidden),
             f"{name} must have dense rows that do not overlap")
    return step if tokens > 1 else hidden


def quantize_rows(x: torch.Tensor, *, out=None):
    """BF16 rows [T, H] (any row stride) -> (q e4m3 [T, H], scales f32
    [T, ceil(H / 128)]).  out: the same pair, to be written."""
    if out is None and isinstance(x, torch.Tensor) and x.dim() == 2 and x.is_cuda:
        out = (torch.empty(x.shape, dtype=E4M3, device=x.device),
               torch.empty((x.shape[0], _groups(x.shape[1])), dtype=_F32, device=x.device))
    q, scales = out if out is not None else (None, None)
    done = _bind().rows(x, None, None, 0.0, 0.0, q, scales, None, None)
    if done is True:
        return q, scales
    _rows(x, "x")
    _no_grad(x)
    index = x.get_device()
    _check(q, "out[0]", E4M3, x.shape, index)
    _check(scales, "out[1]", _F32, (x.shape[0], _groups(x.shape[1])), index)
    _refused("moe_rmsnorm_fp8", done)


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                     eps: float = 1e-6, weight_offset: float = 1.0, normed: bool = True, out=None):
    """r = bf16(x + residual) (x without a residual), y = r * rsqrt(mean(r^2) +
    eps) * (weight_offset + weight).  Returns (q, scales, normed, residual_out):
    y as e4m3 [T, H] with f32 scales, y as BF16 (None with normed=False) and r
    (None without a residual).  weight_offset: 1 for Qwen3_5MoeRMSNorm, whose
    weight is stored around zero; 0 for plain norms.  out: the same four, to be
    written; its residual_out may be `residual` itself and its normed `x`."""
    if out is None and isinstance(x, torch.Tensor) and x.dim() == 2 and x.is_cuda:
        shape, dev = x.shape, x.device
        out = (torch.empty(shape, dtype=E4M3, device=dev),
               torch.empty((shape[0], _groups(shape[1])), dtype=_F32, device=dev),
               torch.empty(shape, dtype=_BF16, device=dev) if normed else None,
               torch.empty(shape, dtype=_BF16, device=dev) if residual is not None else None)
    q, scales, y, r = out if out is not None else (None, None, None, None)
    done = _bind().rows(x, weight, residual, eps, weight_offset, q, scales, y, r) if weight is not None else None
    if done is True:
        return q, scales, y, r
    _rows(x, "x")
    tokens, hidden = shape = x.shape
    index = x.get_device()
    _check(weight, "weight", _BF16, (hidden,), index)
    _no_grad(x, weight, residual)
    if residual is not None:
        _rows(residual, "residual")
        _require(residual.shape == shape and residual.get_device() == index,
                 "residual must have x's shape and device")
    _check(q, "out[0]", E4M3, shape, index)
    _check(scales, "out[1]", _F32, (tokens, _groups(hidden)), index)
    if y is not None:
        _check(y, "out[2]", _BF16, shape, index)
    if r is not None:
        _require(residual is not None, "out[3] without a residual")
        _check(r, "out[3]", _BF16, shape, index)
    _refused("moe_rmsnorm_fp8", done)


def quantize_blocks(w: torch.Tensor, *, out=None):
    """BF16 weights [N, K] or [banks, N, K] -> (q e4m3, scales f32 [(banks,)
    ceil(N / 128), ceil(K / 128)])."""
    q, scales = out if out is not None else (None, None)
    done = _bind().blocks(w, q, scales)
    if isinstance(done, tuple):
        return done
    _require(isinstance(w, torch.Tensor) and w.is_cuda and w.dtype is _BF16 and w.dim() in (2, 3)
             and w.is_contiguous(), "w must be a contiguous CUDA BF16 [N, K] or [banks, N, K] tensor")
    _no_grad(w)
    shape = w.shape
    _require(shape[-2] >= 1 and shape[-1] >= 1, "w has no rows or columns")
    if out is not None:
        _check(q, "out[0]", E4M3, shape, w.get_device())
        _check(scales, "out[1]", _F32, (*shape[:-2], _groups(shape[-2]), _groups(shape[-1])), w.get_device())
    _refused("moe_quantize_fp8_blocks", done)


def linear(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
           out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
           status: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] . w [N, K]^T on the values that the e4m3 tensors and their
    scales stand for -> [T, N] in BF16 or FP32 (out_dtype, or out's).  K must be
    a multiple of 16.  status: a device int32 [1] that becomes 1 if a bounded
    wait inside a kernel gave up (the output then holds NaN)."""
    if out is None:
        _require(out_dtype in (_BF16, _F32), "out_dtype must be BF16 or FP32")
    done = _bind().linear(x, x_scales, w, w_scales, out, out_dtype is _F32, status)
    if isinstance(done, torch.Tensor):
        return done
    _require(isinstance(x, torch.Tensor) and isinstance(w, torch.Tensor) and x.is_cuda and x.dim() == 2
             and w.dim() == 2, "x and w must be CUDA [T, K] and [N, K] tensors")
    tokens, cols = x.shape
    rows, index, groups = w.shape[0], x.get_device(), _groups(cols)
    _require(rows >= 1 and cols >= 16 and cols % 16 == 0, "K must be a positive multiple of 16 and N positive")
    _check(x, "x", E4M3, (tokens, cols), index)
    _check(x_scales, "x_scales", _F32, (tokens, groups), index)
    _check(w, "w", E4M3, (rows, cols), index)
    _check(w_scales, "w_scales", _F32, (_groups(rows), groups), index)
    if out is not None:
        _require(out.dtype in (_BF16, _F32), "out must be BF16 or FP32")
        _check(out, "out", out.dtype, (tokens, rows), index)
    if status is not None:
        _check(status, "status", torch.int32, (1,), index)
    _no_grad(x, x_scales, w, w_scales, out)
    _refused("moe_linear_fp8", done)


def experts(x: torch.Tensor, x_scales: torch.Tensor, gate_up: torch.Tensor, gate_up_scales: torch.Tensor,
            down: torch.Tensor, down_scales: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, *,
            out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The routed experts on FP8 banks: x e4m3 [T, H] with its scales, gate_up
    [E, 2I, H] and down [E, H, I] with their block scales, idx int64 [T, K]
    (ids outside [0, E) contribute nothing), weights BF16 [T, K] -> BF16 [T, H].
    H is a multiple of 16, I of 128.  status as in linear."""
    done = _bind().experts(x, x_scales, gate_up, gate_up_scales, down, down_scales, idx, weights, out, status)
    if isinstance(done, torch.Tensor):
        return done
    _require(all(isinstance(t, torch.Tensor) for t in (x, gate_up, down, idx)) and x.is_cuda and x.dim() == 2
             and gate_up.dim() == 3 and down.dim() == 3 and idx.dim() == 2,
             "expected x [T, H], gate_up [E, 2I, H], down [E, H, I] and idx [T, K] on a CUDA device")
    tokens, hidden = shape = x.shape
    index, groups = x.get_device(), _groups(hidden)
    count, inner, top_k = gate_up.shape[0], down.shape[2], idx.shape[1]
    _check(x, "x", E4M3, shape, index)
    _check(x_scales, "x_scales", _F32, (tokens, groups), index)
    _check(gate_up, "gate_up", E4M3, (count, 2 * inner, hidden), index)
    _check(gate_up_scales, "gate_up_scales", _F32, (count, _groups(2 * inner), groups), index)
    _check(down, "down", E4M3, (count, hidden, inner), index)
    _check(down_scales, "down_scales", _F32, (count, groups, _groups(inner)), index)
    _check(idx, "idx", torch.int64, (tokens, top_k), index)
    _check(weights, "weights", _BF16, (tokens, top_k), index)
    if out is not None:
        _check(out, "out", _BF16, shape, index)
    if status is not None:
        _check(status, "status", torch.int32, (1,), index)
    _no_grad(x_scales, gate_up_scales, down_scales, weights, out)
    _refused("moe_experts_fp8", done)


class ExpertBanks:
    """The FP8 banks of one layer's experts, made from BF16 ones.

    gate_up [E, 2I, H] and down [E, H, I] may live on the CPU or on the device;
    they are brought over and quantised a few experts at a time, so the BF16
    bank is never whole on the device because of this.  shared: a further
    expert (gate [I, H], up [I, H], down [H, I]), kept as expert id E.  extra:
    tensors that go with the layer, copied to the device as they are."""

    CHUNK = 16  # experts quantised at once

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, device, *, shared=(), extra=()):
        count, rows, hidden = gate_up.shape
        inner = rows // 2
        _require(tuple(down.shape) == (count, hidden, inner), "gate_up must be [E, 2I, H] and down [E, H, I]")
        total = count + bool(shared)
        check_widths(hidden, inner, total)
        self.experts, self.hidden, self.inner, self.device = count, hidden, inner, torch.device(device)
        make = lambda n, k: (torch.empty((total, n, k), dtype=E4M3, device=self.device),  # noqa: E731
                             torch.empty((total, _groups(n), _groups(k)), dtype=_F32, device=self.device))
        with torch.inference_mode(False):  # a later load may come from outside inference mode
            self.gate_up, self.gate_up_scales = make(rows, hidden)
            self.down, self.down_scales = make(hidden, inner)
            self.extra = tuple(torch.empty(t.shape, dtype=t.dtype, device=self.device) for t in extra)
        self.load(gate_up, down, shared=shared, extra=extra)

    def takes(self, gate_up: torch.Tensor, down: torch.Tensor, shared=(), extra=()) -> bool:
        """Whether load() has room for these (a shared expert or none, as when the banks were made)."""
        count, hidden, inner = self.experts, self.hidden, self.inner
        return (tuple(gate_up.shape) == (count, 2 * inner, hidden) and tuple(down.shape) == (count, hidden, inner)
                and self.gate_up.shape[0] == count + bool(shared)
                and [(t.shape, t.dtype) for t in extra] == [(t.shape, t.dtype) for t in self.extra])

    def load(self, gate_up: torch.Tensor, down: torch.Tensor, *, shared=(), extra=()) -> None:
        """Brings these weights into the banks' memory, where captured graphs
        that read it find them too."""
        _require(not (self.device.type == "cuda" and torch.cuda.is_current_stream_capturing()),
                 "FP8 banks cannot be made during a graph capture: call the layer once before it")
        count, hidden, inner = self.experts, self.hidden, self.inner
        _require(self.takes(gate_up, down, shared, extra), "the weights do not have the banks' shapes")
        _require(not shared or [tuple(t.shape) for t in shared] == [(inner, hidden)] * 2 + [(hidden, inner)],
                 "the shared expert must have the experts' widths")
        self._sources = []  # held only once all of them are there
        parts = [(a, min(a + self.CHUNK, count)) for a in range(0, count, self.CHUNK)]
        with torch.no_grad():
            for source, q, scales in ((gate_up, self.gate_up, self.gate_up_scales),
                                      (down, self.down, self.down_scales)):
                for a, b in parts:
                    quantize_blocks(source[a:b].detach().to(self.device).contiguous(), out=(q[a:b], scales[a:b]))
            if shared:
                gate, up, last = (t.detach().to(self.device) for t in shared)
                quantize_blocks(torch.cat([gate, up])[None], out=(self.gate_up[count:], self.gate_up_scales[count:]))
                quantize_blocks(last[None].contiguous(), out=(self.down[count:], self.down_scales[count:]))
            for held, t in zip(self.extra, extra):
                held.copy_(t)
        self._sources = [(weakref.ref(t), _version(t)) for t in (gate_up, down, *shared, *extra)]

    def holds(self, *sources: torch.Tensor) -> bool:
        """Whether these are the tensors last loaded (in load's order), unchanged
        since.  Changes made behind autograd's version counter (through .data, or
        to tensors made in inference mode) are not seen."""
        return len(sources) == len(self._sources) and all(
            ref() is t and version == _version(t) for (ref, version), t in zip(self._sources, sources))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size()
                   for t in (self.gate_up, self.gate_up_scales, self.down, self.down_scales, *self.extra))

    def release(self) -> None:
        """Part of the pool's layer interface; the banks go with their tensors."""

    def __call__(self, hidden: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """The experts' forward on BF16 states: quantised rows, then experts()."""
        q, scales = quantize_rows(hidden)
        return experts(q, scales, self.gate_up, self.gate_up_scales, self.down, self.down_scales, idx, weights)


def _version(t: torch.Tensor) -> int:
    return -1 if t.is_inference() else t._version


def check_widths(hidden: int, inner: int, experts: int = 1) -> None:
    """The widths and numbers of experts that the expert kernels take."""
    _require(hidden % 16 == 0 and inner % 128 == 0,
             f"FP8 experts need hidden a multiple of 16 and inner of 128, got {hidden} and {inner}")
    _require(16 <= hidden <= 65536 and 128 <= inner <= 16384 and 1 <= experts <= 1024,
             f"FP8 experts take hidden up to 65536, inner up to 16384 and 1024 experts (a shared one counts), got "
             f"{hidden}, {inner} and {experts}")
