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

`patch_experts(model, mode="b200-fp8", pool=...)` runs a model's experts on
them.  Like the rest of the package they are inference operators: no gradients.
Work is enqueued on the tensors' device's current stream without a host
synchronisation and can be captured in a CUDA graph; `out=` takes outputs that
the caller keeps.
"""

from __future__ import annotations

import contextlib

import torch

from lightreason_b200 import native
from lightreason_b200.native import _require

GROUP = 128
E4M3 = torch.float8_e4m3fn


def _groups(n: int) -> int:
    return -(-n // GROUP)


def _on(device: torch.device):
    """The calls launch on the current device: make it the tensors'."""
    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.device == device and t.shape == shape
            and t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {device}")


def _no_grad(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the FP8 operators have no gradient: call them under torch.no_grad() or "
                           "torch.inference_mode()")


def _rows(t: torch.Tensor, name: str) -> int:
    """The row stride of a [T, H] BF16 CUDA tensor with dense rows."""
    _require(t.is_cuda and t.dtype == torch.bfloat16 and t.dim() == 2, f"{name} must be a CUDA BF16 [T, H] tensor")
    tokens, hidden = t.shape
    _require(hidden >= 1, f"{name} has no columns")
    _require((hidden == 1 or t.stride(1) == 1) and (tokens <= 1 or t.stride(0) >= hidden),
             f"{name} must have dense rows that do not overlap")
    return t.stride(0) if tokens > 1 else hidden


def quantize_rows(x: torch.Tensor, *, out=None):
    """BF16 rows [T, H] (any row stride) -> (q e4m3 [T, H], scales f32
    [T, ceil(H / 128)]).  out: the same pair, to be written."""
    stride = _rows(x, "x")
    _no_grad(x)
    (tokens, hidden), dev = x.shape, x.device
    if out is None:
        out = (torch.empty((tokens, hidden), dtype=E4M3, device=dev),
               torch.empty((tokens, _groups(hidden)), dtype=torch.float32, device=dev))
    q, scales = out
    _check(q, "out[0]", E4M3, (tokens, hidden), dev)
    _check(scales, "out[1]", torch.float32, (tokens, _groups(hidden)), dev)
    with _on(dev):
        native.check(native.lib().moe_rmsnorm_fp8(x.data_ptr(), stride, None, 0, None, 0.0, 0.0, tokens, hidden,
                                                  q.data_ptr(), scales.data_ptr(), None, None, native._stream(dev)),
                     "moe_rmsnorm_fp8")
    return q, scales


def rmsnorm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                     eps: float = 1e-6, weight_offset: float = 1.0, normed: bool = True, out=None):
    """r = bf16(x + residual) (x without a residual), y = r * rsqrt(mean(r^2) +
    eps) * (weight_offset + weight).  Returns (q, scales, normed, residual_out):
    y as e4m3 [T, H] with f32 scales, y as BF16 (None with normed=False) and r
    (None without a residual).  weight_offset: 1 for Qwen3_5MoeRMSNorm, whose
    weight is stored around zero; 0 for plain norms.  out: the same four, to be
    written; its residual_out may be `residual` itself and its normed `x`."""
    stride = _rows(x, "x")
    (tokens, hidden), dev = x.shape, x.device
    _no_grad(x, weight, residual)
    _check(weight, "weight", torch.bfloat16, (hidden,), dev)
    rstride = 0
    if residual is not None:
        rstride = _rows(residual, "residual")
        _require(residual.shape == x.shape and residual.device == dev, "residual must have x's shape and device")
    if out is None:
        bf = dict(dtype=torch.bfloat16, device=dev)
        out = (torch.empty((tokens, hidden), dtype=E4M3, device=dev),
               torch.empty((tokens, _groups(hidden)), dtype=torch.float32, device=dev),
               torch.empty((tokens, hidden), **bf) if normed else None,
               torch.empty((tokens, hidden), **bf) if residual is not None else None)
    q, scales, y, r = out
    _check(q, "out[0]", E4M3, (tokens, hidden), dev)
    _check(scales, "out[1]", torch.float32, (tokens, _groups(hidden)), dev)
    if y is not None:
        _check(y, "out[2]", torch.bfloat16, (tokens, hidden), dev)
    if r is not None:
        _require(residual is not None, "out[3] without a residual")
        _check(r, "out[3]", torch.bfloat16, (tokens, hidden), dev)
    with _on(dev):
        native.check(native.lib().moe_rmsnorm_fp8(
            x.data_ptr(), stride, native._ptr(residual), rstride, weight.data_ptr(), weight_offset, eps, tokens,
            hidden, q.data_ptr(), scales.data_ptr(), native._ptr(y), native._ptr(r), native._stream(dev)),
            "moe_rmsnorm_fp8")
    return out


def quantize_blocks(w: torch.Tensor, *, out=None):
    """BF16 weights [N, K] or [banks, N, K] -> (q e4m3, scales f32 [(banks,)
    ceil(N / 128), ceil(K / 128)])."""
    _require(w.is_cuda and w.dtype == torch.bfloat16 and w.dim() in (2, 3) and w.is_contiguous(),
             "w must be a contiguous CUDA BF16 [N, K] or [banks, N, K] tensor")
    _no_grad(w)
    rows, cols = w.shape[-2:]
    banks = w.shape[0] if w.dim() == 3 else 1
    _require(rows >= 1 and cols >= 1, "w has no rows or columns")
    shape = (*w.shape[:-2], _groups(rows), _groups(cols))
    if out is None:
        out = (torch.empty(w.shape, dtype=E4M3, device=w.device),
               torch.empty(shape, dtype=torch.float32, device=w.device))
    q, scales = out
    _check(q, "out[0]", E4M3, tuple(w.shape), w.device)
    _check(scales, "out[1]", torch.float32, shape, w.device)
    with _on(w.device):
        native.check(native.lib().moe_quantize_fp8_blocks(w.data_ptr(), banks, rows, cols, q.data_ptr(),
                                                          scales.data_ptr(), native._stream(w.device)),
                     "moe_quantize_fp8_blocks")
    return out


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    """Scratch from torch's allocator for one call: calls never share it, and a
    captured graph keeps its own in the graph's pool."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def linear(x: torch.Tensor, x_scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, *,
           out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
           status: torch.Tensor | None = None) -> torch.Tensor:
    """x [T, K] . w [N, K]^T on the values that the e4m3 tensors and their
    scales stand for -> [T, N] in BF16 or FP32 (out_dtype, or out's).  K must be
    a multiple of 16.  status: a device int32 [1] that becomes 1 if a bounded
    wait inside a kernel gave up (the output is then not valid)."""
    _require(x.is_cuda and x.dim() == 2 and w.dim() == 2, "x and w must be CUDA [T, K] and [N, K] tensors")
    (tokens, cols), rows, dev = x.shape, w.shape[0], x.device
    _require(rows >= 1 and cols >= 16 and cols % 16 == 0, "K must be a positive multiple of 16 and N positive")
    _check(x, "x", E4M3, (tokens, cols), dev)
    _check(x_scales, "x_scales", torch.float32, (tokens, _groups(cols)), dev)
    _check(w, "w", E4M3, (rows, cols), dev)
    _check(w_scales, "w_scales", torch.float32, (_groups(rows), _groups(cols)), dev)
    if out is None:
        _require(out_dtype in (torch.bfloat16, torch.float32), "out_dtype must be BF16 or FP32")
        out = torch.empty((tokens, rows), dtype=out_dtype, device=dev)
    else:
        _require(out.dtype in (torch.bfloat16, torch.float32), "out must be BF16 or FP32")
        _check(out, "out", out.dtype, (tokens, rows), dev)
    if status is not None:
        _check(status, "status", torch.int32, (1,), dev)
    so = native.lib()
    ws = _workspace(so.moe_linear_fp8_workspace_bytes(tokens, rows, cols), dev)
    with _on(dev):
        native.check(so.moe_linear_fp8(x.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(), tokens,
                                       rows, cols, out.data_ptr(), int(out.dtype == torch.float32), native._ptr(ws),
                                       ws.numel() if ws is not None else 0, native._ptr(status), native._stream(dev)),
                     "moe_linear_fp8")
    return out


def experts(x: torch.Tensor, x_scales: torch.Tensor, gate_up: torch.Tensor, gate_up_scales: torch.Tensor,
            down: torch.Tensor, down_scales: torch.Tensor, idx: torch.Tensor, weights: torch.Tensor, *,
            out: torch.Tensor | None = None, status: torch.Tensor | None = None) -> torch.Tensor:
    """The routed experts on FP8 banks: x e4m3 [T, H] with its scales, gate_up
    [E, 2I, H] and down [E, H, I] with their block scales, idx int64 [T, K]
    (ids outside [0, E) contribute nothing), weights BF16 [T, K] -> BF16 [T, H].
    H is a multiple of 16, I of 128.  status as in linear."""
    _require(x.is_cuda and x.dim() == 2 and gate_up.dim() == 3 and down.dim() == 3 and idx.dim() == 2,
             "expected x [T, H], gate_up [E, 2I, H], down [E, H, I] and idx [T, K] on a CUDA device")
    (tokens, hidden), dev = x.shape, x.device
    count, inner, top_k = gate_up.shape[0], down.shape[2], idx.shape[1]
    _check(x, "x", E4M3, (tokens, hidden), dev)
    _check(x_scales, "x_scales", torch.float32, (tokens, _groups(hidden)), dev)
    _check(gate_up, "gate_up", E4M3, (count, 2 * inner, hidden), dev)
    _check(gate_up_scales, "gate_up_scales", torch.float32, (count, _groups(2 * inner), _groups(hidden)), dev)
    _check(down, "down", E4M3, (count, hidden, inner), dev)
    _check(down_scales, "down_scales", torch.float32, (count, _groups(hidden), _groups(inner)), dev)
    _check(idx, "idx", torch.int64, (tokens, top_k), dev)
    _check(weights, "weights", torch.bfloat16, (tokens, top_k), dev)
    if out is None:
        out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=dev)
    _check(out, "out", torch.bfloat16, (tokens, hidden), dev)
    if status is not None:
        _check(status, "status", torch.int32, (1,), dev)
    so = native.lib()
    ws = _workspace(so.moe_experts_fp8_workspace_bytes(tokens, count, top_k, hidden, inner), dev)
    with _on(dev):
        native.check(so.moe_experts_fp8(x.data_ptr(), x_scales.data_ptr(), gate_up.data_ptr(),
                                        gate_up_scales.data_ptr(), down.data_ptr(), down_scales.data_ptr(),
                                        idx.data_ptr(), weights.data_ptr(), tokens, count, top_k, hidden, inner,
                                        out.data_ptr(), native._ptr(ws), ws.numel() if ws is not None else 0,
                                        native._ptr(status), native._stream(dev)), "moe_experts_fp8")
    return out
