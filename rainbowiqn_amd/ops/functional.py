"""Autograd wrappers over the HIP kernels (GPU) with torch_ref semantics
(reference: rainbowiqn/agent.py learn() loss math, SURVEY.md section 4.1;
used by the eager-autograd fallback path -- the fast path calls the raw
kernels from runtime/gpu_learner.py instead)."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import get_extension, torch_ref


class _QuantileHuberFn(torch.autograd.Function):
    """Fused n-step target + quantile-Huber loss + grad (kernels K10/K11).

    forward returns (loss, per_sample); backward scales the precomputed
    d(loss)/d(theta) by the incoming scalar gradient.
    """

    @staticmethod
    def forward(ctx, theta, target_q, taus, returns, nonterminals, weights,
                gamma_n: float, kappa: float):
        ext = get_extension()
        B, N = theta.shape
        loss = torch.zeros(1, device=theta.device)
        per_sample = torch.empty(B, device=theta.device)
        grad_theta = torch.empty(B, N, device=theta.device)
        ext.quantile_huber(
            theta.contiguous().float(), target_q.contiguous().float(),
            taus.contiguous().float(), returns.contiguous().float(),
            nonterminals.contiguous().float(),
            None if weights is None else weights.contiguous().float(),
            gamma_n, kappa, loss, per_sample, grad_theta,
        )
        ctx.save_for_backward(grad_theta)
        return loss[0], per_sample

    @staticmethod
    def backward(ctx, grad_loss, _grad_per_sample):
        (grad_theta,) = ctx.saved_tensors
        return grad_theta * grad_loss, None, None, None, None, None, None, None


def quantile_huber_loss_fused(
    theta: torch.Tensor,  # [B, N] online quantiles (requires grad)
    target_q: torch.Tensor,  # [B, Np] target-net quantiles Z'(s', a*)
    taus: torch.Tensor,  # [B, N]
    returns: torch.Tensor,  # [B]
    nonterminals: torch.Tensor,  # [B]
    weights: Optional[torch.Tensor],  # [B]
    discount: float,
    n_step: int,
    kappa: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """GPU: one fused kernel; CPU: torch_ref composition (same semantics)."""
    gamma_n = discount ** n_step
    if theta.is_cuda:
        return _QuantileHuberFn.apply(
            theta, target_q, taus, returns, nonterminals, weights, gamma_n, kappa
        )
    t_theta = torch_ref.n_step_target(target_q, returns, nonterminals, discount, n_step)
    return torch_ref.quantile_huber_loss(theta, t_theta, taus, weights, kappa)


def preprocess_fused(frames_u8: torch.Tensor, out: Optional[torch.Tensor] = None):
    """u8 -> f32/255 (K15)."""
    if frames_u8.is_cuda:
        ext = get_extension()
        if out is None:
            out = torch.empty(frames_u8.shape, dtype=torch.float32,
                              device=frames_u8.device)
        ext.preprocess(frames_u8.contiguous(), out)
        return out
    return torch_ref.preprocess_frames(frames_u8)


# -- layer norm ---------------------------------------------------------------
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis of x [..., C]: (x - mean) / sqrt(var +
    eps) * weight + bias, statistics in fp32, result in x's dtype.

    x: float32, bfloat16 or float16, any strides (rows that are not contiguous
    are copied first); weight and bias [C], contiguous, either or both left
    out, in x's dtype or float32.  Differentiable once in x, weight and bias, in
    reverse mode; forward-mode derivatives on the CPU alone.
    GPU: one kernel forward, two backward, refused under torch.jit.trace, as are
    the operators below; CPU: torch_ref, same semantics.
    """
    if not x.is_cuda:
        _check_norm(x, weight, bias, eps)
        return torch_ref.layer_norm(x, weight, bias, eps)
    return get_extension().layer_norm(x, weight, bias, eps)


# -- 8-bit block matrices -----------------------------------------------------
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class Fp8Blocks(NamedTuple):
    """A matrix [rows, cols] in 8 bits: e4m3 values with one power-of-two scale
    per block of `block_rows` (1 or 128) x 128.

    q      uint8 [rows, 128 nb], nb = ceil(cols / 128): e4m3 bytes; those
           behind column `cols` are zero
    scale  uint8 [ceil(rows / block_rows), nb rounded up to a multiple of 4]:
           the exponents e + 127; a value stands for q 2^e
    """

    q: torch.Tensor
    scale: torch.Tensor
    cols: int
    block_rows: int

    @property
    def shape(self) -> Tuple[int, int]:
        return self.q.shape[0], self.cols


def quantize_fp8_blocks(x: torch.Tensor, block_rows: int = 1) -> Fp8Blocks:
    """x [R, C] in 8 bits: an activation to be kept for a backward pass
    (block_rows=1: rows do not affect each other), or a weight laid out for
    linear_fp8_blocks (block_rows=128).  No gradient flows through it.

    The scale is 2^(floor(log2(amax)) - 7) over a block's finite values, so
    scaling is exact and the values lose only digits past the fourth
    significant bit (a relative error of 2^-4 at most down to 2^-13 of the
    block's largest value).  Values that are not finite become NaN."""
    if not x.is_cuda:
        x = x.detach()
        _check_matrix(x, "x")
        if block_rows not in (1, 128):
            raise RuntimeError("block_rows must be 1 or 128")
        return Fp8Blocks(*torch_ref.quantize_fp8_blocks(x, block_rows),
                         x.shape[1], block_rows)
    if x.dim() == 2 and x.stride(1) != 1:
        x = x.contiguous()
    q, scale = get_extension().fp8_blocks_quant(x, block_rows)
    return Fp8Blocks(q, scale, x.shape[1], block_rows)


def dequantize_fp8_blocks(blocks: Fp8Blocks,
                          dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that `blocks` stands for, [rows, cols] in `dtype`; exact in
    float32 and, but for numbers next to its smallest, in bfloat16."""
    q, scale, cols, block_rows = blocks
    if not q.is_cuda:
        _check_blocks(blocks, "blocks")
        return torch_ref.dequantize_fp8_blocks(q, scale, cols, block_rows, dtype)
    return get_extension().fp8_blocks_dequant(q, scale, cols, block_rows, dtype)


def matmul_fp8_blocks(a: Fp8Blocks, b: Fp8Blocks,
                      bias: Optional[torch.Tensor] = None, relu: bool = False,
                      out_dtype: torch.dtype = torch.bfloat16,
                      exact: bool = True) -> torch.Tensor:
    """a b^T (+ bias, relu): a [M, K], b [N, K], bias [N] -> [M, N].  Exact
    products (of values under 2^-126 what bfloat16 keeps of them), summed in
    fp32, rounded once to `out_dtype`.

    exact=False: results in 16 bits of more than a few rows come from the
    matrix unit's own 8-bit products, up to 1.7 times as fast.  It cuts each to
    a multiple of 2^-13 of the largest of 8 neighbours (by their exponents), so
    a sum is off by up to 7 x 2^-13 of its terms' magnitudes, which is all of it
    where they cancel.  How many rows are a few goes by the sizes.  No
    difference in float32 and on the CPU.

    Has no gradients: a bias that wants one is refused while they are
    recorded."""
    if bias is not None and bias.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("a product of 8-bit blocks has no gradients: pass "
                           "bias.detach(), or train with linear_fp8_blocks")
    if a.cols != b.cols:
        raise RuntimeError(f"a has {a.cols} columns and b {b.cols}")
    if not a.q.is_cuda:
        _check_blocks(a, "a")
        _check_blocks(b, "b")
        _check_bias(bias, b.q.shape[0])
        _check_tangents(bias)
        z = (dequantize_fp8_blocks(a) @ dequantize_fp8_blocks(b).t())
        z = z if bias is None else z + bias.float()
        return (torch.relu(z) if relu else z).to(out_dtype)
    return get_extension().fp8_blocks_matmul(
        a.q, a.scale, a.block_rows, b.q, b.scale, b.block_rows, a.cols, bias,
        relu, out_dtype, exact)


class _LinearFp8CpuFn(torch.autograd.Function):
    """What the extension's linear_fp8 does, in plain PyTorch."""

    @staticmethod
    def forward(ctx, x, weight, bias, relu: bool):
        need = ctx.needs_input_grad
        y, xq, xs, wq, ws, bits = _linear_fwd_cpu(
            _rows(x), weight, bias, relu, need[0], any(need))
        ctx.save_for_backward(xq, xs, wq, ws, bits)
        ctx.shape = x.shape
        ctx.dtypes = (x.dtype, weight.dtype,
                      None if bias is None else bias.dtype)
        # no view: that could not be changed in place
        return torch.ops.aten._unsafe_view(y, [*x.shape[:-1], weight.shape[0]])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        want = [t if n else None
                for t, n in zip(ctx.dtypes, ctx.needs_input_grad)]
        dx, dw, db = _linear_bwd_cpu(_rows(dy), *ctx.saved_tensors,
                                     ctx.shape[-1], *want)
        return None if dx is None else dx.view(ctx.shape), dw, db, None


def linear_fp8_blocks(x: torch.Tensor, weight, bias: Optional[torch.Tensor] = None,
                      relu: bool = False, exact: bool = True) -> torch.Tensor:
    """x W^T + bias (relu): x [..., K], weight [N, K], bias [N] -> [..., N] in
    x's dtype.

    Both operands are taken in 8-bit blocks, x with a scale per 1 x 128 block
    and the weight per 128 x 128.  `weight` is a float matrix, or Fp8Blocks
    that quantize_fp8_blocks(w, 128) laid out once (for serving; no gradients).

    Differentiable once in x, weight and bias, in reverse mode.  For the
    backward pass x is kept in 8 bits only; with g = Q(dz), dz = dy where the
    relu let through:
        dx = g Q(W)    dW = g^T Q(x)    db = sum of dz's rows
    that is, rounding to 8 bits counts as the identity.

    Products of the 8-bit values are exact and summed in fp32, with and without
    gradients alike; `exact=False` makes y and dx by matmul_fp8_blocks' faster
    products, the relu's bits from the same sums."""
    if isinstance(weight, Fp8Blocks):
        if x.dim() > 0 and x.shape[-1] != weight.cols:
            raise RuntimeError(f"x has {x.shape[-1]} columns and weight "
                               f"{weight.cols}")
        if x.is_cuda:
            return get_extension().linear_fp8_serve(
                x, weight.q, weight.scale, weight.block_rows, bias, relu, exact)
        if torch.is_grad_enabled() and (x.requires_grad or (
                bias is not None and bias.requires_grad)):
            raise RuntimeError("a weight in 8-bit blocks is for serving: pass "
                               "the float weight where gradients are wanted")
        _check_tangents(x, bias)
        out = matmul_fp8_blocks(quantize_fp8_blocks(_rows(x)), weight, bias,
                                relu, x.dtype)
        return out.view(*x.shape[:-1], weight.q.shape[0])
    if x.is_cuda:
        return get_extension().linear_fp8(x, weight, bias, relu, exact)
    return _LinearFp8CpuFn.apply(x, weight, bias, relu)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., C] as a matrix of contiguous rows, copied only where it must."""
    if x.dim() != 2:
        if x.dim() == 0:
            raise RuntimeError("a matrix or a vector is wanted, not a number")
        # by the number of rows: C may be 0
        x = x.reshape(x.numel() // max(1, x.shape[-1]), x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] <= 1 else x.contiguous()


# CPU: the semantics of the kernels, in plain PyTorch
def _check_matrix(x, name):
    if x.dim() != 2:
        raise RuntimeError(f"{name} must have 2 dimensions")
    if x.shape[1] < 1:
        raise RuntimeError(f"{name} must have at least one column")
    if x.dtype not in _FLOATS:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got "
                           f"{x.dtype}")


def _check_bias(bias, n):
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != n):
        raise RuntimeError(f"bias must have {n} elements in 1 dimension")


def _check_tangents(*tensors):
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("this operator has no forward-mode derivatives")


def _check_norm(x, weight, bias, eps):
    _check_matrix(_rows(x), "x")
    for t in (weight, bias):
        if t is not None:
            if t.dim() != 1 or t.shape[0] != x.shape[-1]:
                raise RuntimeError("weight and bias must have "
                                   f"{x.shape[-1]} elements in 1 dimension")
            if t.dtype not in (x.dtype, torch.float32):
                raise RuntimeError(
                    "weight and bias must have x's dtype or float32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have one dtype")
    if not eps >= 0:
        raise RuntimeError("eps must not be negative")


def _check_blocks(b: Fp8Blocks, name):
    nb = -(-b.cols // 128)
    if b.block_rows not in (1, 128):
        raise RuntimeError(f"{name}: block_rows must be 1 or 128")
    if b.cols < 1:
        raise RuntimeError(f"{name}: must have 1 to 2^24 columns")
    if b.q.dtype != torch.uint8 or b.scale.dtype != torch.uint8:
        raise RuntimeError(f"{name}: q and scale must be uint8")
    if b.q.dim() != 2 or b.q.shape[1] != nb * 128:
        raise RuntimeError(f"{name}: q must be contiguous [rows, {nb * 128}]")
    want = (-(-b.q.shape[0] // b.block_rows), -(-nb // 4) * 4)
    if tuple(b.scale.shape) != want:
        raise RuntimeError(f"{name}: scale must be contiguous {list(want)}")


def _linear_fwd_cpu(x, w, bias, relu, need_dx, need_bits):
    _check_matrix(x, "x")
    _check_matrix(w, "weight")
    if x.shape[1] != w.shape[1]:
        raise RuntimeError(f"x has {x.shape[1]} columns and weight {w.shape[1]}")
    if w.shape[0] < 1:
        raise RuntimeError("weight must have at least one row")
    _check_bias(bias, w.shape[0])
    xb, wb = quantize_fp8_blocks(x), quantize_fp8_blocks(w, 128)
    z = dequantize_fp8_blocks(xb) @ dequantize_fp8_blocks(wb).t()
    z = z if bias is None else z + bias.float()
    bits = ~(z <= 0) if relu and need_bits else None
    if relu:
        z = torch.relu(z)
    wq = ws = None
    if need_dx:
        wq, ws = torch_ref.quantize_fp8_blocks(
            dequantize_fp8_blocks(wb).t().contiguous(), 128)
    return z.to(x.dtype), xb.q, xb.scale, wq, ws, bits


def _linear_bwd_cpu(dy, xq, xs, wq, ws, bits, cols, dx_type, dw_type, db_type):
    dz = dy.float()
    if bits is not None:
        dz = torch.where(bits, dz, torch.zeros_like(dz))
    g = dequantize_fp8_blocks(quantize_fp8_blocks(dz))
    dx = dw = db = None
    if dx_type is not None:
        w_t = torch_ref.dequantize_fp8_blocks(wq, ws, g.shape[1], 128)
        dx = (g @ w_t.t()).to(dx_type)
    if dw_type is not None:
        x = torch_ref.dequantize_fp8_blocks(xq, xs, cols, 1)
        dw = (g.t() @ x).to(dw_type)
    if db_type is not None:
        db = dz.sum(0).to(db_type)
    return dx, dw, db
