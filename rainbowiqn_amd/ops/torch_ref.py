"""Pure-PyTorch reference implementations of the hot ops.

These define the semantics that the hand-written CDNA4 HIP kernels
(rainbowiqn_amd/ops/csrc) must reproduce; kernel parity tests compare against
these in fp32.  They are also the CPU execution path.
"""

from __future__ import annotations

from typing import Tuple

import torch


def quantile_huber_loss(
    online_quantiles: torch.Tensor,  # [B, N]   theta_i  (requires grad)
    target_quantiles: torch.Tensor,  # [B, N']  T theta_j (no grad)
    taus: torch.Tensor,  # [B, N] quantile fractions of the online samples
    weights: torch.Tensor | None = None,  # [B] PER importance weights
    kappa: float = 1.0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """IQN quantile-Huber loss (Dabney et al. 2018, eq. 3).

    rho_tau(d) = |tau - 1{d<0}| * L_kappa(d) / kappa, d_ij = Ttheta_j - theta_i
    per-sample loss = sum_i mean_j rho ; returns (scalar weighted mean loss,
    per-sample loss detached -- the new PER priorities).

    Reference call site: agent.learn (kernel K11).
    """
    b, n = online_quantiles.shape
    d = target_quantiles.unsqueeze(1) - online_quantiles.unsqueeze(2)  # [B, N, N']
    abs_d = d.abs()
    huber = torch.where(abs_d <= kappa, 0.5 * d * d, kappa * (abs_d - 0.5 * kappa))
    asym = (taus.unsqueeze(2) - (d.detach() < 0).float()).abs()
    rho = asym * huber / kappa
    per_sample = rho.mean(dim=2).sum(dim=1)  # mean over j, sum over i
    if weights is not None:
        loss = (weights * per_sample).mean()
    else:
        loss = per_sample.mean()
    return loss, per_sample.detach()


def n_step_target(
    target_quantiles_next: torch.Tensor,  # [B, N'] Z_tau'(s', a*)
    returns: torch.Tensor,  # [B] n-step discounted returns
    nonterminals: torch.Tensor,  # [B] 1.0 if s' valid
    discount: float,
    n: int,
) -> torch.Tensor:
    """T theta_j = R^(n) + gamma^n * nonterminal * Z_tau'(s', a*)  (kernel K10)."""
    gamma_n = discount ** n
    return returns.unsqueeze(1) + gamma_n * nonterminals.unsqueeze(1) * target_quantiles_next


def preprocess_frames(frames_u8: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """uint8 [.., 84, 84] -> dtype scaled to [0, 1]  (kernel K15)."""
    return frames_u8.to(dtype) / 255.0


def argmax_mean_quantiles(z: torch.Tensor) -> torch.Tensor:
    """z: [B, K, A] -> greedy action per sample  (kernel K9)."""
    return z.mean(dim=1).argmax(dim=1)


# -- 8-bit block matrices and layer norm -------------------------------------
def layer_norm(x, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis, computed in fp32 and rounded once."""
    xf = x.float()
    c = xf - xf.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in fp32 from the exponent field of a double (exact; e >= -127)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64).float()


def quantize_fp8_blocks(x: torch.Tensor, block_rows: int = 1):
    """x [R, C] -> (q, scale) of Fp8Blocks (ops/functional.py).

    Per block of `block_rows` x 128: e = floor(log2(amax)) - 7 over its finite
    values, at least -127, 0 for a block of zeros; q = e4m3(x 2^-e), ties to
    even; values that are not finite become NaN."""
    r, c = x.shape
    t = torch.nn.functional.pad(x.float(), (0, -c % 128, 0, -r % block_rows))
    t = t.reshape(-(-r // block_rows), block_rows, -(-c // 128), 128)
    a = torch.where(torch.isfinite(t), t.abs(), torch.zeros_like(t))
    amax = a.amax(dim=(1, 3), keepdim=True)
    e = torch.clamp((amax.view(torch.int32) >> 23) - 134, min=-127)
    e = torch.where(amax > 0, e, torch.zeros_like(e))
    v = torch.where(torch.isfinite(t), t, torch.full_like(t, float("nan")))
    q = (v * _pow2(-e)).to(torch.float8_e4m3fn).view(torch.uint8)
    q = q.reshape(q.shape[0] * block_rows, q.shape[2] * 128)[:r].contiguous()
    s = (e.reshape(e.shape[0], e.shape[2]) + 127).to(torch.uint8)
    return q, torch.nn.functional.pad(s, (0, -s.shape[1] % 4)).contiguous()


def dequantize_fp8_blocks(q, scale, cols: int, block_rows: int,
                          dtype=torch.float32) -> torch.Tensor:
    e = scale[:, :q.shape[1] // 128].to(torch.int32) - 127
    e = e.repeat_interleave(block_rows, 0)[:q.shape[0]].repeat_interleave(128, 1)
    v = q.view(torch.float8_e4m3fn).float() * _pow2(e)
    return v[:, :cols].to(dtype).contiguous()
