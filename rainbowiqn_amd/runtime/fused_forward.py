"""Fused inference forward for RainbowIQN (MI355X fast path; the model it
reproduces is the reference rainbowiqn/model.py RainbowIQN, SURVEY.md
section 3.1 -- semantics parity-tested against models/model.py).

Binds a bf16 RainbowIQN module to the four hand-written gfx950 kernels in
ops/csrc/model_fwd.hip (fused 3-conv encoder, cos-tau-embed GEMM, concat
noisy-heads GEMM, dueling finish).  One forward = 4 kernel launches instead
of the ~40 eager library launches (MIOpen igemm + NHWC transposes +
hipBLASLt GEMMs + elementwise ReLU/add/mean chains) it replaces.

Weight plumbing (zero repack per step):
  * fc_h_v/fc_h_a ``weight_noisy``/``bias_noisy`` buffers are re-pointed to
    row-slices of ONE concatenated [1024, 3136] buffer, and fc_z_v/fc_z_a
    to slices of a [1+A, 512] buffer, so the per-round noisy_material
    kernels write straight into the GEMM operands;
  * conv1/conv2/iqn weights are read in their natural (flat-param) layout;
  * conv3's 3x3 taps are padded to a 4x4 grid ([64,1024] bf16) by a tiny
    pack kernel -- the only repack, re-run in-graph when weights change.

All methods are hipGraph-capturable: fixed shapes, static scratch buffers
(cached per R), device RNG taus supplied by the caller.
"""

from __future__ import annotations

import os
from typing import Dict, Tuple

import torch

from ..models.model import RainbowIQN
from ..ops import get_extension

# tau_embed variant: -1 = auto (direct accumulator stores at actor-size R,
# LDS-staged rows at learner-size R -- kbench_tau2: 37 -> 28 us at R=8192,
# staged still ahead below R=4096); RIQN_TAU_V2=0/1 forces a variant.
TAU_DIRECT = int(os.environ.get("RIQN_TAU_V2", "-1"))

# RIQN_FUSE_TAU_GEMM=1: route the actor through the single fused
# tau-embed+heads-GEMM kernel (parity-tested, but measured slower -- see
# act_gather; kept as a reachable, gated experiment).
FUSE_TAU_GEMM = os.environ.get("RIQN_FUSE_TAU_GEMM", "0") == "1"

# fp8 path: fuse the MX row quantization into tau_embed's epilogue (the
# bf16 h tensor and the standalone quant pass disappear
# item 4).  RIQN_FP8_FUSE_QUANT=0 falls back to the unfused pair for A/B.
FP8_FUSE_QUANT = os.environ.get("RIQN_FP8_FUSE_QUANT", "1") == "1"


class FusedForward:
    @classmethod
    def for_net(cls, net: RainbowIQN, device,
                fp8_heads: bool = False) -> "FusedForward":
        """One FusedForward per net.  Two instances on one net would each
        re-point weight_noisy to their own concat buffer and the loser's
        GEMM operands would never see another noise reset (colocated
        actor+learner share the online net)."""
        fw = getattr(net, "_fused_forward", None)
        if fw is not None:
            assert fw.fp8_heads == fp8_heads, "fp8 flag mismatch on shared net"
            return fw
        fw = cls(net, device, fp8_heads=fp8_heads)
        net._fused_forward = fw
        return fw

    def __init__(self, net: RainbowIQN, device, fp8_heads: bool = False):
        self.ext = get_extension()
        self.net = net
        self.fp8_heads = fp8_heads
        self.device = torch.device(device)
        p = net.fc_h_v.weight_mu
        assert p.dtype == torch.bfloat16, "fused forward is the bf16 path"
        assert net.feature_norm is None and not net.fp8_train, (
            "fused forward has neither layer norm nor the 8-bit training layer")
        self.A = net.action_space
        d = self.device
        bf = torch.bfloat16

        # concat noisy-weight storage; layer buffers become views into it
        self.wcat = torch.empty(1024, 3136, dtype=bf, device=d)
        self.bcat = torch.empty(1024, dtype=bf, device=d)
        self.wz = torch.empty(1 + self.A, 512, dtype=bf, device=d)
        self.bz = torch.empty(1 + self.A, dtype=bf, device=d)
        slices = [
            (net.fc_h_v, self.wcat[0:512], self.bcat[0:512]),
            (net.fc_h_a, self.wcat[512:1024], self.bcat[512:1024]),
            (net.fc_z_v, self.wz[0:1], self.bz[0:1]),
            (net.fc_z_a, self.wz[1:], self.bz[1:]),
        ]
        for layer, wslice, bslice in slices:
            if getattr(layer, "weight_noisy", None) is None:
                layer.enable_fused_noise()
            with torch.no_grad():
                wslice.copy_(layer.weight_noisy.view(wslice.shape))
                bslice.copy_(layer.bias_noisy.view(bslice.shape))
            layer.weight_noisy = wslice.view(layer.weight_noisy.shape)
            layer.bias_noisy = bslice.view(layer.bias_noisy.shape)

        # raw conv/iqn weights (views into the flat param buffer) ...
        self.w1raw = net.convs[0].weight.detach().view(32, 256)
        self.b1 = net.convs[0].bias.detach()
        self.w2raw = net.convs[2].weight.detach().view(64, 512)
        self.b2 = net.convs[2].bias.detach()
        self.w3raw = net.convs[4].weight.detach().view(64, 576)
        self.b3 = net.convs[4].bias.detach()
        self.wiqnraw = net.iqn_fc.weight.detach()  # [3136, 64]
        self.biqn = net.iqn_fc.bias.detach()
        # ... and their fragment-major packs (one contiguous 1 KB block per
        # MFMA B-fragment load -- see pack_fwd_frag_kernel)
        self.w1 = torch.empty(16 * 512, dtype=bf, device=d)
        self.w2 = torch.empty(64 * 512, dtype=bf, device=d)
        self.w3p = torch.empty(128 * 512, dtype=bf, device=d)
        self.wiqn = torch.empty(392 * 512, dtype=bf, device=d)
        # fp8 MX heads path: e4m3 + e8m0 block scales
        if fp8_heads:
            self.wq = torch.empty(1024, 3200, dtype=torch.uint8, device=d)
            self.wsc = torch.empty(1024, 100, dtype=torch.uint8, device=d)
        self.pack_weights()

        self._scratch: Dict[Tuple[int, int], tuple] = {}

    def pack_weights(self) -> None:
        """Refresh the fragment-major weight packs (call after weight
        changes; graph-capturable)."""
        self.ext.pack_fwd_frag(self.w1raw, self.w2raw, self.w3raw,
                               self.wiqnraw, self.w1, self.w2, self.w3p,
                               self.wiqn)
        if self.fp8_heads:
            self.ext.quant_fp8(self.wcat, self.wq, self.wsc)

    def _bufs(self, B: int, nq: int):
        key = (B, nq)
        if key not in self._scratch:
            d, bf = self.device, torch.bfloat16
            R = B * nq
            extra = ()
            if self.fp8_heads:
                # zeros, not empty: the fused tau-quant kernel writes only
                # k < 3136; the padding bytes/scales must stay zero
                extra = (torch.zeros(R, 3200, dtype=torch.uint8, device=d),
                         torch.zeros(R, 100, dtype=torch.uint8, device=d))
            self._scratch[key] = (
                torch.empty(B, 3136, dtype=bf, device=d),     # feat
                torch.empty(R, 3136, dtype=bf, device=d),     # h
                torch.empty(R, 1024, dtype=bf, device=d),     # hh
            ) + extra
        return self._scratch[key]

    def encode(self, x: torch.Tensor) -> torch.Tensor:
        """Conv trunk only: x [B,4,84,84] bf16 -> features [B,3136] bf16."""
        feat, _, _ = self._bufs(x.shape[0], 1)
        self.ext.conv_encode(x, self.w1, self.b1, self.w2, self.b2, self.w3p,
                             self.b3, feat)
        return feat

    def _trunk(self, x: torch.Tensor, taus: torch.Tensor, nq: int):
        """x [B,4,84,84] bf16, taus [B*nq] f32 -> hh [B*nq, 1024]."""
        B = x.shape[0]
        bufs = self._bufs(B, nq)
        feat, h, hh = bufs[:3]
        self.ext.conv_encode(x, self.w1, self.b1, self.w2, self.b2, self.w3p,
                             self.b3, feat)
        if self.fp8_heads:
            self._tau_heads_fp8(feat, taus, nq, bufs, hh)
        else:
            self.ext.tau_embed(taus.view(-1), self.wiqn, self.biqn, feat, h,
                               nq, direct=TAU_DIRECT)
            self.ext.heads_gemm(h, self.wcat, self.bcat, hh)
        return hh

    def _tau_heads_fp8(self, feat, taus, nq, bufs, hh):
        """tau-embed -> MX-fp8 heads GEMM with the row quantization fused
        into tau-embed's stores (h never exists in bf16 on this path).

        Small R falls back to the bf16 pair: below ~2048 rows the fp8
        GEMM's grid can't fill the chip and loses to bf16 (kbench r02:
        R=256 fp8 ~30 us vs bf16 16.5), and the learner's target forward
        (R = B*N' = 256) sits on the critical path 8x per round."""
        R = hh.shape[0] if hh.dim() == 2 else taus.numel()
        if R < 2048:
            h = bufs[1]
            self.ext.tau_embed(taus.view(-1), self.wiqn, self.biqn, feat, h,
                               nq, direct=TAU_DIRECT)
            self.ext.heads_gemm(h, self.wcat, self.bcat, hh)
            return hh
        hq, hsc = bufs[3], bufs[4]
        if FP8_FUSE_QUANT:
            self.ext.tau_embed_fp8(taus.view(-1), self.wiqn, self.biqn,
                                   feat, hq, hsc, nq)
        else:
            h = bufs[1]
            self.ext.tau_embed(taus.view(-1), self.wiqn, self.biqn, feat, h,
                               nq, direct=TAU_DIRECT)
            self.ext.quant_fp8(h, hq, hsc)
        self.ext.heads_gemm_fp8(hq, hsc, self.wq, self.wsc, self.bcat, hh)
        return hh

    def quantiles(self, x, taus, nq: int, out: torch.Tensor) -> torch.Tensor:
        """Full forward -> quantile values out [B, nq, A] (f32)."""
        hh = self._trunk(x, taus, nq)
        dummy = torch.zeros(1, dtype=torch.int64, device=self.device)
        self.ext.heads_finish(hh, self.wz, self.bz, self.A, nq, 0,
                              out.view(-1, self.A), dummy)
        return out

    def act(self, x, taus, nq: int, actions: torch.Tensor) -> torch.Tensor:
        """argmax_a mean_k Z_tau_k(x, a) -> actions [B] (K9 fused)."""
        hh = self._trunk(x, taus, nq)
        dummy = torch.zeros(1, dtype=torch.float32, device=self.device)
        self.ext.heads_finish(hh, self.wz, self.bz, self.A, nq, 1, dummy,
                              actions)
        return actions

    def act_gather(self, ring: torch.Tensor, env_state: torch.Tensor,
                   history: int, ring_head: int, taus, nq: int,
                   actions: torch.Tensor) -> torch.Tensor:
        """Greedy action straight from the u8 frame ring: conv1 gathers and
        normalizes the frame stack itself (fused K15), so the bf16 stack
        tensor never materializes (actor hot path)."""
        E = env_state.numel() // 4
        bufs = self._bufs(E, nq)
        feat, h, hh = bufs[:3]
        self.ext.conv_encode_gather(ring, env_state, history, ring_head,
                                    self.w1, self.b1, self.w2, self.b2,
                                    self.w3p, self.b3, feat)
        if self.fp8_heads:
            self._tau_heads_fp8(feat, taus, nq, bufs, hh)
        elif FUSE_TAU_GEMM:
            # experiment (off by default): tau-embed fused into the GEMM's
            # A-operand production.  Bit-identical to the pair but measured
            # SLOWER end-to-end (10.6 vs 6.3 ms/round at the bench config:
            # the scattered feat loads + A-image LDS writes stall the main
            # MFMA chain harder than the h round-trip costs).
            self.ext.heads_gemm_tau(taus.view(-1), self.wiqn, self.biqn,
                                    feat, self.wcat, self.bcat, hh, nq)
        else:
            self.ext.tau_embed(taus.view(-1), self.wiqn, self.biqn, feat, h,
                               nq, direct=TAU_DIRECT)
            self.ext.heads_gemm(h, self.wcat, self.bcat, hh)
        dummy = torch.zeros(1, dtype=torch.float32, device=self.device)
        self.ext.heads_finish(hh, self.wz, self.bz, self.A, nq, 1, dummy,
                              actions)
        return actions

    def act_from_feat(self, featv: torch.Tensor, taus, nq: int,
                      actions: torch.Tensor) -> torch.Tensor:
        """Greedy action from precomputed conv features (lets the learner
        batch s and s' through one conv_encode call)."""
        B = featv.shape[0]
        _, h, hh = self._bufs(B, nq)[:3]
        self.ext.tau_embed(taus.view(-1), self.wiqn, self.biqn,
                           featv.contiguous(), h, nq, direct=TAU_DIRECT)
        self.ext.heads_gemm(h, self.wcat, self.bcat, hh)
        dummy = torch.zeros(1, dtype=torch.float32, device=self.device)
        self.ext.heads_finish(hh, self.wz, self.bz, self.A, nq, 1, dummy,
                              actions)
        return actions

    def theta(self, x, taus, nq: int, actions: torch.Tensor,
              out: torch.Tensor) -> torch.Tensor:
        """Z_tau(x, actions[b]) -> out [B, nq] (target-net path, K10 feed)."""
        hh = self._trunk(x, taus, nq)
        self.ext.heads_finish(hh, self.wz, self.bz, self.A, nq, 2,
                              out.view(-1), actions)
        return out


def noisy_pack(net: RainbowIQN, device) -> list:
    """Tensor list for ext.noisy_material4: regenerates noise + materialized
    noisy weights for all four NoisyLinear layers in 2 kernels (vs 8).
    Build AFTER FusedForward so weight_noisy points at the concat storage."""
    ts = []
    for layer in (net.fc_h_v, net.fc_h_a, net.fc_z_v, net.fc_z_a):
        if getattr(layer, "weight_noisy", None) is None:
            layer.enable_fused_noise()
        eps_in = torch.empty(layer.in_features, device=device)
        eps_out = torch.empty(layer.out_features, device=device)
        ts += [layer.weight_mu.detach(), layer.weight_sigma.detach(),
               layer.bias_mu.detach(), layer.bias_sigma.detach(),
               layer.weight_epsilon, layer.bias_epsilon,
               layer.weight_noisy, layer.bias_noisy, eps_in, eps_out]
    return ts
