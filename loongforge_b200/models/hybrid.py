"""Hybrid-attention layers of Qwen3-Next / Qwen3.5: output-gated softmax attention and GatedDeltaNet
linear attention, mixed by ``cfg.layer_types``.

* ``GatedAttention``: the query projection is twice as wide; the second half is a per-element gate,
  ``out = attn(q, k, v) * sigmoid(gate)`` before the output projection; per-head QK RMSNorm
  (zero-centred weight), partial rotary (reference: loongforge/models/foundation/qwen3_next/gated_attention.py:53-).
* ``GatedDeltaNet``: in-projections to (q, k, v, z) and (b, a); depthwise causal conv + SiLU over
  q|k|v; ``beta = sigmoid(b)``, log-decay ``g = -exp(A_log) * softplus(a + dt_bias)``; gated delta rule;
  RMSNorm gated by ``silu(z)``; out-projection (reference: .../qwen3_next/gated_deltanet.py:129-420).
  Heads are split over tensor parallel ranks (value heads, with their share of key heads).
"""
from __future__ import annotations

import math
import zlib
from operator import index
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..ops import functional as OF
from ..ops import linear_attn as LA
from ..parallel import layers as PL
from ..parallel import state as ps
from .config import TransformerConfig
from .transformer import Norm, PackedSeqParams, RotaryInputs, core_attention, fused_qk, fused_qk_applies


class GatedAttention(nn.Module):
    def __init__(self, cfg: TransformerConfig, key: str, *, device=None, parallel_state=None):
        super().__init__()
        st = ps.get_state(parallel_state)
        tp = st.dims.tp
        self.cfg, self.d = cfg, cfg.kv_channels
        self.nq, self.ng = cfg.num_attention_heads, cfg.num_query_groups
        assert self.nq % tp == 0 and self.ng % tp == 0
        self.nq_l, self.ng_l = self.nq // tp, self.ng // tp
        common = dict(sequence_parallel=cfg.sequence_parallel, params_dtype=cfg.params_dtype, device=device,
                      parallel_state=parallel_state)
        # per query group: [q heads | gate heads | k | v], so a TP shard keeps whole groups
        self.r = self.nq // self.ng
        out = (2 * self.nq + 2 * self.ng) * self.d
        self.linear_qgkv = PL.ColumnParallelLinear(cfg.hidden_size, out, bias=False, init_std=cfg.init_method_std,
                                                   key=key + ".linear_qgkv", **common)
        self.q_layernorm = Norm(self.d, cfg, device=device)
        self.k_layernorm = Norm(self.d, cfg, device=device)
        if tp > 1:
            PL.mark_tp_partial_grad(self.q_layernorm)
            PL.mark_tp_partial_grad(self.k_layernorm)
        self.linear_proj = PL.RowParallelLinear(self.nq * self.d, cfg.hidden_size, bias=False,
                                                init_std=cfg.init_method_std / math.sqrt(2.0 * cfg.num_layers),
                                                key=key + ".linear_proj", **common)
        self.scale = cfg.attention_softmax_scale or 1.0 / math.sqrt(self.d)
        self.rot_dim = int(self.d * cfg.rotary_percent)

    def forward(self, x, rotary: Optional[RotaryInputs], packed: Optional[PackedSeqParams], residual=None):
        y = self.linear_qgkv(x)
        T = y.shape[0]
        cu = packed.cu_seqlens if packed is not None else None
        row_length = packed.row_length if packed is not None else None
        if fused_qk_applies(self, y, self.ng_l, self.r, rotary, gated=True):
            q, k, v, gate = fused_qk(self, y, self.ng_l, self.r, rotary, gated=True)
            o = core_attention(q, k, v, causal=True, scale=self.scale, cu_seqlens=cu, cfg=self.cfg, row_length=row_length)
            o = o.view(T, self.ng_l, self.r, self.d) * torch.sigmoid(gate.float()).to(o.dtype)
            return self.linear_proj(o.reshape(T, self.nq_l * self.d), residual)
        y = y.view(T, self.ng_l, 2 * self.r + 2, self.d)
        q = self.q_layernorm(y[:, :, :self.r].reshape(T, self.nq_l, self.d))
        gate = y[:, :, self.r:2 * self.r].reshape(T, self.nq_l * self.d)
        k = self.k_layernorm(y[:, :, 2 * self.r].contiguous())
        v = y[:, :, 2 * self.r + 1]
        if rotary is not None:
            kw = dict(pos_ids=rotary.pos_ids, rot_dim=self.rot_dim, interleaved=self.cfg.rotary_interleaved,
                      mscale=rotary.mscale)
            f = rotary.freqs
            if f.dim() == 3:
                f, kw = f[:, 0], {**kw, "pos_ids": None, "interleaved": False}
            q, k = OF.rope(q, f, **kw), OF.rope(k, f, **kw)
        o = core_attention(q, k, v, causal=True, scale=self.scale, cu_seqlens=cu, cfg=self.cfg, row_length=row_length)
        o = o.reshape(T, self.nq_l * self.d) * torch.sigmoid(gate.float()).to(o.dtype)
        return self.linear_proj(o, residual)


class GatedRMSNorm(nn.Module):
    """y = rmsnorm(x) * w * silu(z), over the value head dim."""

    def __init__(self, dim: int, eps: float, device=None, dtype=torch.float32):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.eps = eps

    def forward(self, x, z):
        xf = x.float()
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight.float()
        return (y * F.silu(z.float())).to(x.dtype)


class GatedDeltaNet(nn.Module):
    def __init__(self, cfg: TransformerConfig, key: str, *, device=None, parallel_state=None):
        super().__init__()
        st = ps.get_state(parallel_state)
        self.cp = st.dims.cp  # > 1: convolution and recurrence run on the gathered sequence (see forward)
        tp = st.dims.tp
        self.cfg = cfg
        self.dk, self.dv = cfg.linear_key_head_dim, cfg.linear_value_head_dim
        self.hk, self.hv = cfg.linear_num_key_heads, cfg.linear_num_value_heads
        assert self.hk % tp == 0 and self.hv % self.hk == 0
        self.hk_l, self.hv_l = self.hk // tp, self.hv // tp
        self.ratio = self.hv // self.hk
        self.K = cfg.linear_conv_kernel_dim
        common = dict(sequence_parallel=cfg.sequence_parallel, params_dtype=cfg.params_dtype, device=device,
                      parallel_state=parallel_state)
        # per key head: [q | k | v (ratio heads) | z (ratio heads)] and [b (ratio) | a (ratio)]
        per_head = 2 * self.dk + 2 * self.ratio * self.dv
        self.in_proj_qkvz = PL.ColumnParallelLinear(cfg.hidden_size, self.hk * per_head, bias=False,
                                                    init_std=cfg.init_method_std, key=key + ".in_proj_qkvz", **common)
        self.in_proj_ba = PL.ColumnParallelLinear(cfg.hidden_size, self.hk * 2 * self.ratio, bias=False,
                                                  init_std=cfg.init_method_std, key=key + ".in_proj_ba", **common)
        # The FULL parameters are drawn from a seed that depends only on the key, then sliced to this rank's heads, so
        # that every tensor-parallel layout starts from the same model. Conv channels are laid out type-major
        # [q heads | k heads | v heads]; a rank keeps its head range of each type.
        g = torch.Generator().manual_seed(zlib.crc32((key + ".conv1d").encode()) & 0x7FFFFFFF)
        full_conv = (torch.rand(self.hk * (2 * self.dk + self.ratio * self.dv), self.K, generator=g) * 2 - 1) * self.K ** -0.5
        qf, kf, vf = full_conv.split([self.hk * self.dk, self.hk * self.dk, self.hv * self.dv], dim=0)
        r0 = st.tp_rank
        local = torch.cat([qf.view(self.hk, self.dk, -1)[r0 * self.hk_l:(r0 + 1) * self.hk_l].reshape(-1, self.K),
                           kf.view(self.hk, self.dk, -1)[r0 * self.hk_l:(r0 + 1) * self.hk_l].reshape(-1, self.K),
                           vf.view(self.hv, self.dv, -1)[r0 * self.hv_l:(r0 + 1) * self.hv_l].reshape(-1, self.K)], 0)
        self.conv_weight = nn.Parameter(local.to(device=device, dtype=cfg.params_dtype))
        self.dt_bias = nn.Parameter(torch.ones(self.hv_l, device=device))
        A = torch.empty(self.hv).uniform_(1e-3, 16.0, generator=g)[r0 * self.hv_l:(r0 + 1) * self.hv_l]
        self.A_log = nn.Parameter(torch.log(A).to(device=device))
        for p in (self.conv_weight, self.dt_bias, self.A_log):
            PL.mark_tp(p, 0 if tp > 1 else None)
        self.out_norm = GatedRMSNorm(self.dv, cfg.layernorm_epsilon, device=device)
        PL.mark_tp(self.out_norm.weight, None)
        if tp > 1:
            PL.mark_tp_partial_grad(self.out_norm)
        self.out_proj = PL.RowParallelLinear(self.hv * self.dv, cfg.hidden_size, bias=False,
                                             init_std=cfg.init_method_std / math.sqrt(2.0 * cfg.num_layers),
                                             key=key + ".out_proj", **common)

    def _project(self, x):
        """(q | k | v convolution channels [T, C], z [T, hv, dv], b [T, hv], a [T, hv]) of this rank's heads."""
        hk, r, dk, dv = self.hk_l, self.ratio, self.dk, self.dv
        qkvz = self.in_proj_qkvz(x)
        T = qkvz.shape[0]
        q, k, v, z = qkvz.view(T, hk, 2 * dk + 2 * r * dv).split([dk, dk, r * dv, r * dv], dim=-1)
        b, a = self.in_proj_ba(x).view(T, hk, 2 * r).split([r, r], dim=-1)
        # conv over [q | k | v] channels, laid out type-major like the conv weight
        mixed = torch.cat([q.reshape(T, -1), k.reshape(T, -1), v.reshape(T, -1)], dim=-1)
        return mixed, z.reshape(T, hk * r, dv), b.reshape(T, -1), a.reshape(T, -1)

    def _heads(self, mixed):
        hk, r, dk, dv = self.hk_l, self.ratio, self.dk, self.dv
        T = mixed.shape[0]
        q, k, v = mixed.split([hk * dk, hk * dk, hk * r * dv], dim=-1)
        return q.view(T, hk, dk), k.view(T, hk, dk), v.view(T, hk * r, dv)

    def _gates(self, b, a):
        beta = torch.sigmoid(b.float())
        return -self.A_log.float().exp() * F.softplus(a.float() + self.dt_bias.float()), beta

    def _finish(self, o, z, residual):
        o = self.out_norm(o, z)
        return self.out_proj(o.reshape(o.shape[0], -1), residual)

    def forward(self, x, rotary=None, packed: Optional[PackedSeqParams] = None, residual=None):
        mixed, z, b, a = self._project(x)
        cu = packed.cu_seqlens if packed is not None else None
        own = None
        if self.cp > 1:
            # The convolution window and the recurrent state cross the chunk boundaries of context parallelism: run
            # both on the gathered sequence (token-wise projections stay local) and keep this rank's outputs.
            from ..parallel.context_parallel import gather_full_sequence
            (mixed, b, a), own = gather_full_sequence([mixed, b, a], packed.row_length if packed is not None else None)
        mixed = LA.causal_conv1d(mixed, self.conv_weight, cu_seqlens=cu, activation="silu")
        o = LA.gated_delta_rule(*self._heads(mixed), *self._gates(b, a), cu_seqlens=cu, qk_l2norm=True)
        if own is not None:
            o = o.index_select(0, own)
        return self._finish(o, z, residual)

    # ------------------------------------------------------------------ decoding
    def new_cache(self, slots: int, device=None):
        """(convolution windows [slots, C, K - 1], states [slots, hv, dk, dv] fp32) for `slots` sequences without tokens."""
        device = self.conv_weight.device if device is None else device
        return (torch.zeros(slots, self.conv_weight.shape[0], self.K - 1, dtype=self.conv_weight.dtype, device=device),
                torch.zeros(slots, self.hv_l, self.dk, self.dv, device=device))

    def _check_decoding(self):
        if self.cp > 1 or (self.cfg.sequence_parallel and ps.get_state().dims.tp > 1):
            raise ValueError("decoding runs without context or sequence parallelism: every rank sees all rows")

    @torch.no_grad()
    def prefill(self, x, cache, slots, *, cu_seqlens=None, residual=None):
        """`forward` over new sequences, one per entry of `slots` (bounds in `cu_seqlens`; None = one sequence); leaves
        their windows and states in those slots of `cache`. The slots are read on the host: they must differ and exist.
        Every sequence begins here: what a slot holds is replaced, not continued. A later part of a sequence goes through
        `step`, token by token."""
        self._check_decoding()
        windows, states = cache
        slots = [index(i) for i in (slots.tolist() if torch.is_tensor(slots) else slots)]
        n = 1 if cu_seqlens is None else len(cu_seqlens) - 1
        if len(slots) != n:
            raise ValueError(f"{n} sequences need as many slots, got {len(slots)}")
        if len(set(slots)) < n or any(i < 0 or i >= states.shape[0] for i in slots):
            raise ValueError(f"slots must be {n} different ones of the cache's {states.shape[0]}, got {slots[:8]}")
        mixed, z, b, a = self._project(x)
        y = LA.causal_conv1d(mixed, self.conv_weight, cu_seqlens=cu_seqlens, activation="silu")
        o, last = LA.gated_delta_rule(*self._heads(y), *self._gates(b, a), cu_seqlens=cu_seqlens, qk_l2norm=True,
                                      output_final_state=True)
        slots = torch.tensor(slots, dtype=torch.long, device=x.device)
        cu = torch.tensor([0, mixed.shape[0]]) if cu_seqlens is None else torch.as_tensor(cu_seqlens)
        cu = cu.to(device=x.device, dtype=torch.long)
        at = cu[1:, None] - torch.arange(self.K - 1, 0, -1, device=x.device)  # the last K - 1 tokens, oldest first
        inside = at >= cu[:-1, None]
        rows = mixed[at.clamp(min=0, max=max(mixed.shape[0] - 1, 0))] if mixed.shape[0] else mixed.new_zeros(*at.shape, mixed.shape[1])
        windows[slots] = torch.where(inside[..., None], rows, torch.zeros_like(rows)).transpose(1, 2).to(windows.dtype)
        states[slots] = last
        return self._finish(o, z, residual)

    @torch.no_grad()
    def step(self, x, cache, *, slots=None, residual=None):
        """One token of every row of x [B, hidden]: row b continues the sequence in slot ``slots[b]`` of `cache` (its own
        number without `slots`; negative = padding row), which is updated in place."""
        self._check_decoding()
        windows, states = cache
        mixed, z, b, a = self._project(x)
        y = LA.causal_conv1d_step(mixed, windows, self.conv_weight, state_indices=slots, activation="silu")
        o = LA.gated_delta_rule_step(*self._heads(y), *self._gates(b, a), states, state_indices=slots, qk_l2norm=True)
        return self._finish(o, z, residual)
