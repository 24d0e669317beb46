"""Gated delta rule (linear attention of Qwen3-Next / Qwen3.5) and the depthwise causal conv in front of it.

Per head, with state ``S [dk, dv]``, decay ``a_t = exp(g_t)`` and write strength ``beta_t``::

    S   <- a_t * S
    d_t  = beta_t * (v_t - S^T k_t)
    S   <- S + k_t d_t^T
    o_t  = S^T q_t

``gated_delta_rule_recurrent`` is that recurrence literally (the oracle); ``gated_delta_rule`` is the
chunk-parallel form (WY representation inside a chunk, one state update per chunk), forward and backward, and
``gated_delta_rule_step`` advances a pool of states by one token per row (decoding). ``causal_conv1d`` /
``causal_conv1d_step`` are the same pair for the convolution. The reference calls library kernels here
(loongforge/models/foundation/qwen3_next/gated_deltanet.py:49-52,354).

On a GPU bf16 inputs run on the kernels of ``csrc/gated_delta_sm100.cu``, ``csrc/gated_delta_step.cu`` and
``csrc/causal_conv.cu``: they read ``cu_seqlens`` on the device (no host synchronisation; capturable into a CUDA
graph) and take fewer key heads than value heads as they are. Their gradients can be taken once: a second derivative
raises, and forward-mode derivatives and ``vmap`` are refused. Other devices, dtypes and head dims take the PyTorch
formulation below, which is also what the kernels are tested against, and which has all of these.
"""
from __future__ import annotations

from operator import index
from typing import Optional

import torch
import torch.nn.functional as F

from . import _ext
from .functional import first_order


def l2norm(x: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    return x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) + eps)


def _share_heads(q, k, hv: int):
    """Key heads serve ``hv / hk`` neighbouring value heads each."""
    hk = q.shape[-2]
    if hk == hv:
        return q, k
    if hk == 0 or hv % hk:
        raise ValueError(f"{hv} value heads are not a multiple of {hk} key heads")
    return q.repeat_interleave(hv // hk, -2), k.repeat_interleave(hv // hk, -2)


def gated_delta_rule_recurrent(q, k, v, g, beta, *, scale: Optional[float] = None, qk_l2norm: bool = True):
    """q, k [T, H, dk] (or fewer key heads than v has); v [T, H, dv]; g, beta [T, H]. Returns o [T, H, dv] (fp32 math)."""
    T, _, dk = q.shape
    H, dv = v.shape[1:]
    q, k, v, g, beta = (t.float() for t in (q, k, v, g, beta))
    if qk_l2norm:
        q, k = l2norm(q), l2norm(k)
    q = q * (scale if scale is not None else dk ** -0.5)
    q, k = _share_heads(q, k, H)
    S = q.new_zeros(H, dk, dv)
    out = []
    for t in range(T):
        S = S * g[t].exp()[:, None, None]
        mem = torch.einsum("hkv,hk->hv", S, k[t])
        d = (v[t] - mem) * beta[t][:, None]
        S = S + k[t][:, :, None] * d[:, None, :]
        out.append(torch.einsum("hkv,hk->hv", S, q[t]))
    return torch.stack(out, 0)


def _chunk_one(q, k, v, g, beta, chunk: int, state=None):
    """One sequence, tensors already head-major: q, k [H, T, dk]; v [H, T, dv]; g, beta [H, T]; state [H, dk, dv] or
    None (zero). Returns (o [H, T, dv], state behind the last token)."""
    H, T, dk = q.shape
    dv = v.shape[-1]
    pad = (-T) % chunk
    if pad:
        q, k, v = (F.pad(t, (0, 0, 0, pad)) for t in (q, k, v))
        g, beta = F.pad(g, (0, pad)), F.pad(beta, (0, pad))
    n = (T + pad) // chunk
    q, k, v = (t.reshape(H, n, chunk, -1) for t in (q, k, v))
    g, beta = g.reshape(H, n, chunk), beta.reshape(H, n, chunk)
    gc = g.cumsum(-1)
    k_beta, v_beta = k * beta[..., None], v * beta[..., None]
    tri = torch.tril(torch.ones(chunk, chunk, dtype=torch.bool, device=q.device))
    strict = torch.tril(torch.ones(chunk, chunk, dtype=torch.bool, device=q.device), -1)
    decay = (gc[..., :, None] - gc[..., None, :]).masked_fill(~tri, float("-inf")).exp()
    L = (k_beta @ k.transpose(-1, -2) * decay).masked_fill(~strict, 0.0)
    eye = torch.eye(chunk, dtype=L.dtype, device=L.device)
    # WY representation of the chunk: (I + L)^-1, unit lower triangular
    A = torch.linalg.solve_triangular(L + eye, eye.expand_as(L), upper=False, unitriangular=True)
    value = A @ v_beta
    k_cum = A @ (k_beta * gc.exp()[..., None])
    S = q.new_zeros(H, dk, dv) if state is None else state
    outs = []
    for c in range(n):
        qc, kc, gcc = q[:, c], k[:, c], gc[:, c]
        local = (qc @ kc.transpose(-1, -2) * decay[:, c]).masked_fill(~tri, 0.0)
        v_new = value[:, c] - k_cum[:, c] @ S
        inter = (qc * gcc.exp()[..., None]) @ S
        outs.append(inter + local @ v_new)
        last = gcc[:, -1]
        S = S * last.exp()[:, None, None] + (kc * (last[:, None] - gcc).exp()[..., None]).transpose(-1, -2) @ v_new
    o = torch.stack(outs, 1).reshape(H, n * chunk, dv)
    return o[:, :T], S


class _GatedDeltaFn(torch.autograd.Function):
    """The chunked kernels. Kept for the backward pass: U and the memory read at each token (both with the remainder of
    their bf16 rounding), the part of o that earlier tokens wrote, the state in front of every chunk and the chunk's
    tiles and 64 x 64 matrices."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, s_in, cu, scale, l2norm, want_state, keep):
        ctx.set_materialize_grads(False)
        C, status = _ext.require(), _status(v)
        inputs = (q, k, v, g, beta, s_in)
        q, k, v, gf, bf = _rows16(q), _rows16(k), _rows16(v), _fp32(g), _fp32(beta)
        # what has a gradient and is not saved as it is below: see first_order
        inputs = tuple(t if need and t is not x else None for t, x, need in zip(inputs, (q, k, v, gf, bf, None), ctx.needs_input_grad))
        bounds, first = (None, None) if cu is None else C.delta_plan(cu, q.shape[0], status)
        o, s_out, kept = C.delta_fwd(q, k, v, gf, bf, bounds, first, scale, l2norm, s_in, want_state, keep, status)
        if keep:
            ctx.save_for_backward(*inputs, q, k, v, gf, bf, bounds, first, kept)
            ctx.cfg = (scale, l2norm, g.dtype, beta.dtype)
        if not want_state:
            ctx.mark_non_differentiable(s_out)
        return o, s_out

    @staticmethod
    def backward(ctx, do, ds_out):
        scale, l2norm, g_dtype, beta_dtype = ctx.cfg
        inputs, (q, k, v, g, beta, bounds, first, kept) = ctx.saved_tensors[:6], ctx.saved_tensors[6:]
        want_ds = ctx.needs_input_grad[5]
        up = (do, ds_out)
        do = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if do is None else _rows16(do.contiguous())
        dq, dk, dv, dg, dbeta, ds_in = _ext.require().delta_bwd(
            do, None if ds_out is None else _dense16(ds_out), q, k, v, g, beta, bounds, first, scale, l2norm, want_ds, kept,
            _status(v))
        grads = (dq, dk, dv, dg.to(g_dtype), dbeta.to(beta_dtype), ds_in if want_ds else None)
        return first_order("gated_delta_rule", grads, *up, *inputs, q, k, v) + (None,) * 5


def _status(t: torch.Tensor) -> torch.Tensor:
    s = _ext._status.get(t.get_device())
    return s if s is not None else _ext.status_tensor(t.device)


def _fp32(t: torch.Tensor) -> torch.Tensor:
    return t.detach().float().contiguous()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself when its rows are unit-stride and 16-byte aligned (what the kernels read), else a copy. A dimension
    of one element may have any stride in a contiguous tensor: the strides themselves are looked at."""
    s = t.stride()
    if s[-1] == 1 and not (s[0] | s[-2]) & 7 and t.data_ptr() % 16 == 0:  # two or three dimensions
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _dense16(t: torch.Tensor) -> torch.Tensor:
    """Contiguous with a 16-byte aligned base."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def gated_delta_rule_native(q, k, v) -> bool:
    """Whether the sm_100a kernels cover these inputs: bf16 on a GPU, head dims 64 or 128."""
    return (v.is_cuda and q.dtype == k.dtype == v.dtype == torch.bfloat16 and q.shape[-1] in (64, 128)
            and v.shape[-1] in (64, 128))


def _check_delta(q, k, v, g, beta, rows: str):
    qs, vs = q.shape, v.shape
    if len(qs) != 3 or k.shape != qs or len(vs) != 3 or vs[0] != qs[0]:
        raise ValueError(f"q, k [{rows}, key heads, dk] and v [{rows}, value heads, dv] expected, got {tuple(qs)}, "
                         f"{tuple(k.shape)}, {tuple(vs)}")
    if g.shape != vs[:2] or beta.shape != vs[:2]:
        raise ValueError(f"g and beta [{rows}, value heads] expected, got {tuple(g.shape)}, {tuple(beta.shape)}")
    if qs[1] == 0 or vs[1] % qs[1]:
        raise ValueError(f"{vs[1]} value heads are not a multiple of {qs[1]} key heads")
    dev = v.device
    if q.device != dev or k.device != dev or g.device != dev or beta.device != dev:
        raise ValueError("q, k, v, g and beta must be on one device")


def _whole(t, name: str):
    if torch.is_tensor(t) and (t.is_floating_point() or t.is_complex()):
        raise ValueError(f"{name} must be whole numbers, got {t.dtype}")


def _host_bounds(cu_seqlens, T: int) -> list:
    """Sequence boundaries as a list; every one of them inside [0, T] and none in front of the one before it."""
    if cu_seqlens is None:
        return [0, T]
    _whole(cu_seqlens, "cu_seqlens")
    b = [index(x) for x in (cu_seqlens.tolist() if torch.is_tensor(cu_seqlens) else cu_seqlens)]
    if len(b) < 2 or b[0] < 0 or b[-1] > T or any(e < s for s, e in zip(b, b[1:])):
        raise ValueError(f"cu_seqlens must be at least two non-decreasing offsets within the {T} rows, got {b[:8]}...")
    return b


def _int32(t: torch.Tensor, device) -> torch.Tensor:
    """Numbers as int32 on `device`; one that does not fit stays out of range instead of wrapping into it."""
    if t.dtype == torch.int64:
        t = t.clamp(-2 ** 31, 2 ** 31 - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def _device_bounds(cu_seqlens, T: int, device) -> Optional[torch.Tensor]:
    """Sequence boundaries as int32 on `device`. Boundaries that are on the host are checked here; those on the device
    are clamped by the kernels (the delta rule also reports a bad one through the status word)."""
    if cu_seqlens is None:
        return None
    if not torch.is_tensor(cu_seqlens) or not cu_seqlens.is_cuda:
        return torch.tensor(_host_bounds(cu_seqlens, T), dtype=torch.int32, device=device)
    _whole(cu_seqlens, "cu_seqlens")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2:
        raise ValueError("cu_seqlens must hold at least two offsets")
    if cu_seqlens.dtype == torch.int32 and cu_seqlens.device == device and cu_seqlens.is_contiguous():
        return cu_seqlens
    return _int32(cu_seqlens, device)


def gated_delta_rule(q, k, v, g, beta, *, cu_seqlens=None, scale: Optional[float] = None, qk_l2norm: bool = True,
                     chunk: int = 64, initial_state: Optional[torch.Tensor] = None, output_final_state: bool = False):
    """Chunk-parallel gated delta rule over packed tokens, differentiable in all tensors.

    q, k ``[T, Hk, dk]``, v ``[T, Hv, dv]`` with ``Hv`` a multiple of ``Hk`` (key head j serves the value heads
    ``[j Hv/Hk, (j+1) Hv/Hk)``), log decay g and write strength beta ``[T, Hv]``. The state starts anew at every boundary
    of ``cu_seqlens`` (list or tensor of N + 1 offsets): from ``initial_state [N, Hv, dk, dv]`` (fp32) or from zero. Rows
    that no sequence covers come back as zeros. Returns ``o [T, Hv, dv]`` in v's dtype, and the fp32 states behind the
    last token of each sequence when ``output_final_state``; a sequence without tokens hands its initial state through.

    On a GPU (bf16, head dims 64 or 128) the chunk is 64 tokens whatever ``chunk`` says. A decay below ``exp(-120)`` counts
    as zero there. Memory goes by chunks, each of up to 64 tokens of ONE sequence: they are taken as ``T / 64 + N``, so that
    many short sequences cost more than their tokens. A chunk takes 39,680 bytes a value head and ``256 (dk + 8)`` a key
    head while the call runs; with gradients enabled these and ``768 dv + 4 dk dv`` bytes a value head (partial results and
    two states) are kept until the backward pass, which itself works on ``4 dk dv + 177 dv`` more. With 16 / 32 heads of 128
    that is 7 MB a chunk: 1.8 GB for one row of 16,384 tokens, 29 GB for 4,096 sequences of one token.

    Precision there: sums and the state along the sequence are fp32; the products take bf16 inputs as they are, and of fp32
    operands 24 bits or, behind a decay, 16 (three or two bf16 parts). Results in bf16 are as exact as their rounding. Final
    states, dg and dbeta are within 1e-6 (2-norm) for heads that forget within some hundred tokens, as fp32 products give
    them, and within 5e-6, ten times that, for decays near one. Inputs in fp32 take the PyTorch form, in fp32 throughout.
    """
    _check_delta(q, k, v, g, beta, "T")
    T, _, dk = q.shape
    H, dv = v.shape[1:]
    scale = float(scale) if scale is not None else dk ** -0.5
    if gated_delta_rule_native(q, k, v):
        cu = _device_bounds(cu_seqlens, T, v.device)
        if initial_state is not None:
            _check_state(initial_state, (1 if cu is None else cu.numel() - 1, H, dk, dv), v.device, "initial_state")
            initial_state = _dense16(initial_state)
        keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                            or beta.requires_grad or (initial_state is not None and initial_state.requires_grad))
        o, last = _GatedDeltaFn.apply(q, k, v, g, beta, initial_state, cu, scale, qk_l2norm, output_final_state, keep)
        return (o, last) if output_final_state else o
    dt = v.dtype
    bounds = _host_bounds(cu_seqlens, T)
    if initial_state is not None:
        _check_state(initial_state, (len(bounds) - 1, H, dk, dv), v.device, "initial_state")
    q, k, v, g, beta = (t.float() for t in (q, k, v, g, beta))
    if qk_l2norm:
        q, k = l2norm(q), l2norm(k)
    q = q * scale
    q, k = _share_heads(q, k, H)
    outs, last = [v.new_zeros(bounds[0], H, dv)], []
    for n, (s, e) in enumerate(zip(bounds, bounds[1:])):
        state = initial_state[n] if initial_state is not None else None
        if e > s:
            o, state = _chunk_one(q[s:e].transpose(0, 1), k[s:e].transpose(0, 1), v[s:e].transpose(0, 1),
                                  g[s:e].t(), beta[s:e].t(), chunk, state)
            outs.append(o.transpose(0, 1))
        last.append(state if state is not None else v.new_zeros(H, dk, dv))
    outs.append(v.new_zeros(T - bounds[-1], H, dv))
    o = torch.cat(outs, 0).to(dt)
    return (o, torch.stack(last)) if output_final_state else o


def _check_state(state, shape, device, name: str):
    if state.shape != shape or state.dtype != torch.float32 or state.device != device:
        raise ValueError(f"{name} must be fp32 {list(shape)} on {device}, got {state.dtype} {list(state.shape)} on "
                         f"{state.device}")


def _step_index(state_indices, rows: int, slots: int, device, native: bool) -> Optional[torch.Tensor]:
    """Slots of the rows as int32 on `device`. Indices on the host are checked here, and so are those that the PyTorch form
    reads; those on the device are else checked by the kernel, which reports a bad one through the status word and leaves
    its row out."""
    if state_indices is None:
        if rows > slots:
            raise ValueError(f"{rows} rows need {rows} state slots, there are {slots}")
        return None
    if native and torch.is_tensor(state_indices) and state_indices.is_cuda:
        if state_indices.shape != (rows,):
            raise ValueError(f"state_indices must hold one slot for each of the {rows} rows")
        if state_indices.dtype == torch.int32 and state_indices.device == device and state_indices.is_contiguous():
            return state_indices
        _whole(state_indices, "state_indices")
        return _int32(state_indices, device)
    _whole(state_indices, "state_indices")
    idx = [index(i) for i in (state_indices.tolist() if torch.is_tensor(state_indices) else state_indices)]
    used = [i for i in idx if i >= 0]
    if len(idx) != rows or any(i >= slots for i in used) or len(set(used)) < len(used):
        raise ValueError(f"state_indices must name {rows} different slots below {slots} (negative: no row)")
    return torch.tensor(idx, dtype=torch.int32, device=device)


def _no_gradient(*tensors):
    if not torch.is_grad_enabled():
        return
    for t in tensors:
        if t is None or not t.requires_grad:
            continue
        raise RuntimeError("the single-token form updates its state in place and has no gradient: call it under "
                           "torch.no_grad()")


def gated_delta_rule_step(q, k, v, g, beta, state: torch.Tensor, *, state_indices=None, scale: Optional[float] = None,
                          qk_l2norm: bool = True) -> torch.Tensor:
    """One token of the gated delta rule for each of B rows: q, k ``[B, Hk, dk]``, v ``[B, Hv, dv]``, g, beta ``[B, Hv]``;
    returns ``o [B, Hv, dv]``. ``state [slots, Hv, dk, dv]`` (fp32, contiguous) is updated IN PLACE: row b uses slot
    ``state_indices[b]`` (its own number without indices). A negative index is a padding row: zeros come back and no state
    changes. Two rows on one slot, or a slot out of range, are an error: raised here for indices on the host and where no
    kernel covers the inputs; else, for indices on the GPU, the later row is left out as a padding row is and the status
    word is set (``_ext.check_status``).
    """
    _check_delta(q, k, v, g, beta, "B")
    _no_gradient(q, k, v, g, beta, state)
    B, _, dk = q.shape
    H, dv = v.shape[1:]
    if state.dim() != 4:
        raise ValueError("state must be [slots, value heads, dk, dv]")
    _check_state(state, (state.shape[0], H, dk, dv), v.device, "state")
    if not state.is_contiguous():
        raise ValueError("state is updated in place and must be contiguous")
    scale = float(scale) if scale is not None else dk ** -0.5
    native = gated_delta_rule_native(q, k, v)
    idx = _step_index(state_indices, B, state.shape[0], v.device, native)
    if native:
        return _ext.require().delta_step(_rows16(q), _rows16(k), _rows16(v), g if g.dtype == torch.float32 and g.is_contiguous() else _fp32(g),
                                         beta if beta.dtype == torch.float32 and beta.is_contiguous() else _fp32(beta), state, idx,
                                         scale, qk_l2norm, _status(v))
    out = v.new_zeros(B, H, dv)
    for b, slot in enumerate(range(B) if idx is None else idx.tolist()):
        if slot < 0:
            continue
        o, s = _chunk_one_token(q[b], k[b], v[b], g[b], beta[b], state[slot], scale, qk_l2norm)
        state[slot] = s
        out[b] = o.to(v.dtype)
    return out


def _chunk_one_token(q, k, v, g, beta, S, scale, qk_l2norm):
    q, k, v, g, beta = (t.float() for t in (q, k, v, g, beta))
    if qk_l2norm:
        q, k = l2norm(q), l2norm(k)
    q, k = _share_heads(q * scale, k, v.shape[0])
    S = S * g.exp()[:, None, None]
    d = (v - torch.einsum("hkv,hk->hv", S, k)) * beta[:, None]
    S = S + k[:, :, None] * d[:, None, :]
    return torch.einsum("hkv,hk->hv", S, q), S


class _CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cu, silu):
        ctx.save_for_backward(x, weight, bias, cu)
        ctx.silu = silu
        return _ext.require().conv1d_fwd(x, weight, bias, cu, silu)

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, cu = ctx.saved_tensors
        dx, dw, db = _ext.require().conv1d_bwd(_dense16(dy), x, weight, bias, cu, ctx.silu)
        return first_order("causal_conv1d", (dx, dw, db if bias is not None else None), dy, x, weight, bias) + (None, None)


_ACTIVATIONS = {None: False, "silu": True, "swish": True}


def _check_conv(x, weight, bias, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be None, 'silu' or 'swish', got {activation!r}")
    if x.dim() != 2 or weight.dim() != 2 or weight.shape[0] != x.shape[1]:
        raise ValueError(f"x [rows, C] and weight [C, K] expected, got {tuple(x.shape)}, {tuple(weight.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias must be [{weight.shape[0]}], got {tuple(bias.shape)}")


def _conv_native(x, weight) -> bool:
    """Whether the sm_100a kernels cover these inputs: bf16 on a GPU, channels in multiples of 8, two to four taps."""
    return x.is_cuda and x.dtype == torch.bfloat16 and x.shape[1] % 8 == 0 and 2 <= weight.shape[1] <= 4


def _plain16(t):
    """Contiguous bf16 parameter with a 16-byte aligned base."""
    if t is None or (t.dtype == torch.bfloat16 and t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return _dense16(t.to(torch.bfloat16))


def causal_conv1d(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, cu_seqlens=None,
                  activation: Optional[str] = "silu") -> torch.Tensor:
    """Depthwise causal convolution over packed tokens. x [T, C]; weight [C, K]. Token t sees t-K+1..t of
    its own sequence only: every sequence begins here, inputs of an earlier part of it are not taken. Rows that no sequence
    covers come back as zeros. ``activation`` is "silu" ("swish") or None, others are refused, and so are boundaries on the
    host that leave the rows or go back; those on a GPU are clamped."""
    _check_conv(x, weight, bias, activation)
    T, C = x.shape
    K = weight.shape[-1]
    if _conv_native(x, weight):
        # the weight is rounded to x's dtype, as in the PyTorch form
        return _CausalConvFn.apply(_rows16(x), _plain16(weight), _plain16(bias), _device_bounds(cu_seqlens, T, x.device),
                                   _ACTIVATIONS[activation])
    bounds = _host_bounds(cu_seqlens, T)
    outs = [x.new_zeros(bounds[0], C)]
    for s, e in zip(bounds, bounds[1:]):
        if e > s:
            seg = F.pad(x[s:e].t().unsqueeze(0), (K - 1, 0))
            y = F.conv1d(seg, weight.unsqueeze(1).to(x.dtype), None if bias is None else bias.to(x.dtype), groups=C)[0].t()
            outs.append(F.silu(y) if _ACTIVATIONS[activation] else y)
    outs.append(x.new_zeros(T - bounds[-1], C))
    return torch.cat(outs, 0)


def causal_conv1d_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                       state_indices=None, activation: Optional[str] = "silu") -> torch.Tensor:
    """One token of ``causal_conv1d`` for each of B rows, x ``[B, C]``: ``state [slots, C, K - 1]`` (x's dtype, contiguous)
    holds the last inputs of every sequence, oldest first, and is shifted IN PLACE. ``state_indices`` as in
    ``gated_delta_rule_step``."""
    _check_conv(x, weight, bias, activation)
    _no_gradient(x, weight, bias, state)
    B, C = x.shape
    K = weight.shape[1]
    if state.dim() != 3 or state.shape[1:] != (C, K - 1) or state.dtype != x.dtype or state.device != x.device or not state.is_contiguous():
        raise ValueError(f"state must be contiguous {x.dtype} [slots, {C}, {K - 1}] on {x.device}, got {state.dtype} "
                         f"{list(state.shape)} on {state.device}")
    native = _conv_native(x, weight)
    idx = _step_index(state_indices, B, state.shape[0], x.device, native)
    if native:
        return _ext.require().conv1d_step(_rows16(x), state, _plain16(weight), _plain16(bias), idx, _ACTIVATIONS[activation],
                                          _status(x))
    out = torch.zeros_like(x)
    for b, slot in enumerate(range(B) if idx is None else idx.tolist()):
        if slot < 0:
            continue
        window = torch.cat([state[slot], x[b, :, None]], -1)
        y = (window.float() * weight.to(x.dtype).float()).sum(-1)
        y = y if bias is None else y + bias.to(x.dtype).float()
        state[slot] = window[:, 1:]
        out[b] = (F.silu(y) if _ACTIVATIONS[activation] else y).to(x.dtype)
    return out
