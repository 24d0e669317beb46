"""The autograd functions around the kernels, on the CPU with a stand-in for the extension."""
from types import SimpleNamespace

import pytest
import torch

from loongforge_b200.ops import _ext
from loongforge_b200.ops import functional as OF
from loongforge_b200.ops import linear_attn as LA


def test_second_derivatives_are_an_error_not_a_part_of_one(monkeypatch):
    """Backward kernels run outside autograd: without a mark the second derivative would lack their part and not say so."""
    T, C, K = 6, 8, 4
    bwd = {"conv1d_bwd": lambda dy, x, w, *a: (dy.clone(), torch.zeros_like(w), torch.zeros(8)),
           "delta_bwd": lambda do, ds, q, k, v, g, b, *a: tuple(map(torch.clone, (q, k, do, g, b))) + (torch.zeros(1, 1, 8, 8),),
           "qk_norm_rope_bwd": lambda dq, dk, dv, dg, x, G, R, gated, qw, kw, *a: (x.clone(), qw.clone(), kw.clone())}
    fake = SimpleNamespace(conv1d_fwd=lambda x, *a: x.clone(), delta_fwd=lambda q, k, v, *a: (v.clone(), torch.zeros(0), torch.zeros(1)),
                           qk_norm_rope_fwd=lambda x, *a: (x[:, :4].clone(), x[:, 4:6].clone(), x[:, 6:]), **bwd)
    monkeypatch.setattr(_ext, "require", lambda: fake)
    monkeypatch.setattr(_ext, "status_tensor", lambda d=None: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(LA, "_status", lambda t: torch.zeros(1, dtype=torch.int32))
    one = lambda *shape: torch.randn(*shape, requires_grad=True)  # noqa: E731
    for name, f, leaves in (
            ("causal_conv1d", lambda x, w, b: LA._CausalConvFn.apply(x, w, b, None, True), (one(T, C), one(C, K), one(C))),
            ("gated_delta_rule", lambda *t: LA._GatedDeltaFn.apply(*t, None, 1.0, True, False, True)[0],
             (one(T, 1, C), one(T, 1, C), one(T, 1, C), one(T, 1), one(T, 1), one(1, 1, C, C))),
            ("qk_norm_rope", lambda *t: OF._QKNormRopeFn.apply(*t, 1, 2, False, None, None, None, None, 2, False, 1.0, 1e-6, 0.0)[0],
             (one(T, C), one(2), one(2)))):
        y = f(*leaves)
        assert all(d is not None for d in torch.autograd.grad(y.sum(), leaves, retain_graph=True))
        for loss in (y.sum(), y.square().sum()):
            d = torch.autograd.grad(loss + sum(t.square().sum() for t in leaves), leaves, create_graph=True, retain_graph=True)
            for leaf in leaves:  # each reaches the loss by another way too
                with pytest.raises(RuntimeError, match=f"{name}.*second derivative"):
                    torch.autograd.grad(sum(t.square().sum() for t in d), leaf, retain_graph=True)


def test_rows_for_the_kernels_have_strides_of_whole_16_byte_pieces():
    """A single row cut out of a wider one counts as contiguous whatever its row stride."""
    wide = torch.randn(3, 65).bfloat16()
    for t in (wide[:1, :64], wide[:, :64], wide[:1, :64].view(1, 1, 64), wide[:1, 1:], torch.randn(1, 67, dtype=torch.bfloat16)[:, None, :64]):
        r = LA._rows16(t)
        assert torch.equal(r, t) and r.stride(-1) == 1 and all(s % 8 == 0 for s in r.stride()[:-1]) and r.data_ptr() % 16 == 0
    even = torch.randn(4, 72).bfloat16()[:, :64]
    assert LA._rows16(even) is even


def test_inputs_are_saved_once(monkeypatch):
    """What offloads saved tensors moves each of them as often as it is saved."""
    fake = SimpleNamespace(delta_fwd=lambda q, k, v, *a: (v.clone(), torch.zeros(0), torch.zeros(1)))
    monkeypatch.setattr(_ext, "require", lambda: fake)
    monkeypatch.setattr(LA, "_status", lambda t: torch.zeros(1, dtype=torch.int32))
    q, k, v = (torch.randn(6, 1, 8, requires_grad=True) for _ in range(3))
    g, seen = torch.randn(6, 1, requires_grad=True), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.data_ptr()) or t, lambda t: t):
        LA._GatedDeltaFn.apply(q, k, v, g, g, None, None, 1.0, True, False, True)
    assert [seen.count(t.data_ptr()) for t in (q, k, v)] == [1, 1, 1]
