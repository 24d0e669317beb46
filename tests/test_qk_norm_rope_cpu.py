"""Norm + rotation of query and key heads on the CPU: the PyTorch form against the formula in 64 bits, against the separate
passes and against differences, and the refusals."""
import pytest
import torch

from loongforge_b200.ops import functional as OF


def formula(qkv, qw, kw, G, R, gated, ang, rot, interleaved, mscale, eps, off):
    """q, k, v (, gate) in the dtype of the inputs; ang [T, rot / 2]."""
    P = 2 * R + 2 if gated else R + 2
    x = qkv.view(qkv.shape[0], G, P, qkv.shape[1] // (G * P))
    i = torch.arange(rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    c, s = torch.cos(ang)[:, None] * mscale, torch.sin(ang)[:, None] * mscale

    def one(t, w):
        n = t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * (w + off)
        y = n.clone()
        y[..., lo], y[..., hi] = n[..., lo] * c - n[..., hi] * s, n[..., hi] * c + n[..., lo] * s
        return y

    out = (one(x[:, :, :R].reshape(len(x), G * R, x.shape[-1]), qw), one(x[:, :, -2], kw), x[:, :, -1])
    return out + ((x[:, :, R:2 * R],) if gated else ())


@pytest.mark.parametrize("T,G,R,D,rot,kw", [
    (1, 1, 1, 8, 8, {}), (5, 2, 3, 16, 8, dict(gated=True, off=1.0)), (7, 1, 4, 16, 16, dict(interleaved=True)),
    (6, 3, 1, 32, 12, dict(mscale=1.25)), (9, 2, 2, 16, 16, dict(axes=3, gated=True)), (0, 1, 2, 16, 16, {})])
def test_reference_form_is_the_formula(T, G, R, D, rot, kw):
    gated, off = kw.get("gated", False), kw.get("off", 0.0)
    il, ms, axes = kw.get("interleaved", False), kw.get("mscale", 1.0), kw.get("axes", 1)
    torch.manual_seed(0)
    qkv, qw, kw_ = torch.randn(T, G * (2 * R + 2 if gated else R + 2) * D), torch.randn(D), torch.randn(D)
    inv, ids = torch.rand(rot // 2), torch.randint(0, 300, (axes, T), dtype=torch.int32)
    axis = torch.randint(0, axes, (rot // 2,), dtype=torch.int32)
    ang = (ids.double()[axis.long()].t() * inv.double()) if axes > 1 else ids[0].double()[:, None] * inv.double()
    ins = [t.requires_grad_() for t in (qkv, qw, kw_)]
    got = OF.qk_norm_rope(qkv, G, R, qw, kw_, inv_freq=inv, pos_ids=ids if axes > 1 else ids[0], axis=axis if axes > 1 else None,
                          rot_dim=rot, interleaved=il, mscale=ms, w_offset=off, gated=gated)
    rins = [t.detach().double().requires_grad_() for t in ins]
    want = formula(*rins, G, R, gated, ang, rot, il, ms, 1e-6, off)
    assert [t.shape for t in got] == [t.shape for t in want]
    ups = [torch.randn(t.shape) for t in got]
    grads = torch.autograd.grad(got, ins, ups)
    rgrads = torch.autograd.grad(want, rins, [u.double() for u in ups])
    # fp32 angles of up to 300 are off by 2^-16 at most (half a step of 256 .. 512, and of the product), which is what an
    # element can move by in parts of its pair; the sums over 32 elements and T tokens are far finer
    for a, b in zip((*got, *grads), (*want, *rgrads)):
        if b.numel():
            assert ((a.double() - b).abs() <= 2.0 ** -14 * b.abs().max()).all(), (a.double() - b).abs().max()


def test_reference_form_equals_norm_and_rotation_apart():
    torch.manual_seed(1)
    T, G, R, D = 11, 2, 3, 16
    qkv, w, k_w = torch.randn(T, G * (R + 2) * D), torch.randn(D), torch.randn(D)
    freqs = OF.rope_freqs(torch.arange(T), D, 1e4)
    q, k, v = OF.qk_norm_rope(qkv, G, R, w, k_w, freqs=freqs)
    x = qkv.view(T, G, R + 2, D)
    assert torch.allclose(q, OF.rope(OF.rmsnorm(x[:, :, :R].reshape(T, G * R, D), w, 1e-6), freqs), atol=1e-5)
    assert torch.allclose(k, OF.rope(OF.rmsnorm(x[:, :, R].contiguous(), k_w, 1e-6), freqs), atol=1e-5)
    assert torch.equal(v, x[:, :, R + 1])


def test_gradient_against_differences():
    """Along a random direction, in 64 bits: central differences of step 1e-5 are off by about 1e-10 of the slope."""
    torch.manual_seed(2)
    T, G, R, D, rot = 4, 1, 2, 16, 8
    ins = [torch.randn(T, G * (2 * R + 2) * D, dtype=torch.float64), torch.randn(D, dtype=torch.float64), torch.randn(D, dtype=torch.float64)]
    ang = torch.rand(T, rot // 2, dtype=torch.float64)
    ups = None

    def value(ts):
        nonlocal ups
        out = formula(*ts, G, R, True, ang, rot, False, 1.0, 1e-6, 1.0)
        ups = ups or [torch.randn_like(t) for t in out]
        return sum((a * u).sum() for a, u in zip(out, ups))

    way = [torch.randn_like(t) for t in ins]
    reqs = [t.clone().requires_grad_() for t in ins]
    slope = sum((g * w).sum() for g, w in zip(torch.autograd.grad(value(reqs), reqs), way))
    h = 1e-5
    diff = (value([t + h * w for t, w in zip(ins, way)]) - value([t - h * w for t, w in zip(ins, way)])) / (2 * h)
    assert abs(diff - slope) <= 1e-6 * max(1.0, abs(slope))


def test_refusals():
    T, G, R, D = 4, 2, 2, 16
    x, w = torch.randn(T, G * (R + 2) * D), torch.ones(D)
    f, inv = torch.rand(T, D // 2), torch.rand(D // 2)
    pos = torch.arange(T, dtype=torch.int32)
    bad = [
        (dict(), "either"), (dict(freqs=f, inv_freq=inv), "either"), (dict(inv_freq=inv), "pos_ids"),
        (dict(inv_freq=inv, pos_ids=pos[:3]), "pos_ids"), (dict(inv_freq=inv, pos_ids=pos.expand(2, T)), "axis"),
        (dict(inv_freq=inv, pos_ids=pos, axis=torch.zeros(3, dtype=torch.int32)), "axis"),
        (dict(freqs=f[:3]), "cover"), (dict(freqs=f, pos_ids=pos[:3]), "cover"), (dict(freqs=f[:, :4]), "angles"),
        (dict(inv_freq=inv, pos_ids=pos + 0.5), "whole"), (dict(inv_freq=inv, pos_ids=pos, axis=torch.zeros(D // 2)), "whole"),
        (dict(freqs=f, rot_dim=7), "rot_dim"), (dict(freqs=f, rot_dim=32), "rot_dim"), (dict(freqs=f, gated=True), "heads"),
    ]
    for kw, what in bad:
        with pytest.raises(ValueError, match=what):
            OF.qk_norm_rope(x, G, R, w, w, **kw)
    with pytest.raises(ValueError, match="weights"):
        OF.qk_norm_rope(x, G, R, w[:8], w, freqs=f)
    with pytest.raises(ValueError, match="heads"):
        OF.qk_norm_rope(x[:, :-1], G, R, w, w, freqs=f)


def test_rows_and_axes_out_of_range_are_refused():
    """A row below zero is no row from the table's end."""
    x, w, f = torch.randn(4, 4 * 16), torch.ones(16), torch.rand(5, 8)
    for pos in ([0, 1, 2, -1], [0, 5, 0, 0], [2 ** 40, 0, 0, 0]):
        with pytest.raises(ValueError, match="out of range"):
            OF.qk_norm_rope(x, 1, 2, w, w, freqs=f, pos_ids=torch.tensor(pos))
    with pytest.raises(ValueError, match="out of range"):
        OF.qk_norm_rope(x, 1, 2, w, w, freqs=f[:0], pos_ids=torch.zeros(4, dtype=torch.long))
    inv, pos = torch.rand(8), torch.arange(8).view(2, 4)
    for ax in (-1, 2):
        with pytest.raises(ValueError, match="out of range"):
            OF.qk_norm_rope(x, 1, 2, w, w, inv_freq=inv, pos_ids=pos, axis=torch.full((8,), ax))
