"""Per-head norm + rotation of queries and keys in one pass, against the formula in 64 bits and its gradients.

The kernel works in fp32 and rounds once: 2^-8 of every element, and 2^-14 of the largest one for fp32 sums of up to 256
squares or products and the rotation's two terms. Weight gradients add up to all tokens and heads in fp32.
"""
import pytest
import torch

from loongforge_b200.ops import _ext
from loongforge_b200.ops import functional as OF

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rotate(x, ang, rot, interleaved, mscale):
    c, s = torch.cos(ang)[:, None] * mscale, torch.sin(ang)[:, None] * mscale
    i = torch.arange(rot // 2, device=x.device)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y = x.clone()
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    return y


def oracle(qkv, qw, kw, G, R, gated, ang, rot, interleaved, mscale, eps, off):
    T = qkv.shape[0]
    x = qkv.view(T, G, 2 * R + 2 if gated else R + 2, -1)

    def one(t, w):
        return rotate(t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * (w + off), ang, rot, interleaved, mscale)

    out = (one(x[:, :, :R].reshape(T, G * R, -1), qw), one(x[:, :, -2], kw), x[:, :, -1])
    return out + ((x[:, :, R:2 * R],) if gated else ())


def near(a, b, what):
    lim = b.abs() * 2.0 ** -8 + b.abs().max() * 2.0 ** -14
    assert ((a.double() - b).abs() <= lim).all(), (what, (a.double() - b).abs().max().item())


def check(T, G, R, D, rot, *, gated=False, axes=1, table=False, interleaved=False, mscale=1.0, off=0.0, far=0, seed=0, pos=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(BF16)  # noqa: E731
    P = 2 * R + 2 if gated else R + 2
    qkv, qw, kw = rn(T, G * P * D), rn(D), rn(D)
    inv = (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda()
    ids = torch.randint(far, far + 500, (axes, T), generator=gen, device="cuda", dtype=torch.int32)
    axis = torch.randint(0, axes, (rot // 2,), generator=gen, device="cuda", dtype=torch.int32)
    if table:
        tab = torch.outer(torch.arange(far + 500, device="cuda").float(), inv)
        where = dict(freqs=tab, pos_ids=ids[0] if pos else None)
        ang = (tab[ids[0].long()] if pos else tab[:T]).double()
    else:
        where = dict(inv_freq=inv, pos_ids=ids if axes > 1 else ids[0], axis=axis if axes > 1 else None)
        ang = ids.double()[axis.long()].t() * inv.double() if axes > 1 else ids[0].double()[:, None] * inv.double()
    ins = [t.requires_grad_() for t in (qkv, qw, kw)]
    got = OF.qk_norm_rope(qkv, G, R, qw, kw, rot_dim=rot, interleaved=interleaved, mscale=mscale, eps=1e-6, w_offset=off, gated=gated, **where)
    ups = [rn(*t.shape) for t in got]
    grads = torch.autograd.grad(got, ins, ups)
    rins = [t.detach().double().requires_grad_() for t in ins]
    want = oracle(*rins, G, R, gated, ang, rot, interleaved, mscale, 1e-6, off)
    rgrads = torch.autograd.grad(want, rins, [u.double() for u in ups])
    _ext.check_status()
    for n, a, b in zip(("q", "k", "v", "gate"), got, want):
        near(a, b, n)
    near(grads[0], rgrads[0], "dqkv")
    for n, a, b in zip(("dqw", "dkw"), grads[1:], rgrads[1:]):
        near(a, b, n)


@pytest.mark.parametrize("T,G,R,D,rot", [(1, 1, 1, 64, 64), (3, 2, 4, 128, 128), (4, 1, 8, 256, 64), (5, 3, 3, 64, 32), (130, 2, 5, 128, 16), (9, 1, 2, 256, 256), (7, 2, 2, 128, 24)])
@pytest.mark.parametrize("gated", [False, True])
def test_qk_norm_rope_shapes(T, G, R, D, rot, gated):
    check(T, G, R, D, rot, gated=gated)


@pytest.mark.parametrize("kw", [dict(axes=2), dict(axes=3, gated=True, off=1.0), dict(table=True), dict(table=True, pos=False),
                                dict(table=True, interleaved=True), dict(interleaved=True), dict(mscale=1.3), dict(off=1.0)])
def test_qk_norm_rope_positions(kw):
    check(70, 2, 3, 128, 64, **kw)


def test_qk_norm_rope_far_positions():
    """Angles of positions around two million keep their fraction of a turn."""
    check(40, 1, 2, 128, 128, far=2_000_000)
    check(40, 1, 2, 128, 128, far=1_000_000, axes=3)


def test_qk_norm_rope_zero_rows_and_strides():
    qkv = torch.randn(20, 4 * 128 + 8, device="cuda").to(BF16)[:, :4 * 128]
    w = torch.randn(128, device="cuda").to(BF16)
    freqs = torch.rand(20, 64, device="cuda")
    a = OF.qk_norm_rope(qkv, 1, 2, w, w, freqs=freqs)
    b = OF.qk_norm_rope(qkv.contiguous(), 1, 2, w, w, freqs=freqs)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    odd = torch.randn(20, 4 * 128 + 1, device="cuda").to(BF16)[:, 1:]
    c = OF.qk_norm_rope(odd, 1, 2, w, w, freqs=freqs)
    assert all(torch.equal(x, y) for x, y in zip(c, OF.qk_norm_rope(odd.contiguous(), 1, 2, w, w, freqs=freqs)))
    z = torch.zeros(3, 4 * 128, device="cuda", dtype=BF16, requires_grad=True)
    q, k, v = OF.qk_norm_rope(z, 1, 2, w, w, freqs=freqs)
    d = torch.autograd.grad([q, k, v], z, [torch.ones_like(t) for t in (q, k, v)])[0]
    assert not q.any() and d.isfinite().all()
    e = torch.zeros(0, 4 * 128, device="cuda", dtype=BF16, requires_grad=True)
    wr = w.clone().requires_grad_()
    q, k, v = OF.qk_norm_rope(e, 1, 2, wr, w, freqs=freqs)
    assert q.shape == (0, 2, 128) and not torch.autograd.grad(q.sum(), wr)[0].any()


def test_qk_norm_rope_bad_rows_turn_by_zero_and_are_reported():
    x = torch.randn(4, 4 * 128, device="cuda").to(BF16)
    w = torch.ones(128, device="cuda").to(BF16)
    freqs = torch.rand(10, 64, device="cuda") + 0.5
    pos = torch.tensor([3, 10, -1, 1 << 30], device="cuda", dtype=torch.int32)
    q, _, _ = OF.qk_norm_rope(x, 1, 2, w, w, freqs=freqs, pos_ids=pos)
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()
    still, _, _ = OF.qk_norm_rope(x, 1, 2, w, w, freqs=torch.zeros_like(freqs), pos_ids=pos.clamp(0, 9))
    assert torch.equal(q[1:], still[1:]) and not torch.equal(q[0], still[0])
    inv, axis = torch.rand(64, device="cuda") + 0.5, torch.full((64,), 2, device="cuda", dtype=torch.int32)
    OF.qk_norm_rope(x, 1, 2, w, w, inv_freq=inv, axis=axis, pos_ids=torch.ones(2, 4, device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()


def test_qk_norm_rope_matches_the_separate_passes_on_attention():
    """As the attention layer uses it: the fused pass and norm, then rotation, give the same attention but for one rounding
    of q and k (2^-8 of each score's terms; scores of order sqrt(128) at most move a probability by a few per cent of it)."""
    torch.manual_seed(0)
    T, G, R, D = 200, 2, 4, 128
    qkv = torch.randn(T, G * (R + 2) * D, device="cuda").to(BF16)
    w = torch.rand(D, device="cuda").to(BF16)
    freqs = OF.rope_freqs(torch.arange(T, device="cuda"), D, 1e4)
    q, k, v = OF.qk_norm_rope(qkv, G, R, w, w, freqs=freqs)
    x = qkv.view(T, G, R + 2, D)
    q2 = OF.rope(OF.rmsnorm(x[:, :, :R].reshape(T, G * R, D), w, 1e-6), freqs)
    k2 = OF.rope(OF.rmsnorm(x[:, :, R].contiguous(), w, 1e-6), freqs)
    assert torch.equal(v, x[:, :, R + 1])
    assert (q.float() - q2.float()).abs().max() <= 3 * 2.0 ** -8 * q.float().abs().max()
    a, b = OF.attention(q, k, v), OF.attention(q2, k2, x[:, :, R + 1])
    assert (a.float() - b.float()).norm() / b.float().norm() < 0.03


@pytest.mark.parametrize("T,G,R,D,rot,kw", [(1500, 1, 1, 64, 64, {}), (2100, 4, 4, 64, 16, dict(gated=True)), (701, 2, 16, 64, 24, {}),
                                            (1201, 1, 8, 256, 8, dict(interleaved=True)), (3, 8, 3, 128, 40, dict(interleaved=True)),
                                            (2500, 3, 2, 128, 128, dict(interleaved=True, axes=2))])
def test_qk_norm_rope_layouts(T, G, R, D, rot, kw):
    """Many tokens and few, one head of a kind and many: a lane keeps from one to eight heads of its token."""
    check(T, G, R, D, rot, **kw)


def test_qk_norm_rope_values_and_gates_keep_to_themselves():
    """NaN in the value and gate heads, and in one query head, reaches no other head; their gradients go straight through."""
    torch.manual_seed(3)
    T, G, R, D = 9, 2, 3, 128
    w = torch.randn(D, device="cuda").to(BF16)
    freqs = torch.rand(T, D // 2, device="cuda")
    clean = torch.randn(T, G, 2 * R + 2, D, device="cuda").to(BF16)
    sick = clean.clone()
    sick[:, :, R:2 * R] = sick[:, :, -1] = float("nan")
    sick[4, 1, 0, 5] = float("inf")
    xs = [t.view(T, -1).requires_grad_() for t in (clean, sick)]
    a, b = (OF.qk_norm_rope(x, G, R, w, w, freqs=freqs, gated=True) for x in xs)
    ups = [torch.randn_like(t) for t in a]
    da, db = (torch.autograd.grad(o, x, ups)[0].view(T, G, 2 * R + 2, D) for o, x in zip((a, b), xs))
    there = torch.ones(T, G * R, dtype=torch.bool, device="cuda")
    there[4, R] = False
    assert torch.equal(a[0][there], b[0][there]) and torch.equal(a[1], b[1])
    keep = torch.ones(T, G, 2 * R + 2, dtype=torch.bool, device="cuda")
    keep[4, 1, 0] = False
    assert torch.equal(da[keep], db[keep]) and torch.equal(db[:, :, R:2 * R], ups[3]) and torch.equal(db[:, :, -1], ups[2])


def test_qk_norm_rope_upstream_layouts_streams_and_replay():
    torch.manual_seed(4)
    T, G, R, D = 300, 2, 4, 128
    qkv = torch.randn(T, G * (R + 2) * D, device="cuda").to(BF16)
    w = torch.randn(D, device="cuda").to(BF16)
    inv, pos = torch.rand(D // 2, device="cuda"), torch.arange(T, device="cuda", dtype=torch.int32)
    ups = [torch.randn(G * R, T, D, device="cuda").to(BF16).transpose(0, 1), torch.randn(1, 1, D, device="cuda").to(BF16).expand(T, G, D),
           torch.randn(T, G, 2 * D, device="cuda").to(BF16)[..., :D]]

    def run(x, qw, kw, up):
        out = OF.qk_norm_rope(x, G, R, qw, kw, inv_freq=inv, pos_ids=pos)
        return [*(t.detach().clone() for t in out), *torch.autograd.grad(out, (x, qw, kw), up)]

    def leaves():
        return [t.detach().clone().requires_grad_() for t in (qkv, w, w)]

    want = run(*leaves(), [u.contiguous() for u in ups])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*leaves(), ups)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ins = leaves()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(*ins, ups)
    with torch.no_grad():
        qkv.copy_(qkv.flip(0))
        ins[0].copy_(qkv)
        pos.add_(17)
    graph.replay()
    torch.cuda.synchronize()
    want = run(*leaves(), ups)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_qk_norm_rope_bad_rows_in_the_pytorch_form():
    """Shapes without a kernel (head dim 48, fp32) treat rows and axes out of range as the kernel does."""
    x, w, freqs = torch.randn(4, 4 * 48, device="cuda"), torch.ones(48, device="cuda"), torch.rand(10, 24, device="cuda") + 0.5
    pos = torch.tensor([3, 10, -1, 1 << 40], device="cuda")
    q, _, _ = OF.qk_norm_rope(x, 1, 2, w, w, freqs=freqs, pos_ids=pos)
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()
    still, _, _ = OF.qk_norm_rope(x, 1, 2, w, w, freqs=torch.zeros_like(freqs), pos_ids=pos.clamp(0, 9))
    assert torch.equal(q[1:], still[1:]) and not torch.equal(q[0], still[0])
    _ext.check_status()
    OF.qk_norm_rope(x, 1, 2, w, w, inv_freq=freqs[0], axis=torch.full((24,), 2, device="cuda"), pos_ids=pos[:1].expand(2, 4))
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()


def test_qk_norm_rope_without_eps():
    """Lanes that have no head or token left must not bring the root of nothing into the weights' gradients."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    for T, G, R, D in ((1, 1, 1, 64), (3, 2, 3, 128), (301, 1, 5, 256)):
        x, w = (torch.randn(*s, generator=gen, device="cuda").to(BF16).requires_grad_() for s in ((T, G * (R + 2) * D), (D,)))
        f = torch.rand(T, D // 2, device="cuda")
        got = OF.qk_norm_rope(x, G, R, w, w, freqs=f, eps=0.0)
        ups = [torch.randn(t.shape, generator=gen, device="cuda").to(BF16) for t in got]
        rx, rw = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want = oracle(rx, rw, rw, G, R, False, f.double(), D, False, 1.0, 0.0, 0.0)
        a, b = torch.autograd.grad(got, (x, w), ups), torch.autograd.grad(want, (rx, rw), [u.double() for u in ups])
        near(a[0], b[0], "dqkv")
        # dw of the queries and of the keys are each rounded, and their sum once more
        assert ((a[1].double() - b[1]).abs() <= 3 * 2.0 ** -8 * b[1].abs().max()).all()
