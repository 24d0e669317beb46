"""Gated delta rule and causal convolution kernels against the recurrence / the sum over taps in 64 bits.

Tolerances. One rounding to bf16 is off by at most 2^-8 of the value. The kernels cut fp32 operands into a bf16 high and
low part whose remainder is at most 2^-18 of the value, so each product of the chain is off by about 2^-17 of its terms;
an fp32 result is the end of at most four such products (state, K S, U, state): 4 * 2^-17 in the 2-norm. dq and dk take
up to two operands at their high part alone and round once more: 3 * 2^-8 in the 2-norm. Of o and dv, rounded once, every
element is held: 2^-8 of itself, plus 2^-12 of the largest one for the products (2^-17 of a sum of at most 192 terms
whose absolute sum is taken as 32 times the largest result).
"""
import pytest
import torch

from loongforge_b200.ops import _ext
from loongforge_b200.ops import linear_attn as LA

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def make(lens, hk, hv, dk, dv, seed=0, mean=0.3, decay=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lens)
    q, k = randn(gen, T, hk, dk, dtype=BF16), (randn(gen, T, hk, dk) + mean).to(BF16)
    v, do = randn(gen, T, hv, dv, dtype=BF16), randn(gen, T, hv, dv, dtype=BF16)
    g = -torch.rand(T, hv, generator=gen, device="cuda") * decay * torch.rand(hv, generator=gen, device="cuda")
    beta = torch.rand(T, hv, generator=gen, device="cuda")
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")
    return q, k, v, g, beta, do, cu


def oracle(q, k, v, g, beta, bounds, state=None, scale=None, l2=True):
    """The recurrence in 64 bits; rows outside the bounds are zero."""
    hv, dk, dv = v.shape[1], q.shape[2], v.shape[2]
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    if l2:
        q, k = (t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q = (q * (dk ** -0.5 if scale is None else scale)).repeat_interleave(hv // q.shape[1], 1)
    k = k.repeat_interleave(hv // k.shape[1], 1)
    out, last = {}, []
    for n, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        S = torch.zeros(hv, dk, dv, dtype=torch.float64, device=v.device) if state is None else state[n].double()
        for t in range(lo, hi):
            S = torch.exp(g[t])[:, None, None] * S
            u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None, :]
            out[t] = (S * q[t][:, :, None]).sum(1)
        last.append(S)
    zero = torch.zeros(hv, dv, dtype=torch.float64, device=v.device)
    return torch.stack([out.get(t, zero) for t in range(v.shape[0])]) if v.shape[0] else v, torch.stack(last)


def rel(a, b):
    return ((a.double() - b).norm() / b.norm().clamp_min(1e-30)).item()


def close(a, b, what):
    """Every element within one rounding and the products' error (see above)."""
    lim = b.abs() * 2.0 ** -8 + b.abs().max() * 2.0 ** -12
    bad = ((a.double() - b).abs() > lim) | ~torch.isfinite(a.double())
    assert not bad.any(), (what, int(bad.sum()), (a.double() - b).abs().max().item(), b.abs().max().item())


def check(lens, hk, hv, dk=128, dv=128, *, state=False, final=False, scale=None, l2=True, edit=None, seed=0, zero_dg=False, **kw):
    q, k, v, g, beta, do, cu = make(lens, hk, hv, dk, dv, seed, **kw)
    if edit:
        edit(q, k, v, g, beta)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    s0 = randn(gen, len(lens), hv, dk, dv) if state else None
    ds = randn(gen, len(lens), hv, dk, dv) if final else None
    ins = [t.detach().requires_grad_() for t in (q, k, v, g, beta)] + ([s0.detach().requires_grad_()] if state else [])
    o, last = LA.gated_delta_rule(*ins[:5], cu_seqlens=cu, scale=scale, qk_l2norm=l2, initial_state=ins[5] if state else None,
                                  output_final_state=True)
    outs, ups = ([o, last], [do, ds]) if final else ([o], [do])
    grads = torch.autograd.grad(outs, ins, ups)
    rins = [t.detach().double().requires_grad_() for t in ins]
    ro, rlast = oracle(*rins[:5], cu.tolist(), rins[5] if state else None, scale, l2)
    loss = (ro * do.double()).sum() + ((rlast * ds.double()).sum() if final else 0)
    rgrads = torch.autograd.grad(loss, rins)
    _ext.check_status()
    close(o, ro, "o")
    assert rel(last, rlast) < 4 * 2.0 ** -17, rel(last, rlast)
    for name, a, b in zip(("dq", "dk"), grads[:2], rgrads[:2]):
        assert rel(a, b) < 3 * 2.0 ** -8, (name, rel(a, b))
    close(grads[2], rgrads[2], "dv")
    more = 1
    if zero_dg:
        # The value is zero: what comes back is what is left of its terms, o . do and v . dv of up to 64 tokens, each off
        # by 2^-17 of itself at most four times over.
        terms = ((ro * do.double()).sum(-1).abs() + (rins[2] * rgrads[2]).sum(-1).abs()).sum(0)
        assert rgrads[3].abs().max() < 1e-7 and (grads[3].abs() < 4 * 2.0 ** -17 * terms).all()
        # With equal keys and full strength A - I is minus its first lower diagonal: X_i = dU_i - dU_{i+1}, differences of
        # sums over up to 64 tokens' do that share all terms but one: X is 1 / sqrt(64) of the dU that carries the error.
        more = 8
    for name, a, b in list(zip(("dg", "dbeta", "dstate"), grads[3:], rgrads[3:]))[1 if zero_dg else 0:]:
        assert rel(a, b) < more * 4 * 2.0 ** -17, (name, rel(a, b))


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [128], [1, 63, 64, 65, 7], [0, 5, 0, 0, 70, 0], [300]])
def test_gated_delta_rule_lengths(lens):
    check(lens, 2, 4)


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64)])
def test_gated_delta_rule_head_dims(dk, dv):
    check([70, 130], 1, 3, dk, dv, state=True, final=True)


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("decay", [1e-3, 1.0])
def test_gated_delta_rule_key_and_query_gradients_element_by_element(dk, dv, decay):
    """With decays near one most of dq and dk comes from the states in front of and behind a chunk. Every operand keeps 16
    bits, so an element is off by its rounding and by 2^-17 of its terms, twice that where both operands are cut: the bound
    of `close` with a second 2^-12 of the largest result."""
    q, k, v, g, beta, do, cu = make([250], 2, 4, dk, dv, 11, decay=decay)
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    got = torch.autograd.grad(LA.gated_delta_rule(*ins, cu_seqlens=cu), ins[:2], do)
    rins = [t.detach().double().requires_grad_() for t in ins]
    want = torch.autograd.grad((oracle(*rins, [0, 250])[0] * do.double()).sum(), rins[:2])
    for name, a, b in zip(("dq", "dk"), got, want):
        off = (a.double() - b).abs() - b.abs() * 2.0 ** -8
        assert (off <= b.abs().max() * 2.0 ** -11).all(), (name, (off.max() / b.abs().max()).item() * 2.0 ** 11)


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_gated_delta_rule_fp32_results_with_the_gates_of_a_new_layer(dk, dv):
    """Gradients of the gates and final states where heads forget within some tokens, as the layer starts: U, what it is made
    of and P enter their products with 24 bits, and what is still cut to 16 (the state, the inverse, the state's gradient)
    carries a decay, so that its 2^-18 counts half at most."""
    gen = torch.Generator(device="cuda").manual_seed(15)
    q, k, v, _, _, do, cu = make([300, 64, 90], 2, 4, dk, dv, 15)
    x = torch.nn.functional.softplus(torch.randn(454, 4, generator=gen, device="cuda") + 1)
    g, beta = -x * torch.tensor([4.0, 8.0, 12.0, 16.0], device="cuda"), torch.rand(454, 4, generator=gen, device="cuda").sigmoid()
    s0 = randn(gen, 3, 4, dk, dv, scale=0.1)
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    o, last = LA.gated_delta_rule(*ins, cu_seqlens=cu, initial_state=s0, output_final_state=True)
    got = torch.autograd.grad(o, ins[3:], do)
    rins = [t.detach().double().requires_grad_() for t in ins]
    ro, rlast = oracle(*rins, cu.tolist(), s0)
    want = torch.autograd.grad((ro * do.double()).sum(), rins[3:])
    for name, a, b in (("last", last, rlast), ("dg", got[0], want[0]), ("dbeta", got[1], want[1])):
        assert rel(a, b) < 2.0 ** -19, (name, rel(a, b))


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
def test_gated_delta_rule_bf16_results_are_the_rounded_values(dk, dv):
    """With the gates of a new layer the part of a result that no decay has made small keeps 24 bits, and the rest is off by
    2^-18 of a part that counts half at most: a result lies that near to a border between two bf16 values, 2^-8 apart, with
    a chance of 2^-10 at most, counted half since the values spread over twice their lowest. dq and dk add heads and take
    the norm's part off, each of the same kind."""
    gen = torch.Generator(device="cuda").manual_seed(19)
    q, k, v, _, _, do, cu = make([300, 64, 90], 2, 4, dk, dv, 19)
    g = -torch.nn.functional.softplus(torch.randn(454, 4, generator=gen, device="cuda") + 1) * torch.tensor([4.0, 8.0, 12.0, 16.0], device="cuda")
    ins = [t.requires_grad_() for t in (q, k, v, g, torch.rand(454, 4, generator=gen, device="cuda"))]
    o = LA.gated_delta_rule(*ins, cu_seqlens=cu)
    got = [o.detach(), *torch.autograd.grad(o, ins[:3], do)]
    rins = [t.detach().double().requires_grad_() for t in ins]
    ro, _ = oracle(*rins, cu.tolist())
    want = [ro.detach(), *torch.autograd.grad((ro * do.double()).sum(), rins[:3])]
    for name, a, b in zip(("o", "dq", "dk", "dv"), got, want):
        other = (a != b.to(BF16)).double().mean().item()
        assert other < 2.0 ** -11, (name, other * 2.0 ** 11)


@pytest.mark.parametrize("hk,hv", [(1, 1), (3, 3), (2, 6)])
def test_gated_delta_rule_states_and_shared_heads(hk, hv):
    check([100, 0, 37], hk, hv, state=True, final=True)


def test_gated_delta_rule_no_decay_and_full_strength():
    def edit(q, k, v, g, beta):
        g.zero_()
        beta.fill_(1.0)
    check([200], 1, 2, edit=edit)


def test_gated_delta_rule_equal_keys():
    """Every token overwrites what the last one wrote: the chunk's triangular matrix is as far from I as it gets, and no
    decay matters (the gradient of g is zero)."""
    def edit(q, k, v, g, beta):
        k.copy_(k[:1].expand_as(k))
        beta.fill_(1.0)
        g.mul_(0.01)
    check([130], 1, 2, edit=edit, zero_dg=True)


def test_gated_delta_rule_resets_and_strong_decay():
    """A decay of zero in the middle of a chunk cuts the sequence there; strong ones keep their neighbours exact."""
    def edit(q, k, v, g, beta):
        g.mul_(20.0)
        g[10] = -500.0
        g[90:93] = float("-inf")
        g[0] = float("-inf")

    q, k, v, g, beta, do, cu = make([150], 1, 2, 128, 128, 3)
    edit(q, k, v, g, beta)
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    o = LA.gated_delta_rule(*ins, cu_seqlens=cu)
    grads = torch.autograd.grad(o, ins, do)
    rins = [t.detach().double().requires_grad_() for t in ins]
    # exp(-inf) has a derivative of zero times a sum: take the oracle's at the smallest decay that 64 bits hold as zero
    rins[3] = rins[3].detach().clamp(min=-800.0).requires_grad_()
    ro, _ = oracle(*rins, [0, 150])
    rgrads = torch.autograd.grad((ro * do.double()).sum(), rins)
    close(o, ro, "o")
    close(grads[2], rgrads[2], "dv")
    assert rel(grads[0], rgrads[0]) < 3 * 2.0 ** -8 and rel(grads[1], rgrads[1]) < 3 * 2.0 ** -8
    assert rel(grads[3], rgrads[3]) < 4 * 2.0 ** -17 and rel(grads[4], rgrads[4]) < 4 * 2.0 ** -17


def test_gated_delta_rule_tokens_that_write_nothing():
    """beta = 0 in some rows: they read, and their beta still has its gradient."""
    def edit(q, k, v, g, beta):
        beta[::3] = 0.0
        beta[40:80] = 0.0
    check([120], 1, 2, edit=edit)


def test_gated_delta_rule_without_norms():
    def edit(q, k, v, g, beta):
        q.mul_(0.1)
        k.mul_(0.06)
    check([100, 90], 1, 2, l2=False, scale=0.7, state=True, edit=edit)


def test_gated_delta_rule_reads_strided_rows():
    gen = torch.Generator(device="cuda").manual_seed(5)
    T, hk, hv, d = 77, 2, 4, 128
    fused = randn(gen, T, (2 * hk + hv) * d + 8, dtype=BF16)
    q, k, v = (t.unflatten(1, (-1, d)) for t in (fused[:, :hk * d], fused[:, hk * d:2 * hk * d], fused[:, 2 * hk * d:(2 * hk + hv) * d]))
    g, beta = -torch.rand(hv, T, device="cuda").t(), torch.rand(T, 2 * hv, device="cuda")[:, ::2]
    a = LA.gated_delta_rule(q, k, v, g, beta)
    b = LA.gated_delta_rule(*(t.contiguous() for t in (q, k, v, g, beta)))
    assert torch.equal(a, b)
    odd = randn(gen, T, hk * d + 1, dtype=BF16)[:, 1:].unflatten(1, (hk, d))  # rows off the 16-byte grid
    assert torch.equal(LA.gated_delta_rule(odd, k, v, g, beta), LA.gated_delta_rule(odd.contiguous(), k, v, g, beta))


def test_gated_delta_rule_bf16_gates_and_float_gradients():
    q, k, v, g, beta, do, cu = make([90], 1, 2, 128, 128)
    gb, bb = g.to(BF16).requires_grad_(), beta.to(BF16).requires_grad_()
    o = LA.gated_delta_rule(q, k, v, gb, bb)
    dg, db = torch.autograd.grad(o, [gb, bb], do)
    assert dg.dtype == db.dtype == BF16
    assert torch.equal(o, LA.gated_delta_rule(q, k, v, gb.detach().float(), bb.detach().float()))


def test_gated_delta_rule_rows_outside_the_sequences_are_zero():
    q, k, v, g, beta, do, _ = make([200], 1, 2, 128, 128)
    for bounds in ([10, 80, 150], torch.tensor([10, 80, 150], device="cuda")):
        ins = [t.detach().requires_grad_() for t in (q, k, v, g, beta)]
        o = LA.gated_delta_rule(*ins, cu_seqlens=bounds)
        grads = torch.autograd.grad(o, ins, do)
        for t in (o, *grads):
            assert t.isfinite().all() and not t[:10].any() and not t[150:].any() and t[10:150].any()
        ro, _ = oracle(q, k, v, g, beta, [10, 80, 150])
        close(o, ro, "o")


def test_gated_delta_rule_bad_device_boundaries_are_clamped_and_reported():
    q, k, v, g, beta, _, _ = make([100], 1, 2, 128, 128)
    for bad in ([0, 60, 30, 100], [0, 50, 400], [-5, 100]):
        LA.gated_delta_rule(q, k, v, g, beta, cu_seqlens=torch.tensor(bad, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            _ext.check_status()


def test_gated_delta_rule_no_tokens():
    q, k, v, g, beta, _, _ = make([0], 1, 2, 128, 128)
    s0 = torch.randn(1, 2, 128, 128, device="cuda")
    ins = [t.requires_grad_() for t in (q, k, v, g, beta, s0)]
    o, last = LA.gated_delta_rule(*ins[:5], initial_state=s0, output_final_state=True)
    assert o.shape == v.shape and torch.equal(last, s0)
    ds = torch.randn_like(s0)
    d = torch.autograd.grad([last], ins, [ds], allow_unused=True)
    assert torch.equal(d[5], ds) and d[0].shape == q.shape


def test_gated_delta_rule_final_state_alone_has_gradients():
    q, k, v, g, beta, _, cu = make([70, 20], 1, 2, 128, 128)
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    _, last = LA.gated_delta_rule(*ins, cu_seqlens=cu, output_final_state=True)
    up = torch.randn_like(last)
    got = torch.autograd.grad(last, ins, up)
    rins = [t.detach().double().requires_grad_() for t in ins]
    _, rlast = oracle(*rins, cu.tolist())
    want = torch.autograd.grad((rlast * up.double()).sum(), rins, allow_unused=True)
    assert not got[0].any()
    assert rel(got[1], want[1]) < 3 * 2.0 ** -8
    close(got[2], want[2], "dv")
    assert rel(got[3], want[3]) < 4 * 2.0 ** -17 and rel(got[4], want[4]) < 4 * 2.0 ** -17


def test_gated_delta_rule_gradient_against_differences():
    """One directional derivative of a smooth function of all inputs, by central differences of the 64-bit recurrence."""
    q, k, v, g, beta, do, cu = make([90], 1, 2, 128, 128, 9)
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    grads = torch.autograd.grad(LA.gated_delta_rule(*ins, cu_seqlens=cu), ins, do)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(5):
        d = randn(gen, *ins[i].shape).double()
        side = []
        for s in (1e-5, -1e-5):
            x = [t.detach().double() for t in ins]
            x[i] = x[i] + s * d
            side.append((oracle(*x, cu.tolist())[0] * do.double()).sum())
        want = ((side[0] - side[1]) / 2e-5).item()
        got = (grads[i].double() * d).sum().item()
        # roundings of 2^-8 of each gradient element, independent: their sum is off by 2^-8 of the 2-norm or so; three
        # of them (dq, dk), four standard deviations
        lim = (12 if i < 3 else 0.1) * 2.0 ** -8 * (grads[i].double() * d).norm().item()
        assert abs(got - want) < lim, (i, got, want, lim)


def test_gated_delta_rule_is_reproducible_and_runs_on_side_streams():
    q, k, v, g, beta, do, cu = make([500, 300], 2, 4, 128, 128)

    def run():
        ins = [t.detach().requires_grad_() for t in (q, k, v, g, beta)]
        o = LA.gated_delta_rule(*ins, cu_seqlens=cu)
        return [o.detach(), *torch.autograd.grad(o, ins, do)]

    a = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = run()
        c = run()
    s.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_gated_delta_rule_captured_forward_and_backward():
    q, k, v, g, beta, do, cu = make([100, 60], 1, 2, 128, 128)
    q2, k2, v2, g2, beta2, do2, _ = make([100, 60], 1, 2, 128, 128, 7)
    cu2 = torch.tensor([0, 30, 160], dtype=torch.int32, device="cuda")

    def run(ins):
        o = LA.gated_delta_rule(*ins, cu_seqlens=cu)
        return [o, *torch.autograd.grad(o, ins, do)]

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        run([t.detach().clone().requires_grad_() for t in (q, k, v, g, beta)])
    torch.cuda.current_stream().wait_stream(warm)
    ins = [t.detach().clone().requires_grad_() for t in (q, k, v, g, beta)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(ins)
    with torch.no_grad():
        for t, n in zip(ins, (q2, k2, v2, g2, beta2)):
            t.copy_(n)
        do.copy_(do2)
        cu.copy_(cu2)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in outs]
    want = run([t.detach().clone().requires_grad_() for t in (q2, k2, v2, g2, beta2)])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------ single tokens


@pytest.mark.parametrize("B,hk,hv,dk,dv", [(1, 2, 4, 128, 128), (3, 1, 1, 64, 128), (70, 4, 4, 128, 64), (5, 1, 3, 64, 64)])
def test_delta_step_matches_one_token(B, hk, hv, dk, dv):
    q, k, v, g, beta, _, _ = make([1] * B, hk, hv, dk, dv)
    pool = torch.randn(B + 3, hv, dk, dv, device="cuda")
    slots = torch.randperm(B + 3, device="cuda")[:B].to(torch.int32)
    want_o, want_s = oracle(q, k, v, g, beta, list(range(B + 1)), pool[slots.long()])
    kept = pool.clone()
    o = LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=slots)
    _ext.check_status()
    close(o, want_o, "o")
    assert rel(pool[slots.long()], want_s) < 4 * 2.0 ** -22  # fp32 throughout: roundings of 2^-24 and sums of 128
    rest = torch.ones(B + 3, dtype=torch.bool, device="cuda")
    rest[slots.long()] = False
    assert torch.equal(pool[rest], kept[rest])


def test_delta_step_padding_rows_and_bad_slots():
    q, k, v, g, beta, _, _ = make([1] * 5, 1, 2, 128, 128)
    pool = torch.randn(4, 2, 128, 128, device="cuda")
    kept = pool.clone()
    o = LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=torch.tensor([2, -1, 0, -1, -7], device="cuda"))
    _ext.check_status()
    assert not o[1].any() and not o[3].any() and not o[4].any() and o[0].any() and o[2].any()
    assert torch.equal(pool[[1, 3]], kept[[1, 3]]) and not torch.equal(pool[2], kept[2])
    for bad in ([0, 1, 4, -1, -1], [3, 1, 3, 0, 1 << 30]):
        kept = pool.clone()
        o = LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert not o[2].any() and o[0].any()
        assert torch.equal(pool[2], kept[2])
        with pytest.raises(RuntimeError, match="out of range"):
            _ext.check_status()


def test_delta_prefill_then_steps_match_one_pass():
    """The operators as a decoder uses them: convolution and delta rule over a prompt, then token by token."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    B, L, P, hk, hv, d, K = 3, 90, 71, 1, 2, 128, 4
    C = (2 * hk + hv) * d
    w = randn(gen, C, K, dtype=BF16, scale=0.5)
    x = randn(gen, B, L, C, dtype=BF16)
    g, beta = -torch.rand(B, L, hv, generator=gen, device="cuda"), torch.rand(B, L, hv, generator=gen, device="cuda")

    def heads(y):
        return y[:, :hk * d].unflatten(1, (hk, d)), y[:, hk * d:2 * hk * d].unflatten(1, (hk, d)), y[:, 2 * hk * d:].unflatten(1, (hv, d))

    def run(lo, hi, state):
        n = hi - lo
        cu = torch.arange(B + 1, device="cuda", dtype=torch.int32) * n
        y = LA.causal_conv1d(x[:, lo:hi].reshape(B * n, C), w, cu_seqlens=cu)
        return LA.gated_delta_rule(*heads(y), g[:, lo:hi].reshape(-1, hv), beta[:, lo:hi].reshape(-1, hv), cu_seqlens=cu,
                                   initial_state=state, output_final_state=True)

    with torch.no_grad():
        whole, last = run(0, L, None)
        first, state = run(0, P, None)
        window = x[:, P - K + 1:P].transpose(1, 2).contiguous()
        steps = []
        for t in range(P, L):
            y = LA.causal_conv1d_step(x[:, t], window, w)
            steps.append(LA.gated_delta_rule_step(*heads(y), g[:, t], beta[:, t], state))
    _ext.check_status()
    got = torch.cat([first.view(B, P, hv, d), torch.stack(steps, 1)], 1)
    close(got.reshape(B * L, hv, d), whole.double(), "o")  # two results that each are within half of it
    assert rel(state, last.double()) < 8 * 2.0 ** -17


# -------------------------------------------------------------------------------------------------------- convolution


def conv_oracle(x, w, b, bounds, silu):
    K = w.shape[1]
    out = []
    for t in range(x.shape[0]):
        lo = max([s for s, e in zip(bounds, bounds[1:]) if s <= t < e], default=None)
        if lo is None:
            out.append(torch.zeros_like(x[t]))
            continue
        y = b.clone() if b is not None else torch.zeros_like(x[t])
        for i in range(min(K, t - lo + 1)):
            y = y + w[:, K - 1 - i] * x[t - i]
        out.append(y * torch.sigmoid(y) if silu else y)
    return torch.stack(out)


@pytest.mark.parametrize("lens,C,K,bias,silu", [([1], 8, 4, True, True), ([1, 2, 3, 4, 5], 64, 4, False, True), ([40], 520, 3, True, False),
                                                ([15, 0, 17, 1, 130], 1032, 4, True, True), ([33, 64], 24, 2, False, False)])
def test_causal_conv1d_forward_and_backward(lens, C, K, bias, silu):
    gen = torch.Generator(device="cuda").manual_seed(3)
    T = sum(lens)
    bounds = [0] + torch.tensor(lens).cumsum(0).tolist()
    x, dy = randn(gen, T, C, dtype=BF16), randn(gen, T, C, dtype=BF16)
    w, b = randn(gen, C, K, dtype=BF16, scale=0.5), randn(gen, C, dtype=BF16) if bias else None
    ins = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = LA.causal_conv1d(x, w, b, cu_seqlens=torch.tensor(bounds, device="cuda"), activation="silu" if silu else None)
    grads = torch.autograd.grad(y, ins, dy)
    rins = [t.detach().double().requires_grad_() for t in ins]
    ry = conv_oracle(rins[0], rins[1], rins[2] if bias else None, bounds, silu)
    rgrads = torch.autograd.grad((ry * dy.double()).sum(), rins)
    # fp32 sums of at most T + 5 terms and one rounding at the end
    for a, r in zip((y, *grads), (ry, *rgrads)):
        lim = r.abs() * 2.0 ** -8 + r.abs().max() * 2.0 ** -16
        assert ((a.double() - r).abs() <= lim).all(), (a.double() - r).abs().max()


def test_causal_conv1d_padding_strides_and_nan_next_door():
    gen = torch.Generator(device="cuda").manual_seed(4)
    wide = randn(gen, 50, 80, dtype=BF16)
    w = randn(gen, 64, 4, dtype=BF16)
    x = wide[:, 8:72]
    assert torch.equal(LA.causal_conv1d(x, w), LA.causal_conv1d(x.contiguous(), w))
    cu = torch.tensor([5, 20, 30], device="cuda")
    y = LA.causal_conv1d(x, w, cu_seqlens=cu)
    assert not y[:5].any() and not y[30:].any()
    sick = x.clone()
    sick[19] = float("nan")  # the last token of the first sequence, and everything outside
    sick[:5] = float("nan")
    sick[30:] = float("inf")
    sick.requires_grad_()
    ys = LA.causal_conv1d(sick, w, cu_seqlens=cu)
    assert torch.equal(ys[20:30], y[20:30]) and torch.equal(ys[5:19], y[5:19]) and not ys[30:].any()
    d = torch.autograd.grad(ys[20:30].float().sum(), sick)[0]
    assert d[20:30].isfinite().all() and not d[:5].any() and not d[30:].any()
    assert LA.causal_conv1d(x[:0], w).shape == (0, 64)
    e, wr = x[:0].clone().requires_grad_(), w.clone().requires_grad_()
    dw = torch.autograd.grad(LA.causal_conv1d(e, wr).sum(), [e, wr])[1]
    assert not dw.any()


@pytest.mark.parametrize("B,C,K,bias", [(1, 8, 4, True), (4, 1032, 3, False), (9, 64, 2, True)])
def test_causal_conv1d_step(B, C, K, bias):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, state = randn(gen, B, C, dtype=BF16), randn(gen, B + 2, C, K - 1, dtype=BF16)
    w, b = randn(gen, C, K, dtype=BF16), randn(gen, C, dtype=BF16) if bias else None
    slots = torch.randperm(B + 2, device="cuda")[:B]
    win = torch.cat([state[slots], x[..., None]], -1).double()
    want = (win * w.double()).sum(-1) + (b.double() if bias else 0)
    want = want * torch.sigmoid(want)
    kept = state.clone()
    y = LA.causal_conv1d_step(x, state, w, b, state_indices=slots)
    lim = want.abs() * 2.0 ** -8 + want.abs().max() * 2.0 ** -16
    assert ((y.double() - want).abs() <= lim).all()
    assert torch.equal(state[slots], win[..., 1:].to(BF16))
    rest = torch.ones(B + 2, dtype=torch.bool, device="cuda")
    rest[slots] = False
    assert torch.equal(state[rest], kept[rest])
    _ext.check_status()
    slots[-1] = B + 2
    y = LA.causal_conv1d_step(x, state, w, b, state_indices=slots)
    assert not y[-1].any()
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()


def test_causal_conv1d_far_ends_of_silu():
    """Sums of tens of thousands either way: silu and its derivative are the sum and one, or zero and zero."""
    x = torch.tensor([[3e4, -3e4, 90.0, -90.0, 0.0, 1e-30, -1e38, 1e38]], device="cuda").to(BF16).requires_grad_()
    w = torch.zeros(8, 4, device="cuda", dtype=BF16)
    w[:, -1] = 1
    y = LA.causal_conv1d(x, w)
    d = torch.autograd.grad(y, x, torch.ones_like(y))[0]
    r = x.detach().double()
    s = torch.sigmoid(r)
    for a, b in ((y, r * s), (d, s + r * s * (1 - s))):
        assert ((a.double() - b).abs() <= b.abs() * 2.0 ** -8 + 2.0 ** -40).all(), (a, b)


def test_single_tokens_captured_and_on_a_side_stream():
    """Convolution and memory of one token as a decoder captures them: slots and inputs change between replays."""
    gen = torch.Generator(device="cuda").manual_seed(8)
    B, hk, hv, dk, dv, S, K = 3, 1, 2, 128, 128, 6, 4
    C = 2 * hk * dk + hv * dv
    x, w = randn(gen, B, C, dtype=BF16), randn(gen, C, K, dtype=BF16)
    g, beta = -torch.rand(B, hv, generator=gen, device="cuda"), torch.rand(B, hv, generator=gen, device="cuda")
    win0, mem0 = randn(gen, S, C, K - 1, dtype=BF16), randn(gen, S, hv, dk, dv)
    slots = torch.tensor([4, 0, 2], device="cuda", dtype=torch.int32)

    def token(win, mem):
        y = LA.causal_conv1d_step(x, win, w, state_indices=slots)
        q, k, v = y.split([hk * dk, hk * dk, hv * dv], -1)
        return LA.gated_delta_rule_step(q.view(B, hk, dk), k.view(B, hk, dk), v.view(B, hv, dv), g, beta, mem, state_indices=slots)

    with torch.no_grad():
        win, mem = win0.clone(), mem0.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            token(win, mem)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = token(win, mem)
        win.copy_(win0)
        mem.copy_(mem0)
        rwin, rmem = win0.clone(), mem0.clone()
        for step in range(3):
            x.copy_(randn(gen, B, C, dtype=BF16))
            slots.copy_(torch.tensor([[4, 0, 2], [1, -1, 5], [4, 3, 0]][step], dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            want = token(rwin, rmem)
            assert torch.equal(o, want) and torch.equal(win, rwin) and torch.equal(mem, rmem)
    _ext.check_status()


def test_no_rows_of_single_tokens():
    mem, win = torch.randn(2, 2, 64, 64, device="cuda"), torch.randn(2, 64, 3, device="cuda").to(BF16)
    m0, w0 = mem.clone(), win.clone()
    e = torch.empty(0, 2, 64, device="cuda", dtype=BF16)
    gates = torch.empty(0, 2, device="cuda")
    with torch.no_grad():
        assert LA.gated_delta_rule_step(e, e, e, gates, gates, mem).shape == (0, 2, 64)
        assert LA.causal_conv1d_step(e.view(0, 128)[:, :64], win, torch.zeros(64, 4, device="cuda", dtype=BF16)).shape == (0, 64)
    assert torch.equal(mem, m0) and torch.equal(win, w0)


def test_two_training_calls_at_once_on_two_streams():
    """Neither call's workspace is the other's."""
    sets = [make([700, 33], 2, 4, 128, 128, seed) for seed in (1, 2)]

    def run(s):
        q, k, v, g, beta, do, cu = s
        ins = [t.detach().requires_grad_() for t in (q, k, v, g, beta)]
        o = LA.gated_delta_rule(*ins, cu_seqlens=cu)
        return [o.detach(), *torch.autograd.grad(o, ins, do)]

    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(run(s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_wide_indices_do_not_wrap_into_range():
    """2^32 is no slot, no boundary and no row of a table, although its low 32 bits are zero."""
    from loongforge_b200.ops import functional as OF
    gen = torch.Generator(device="cuda").manual_seed(9)
    mem = randn(gen, 2, 1, 64, 64)
    m0 = mem.clone()
    x = randn(gen, 1, 1, 64, dtype=BF16)
    gate = torch.zeros(1, 1, device="cuda")
    far = torch.tensor([2 ** 32], device="cuda")
    with torch.no_grad():
        o = LA.gated_delta_rule_step(x, x, x, gate, gate + 1, mem, state_indices=far)
    assert not o.any() and torch.equal(mem, m0)
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()
    xs = randn(gen, 10, 64, dtype=BF16)
    y = LA.causal_conv1d(xs, randn(gen, 64, 4, dtype=BF16), cu_seqlens=torch.tensor([0, 2 ** 32 + 4], device="cuda"))
    assert y[4:].any()  # clamped to the ten rows
    OF.qk_norm_rope(randn(gen, 1, 192, dtype=BF16), 1, 1, *(torch.ones(64, device="cuda", dtype=BF16),) * 2,
                    freqs=torch.rand(4, 32, device="cuda"), pos_ids=far)
    with pytest.raises(RuntimeError, match="out of range"):
        _ext.check_status()


def test_one_row_out_of_a_wider_one():
    """A single row whose stride is odd, as inputs of all four operators and as the gradient that comes back."""
    gen = torch.Generator(device="cuda").manual_seed(12)
    d = 64

    def odd(*shape):  # the first elements of a row that is three longer
        n = shape[-1]
        for s in shape[1:-1]:
            n *= s
        return randn(gen, 1, n + 3, dtype=BF16)[:, :n].unflatten(1, shape[1:]) if len(shape) > 2 else randn(gen, 1, n + 3, dtype=BF16)[:, :n]

    for hv in (1, 2):
        q, k, v, up = odd(1, 1, d), odd(1, 1, d), odd(1, hv, d), odd(1, hv, d)
        g, beta = -torch.rand(1, hv, device="cuda"), torch.rand(1, hv, device="cuda")
        rows = [t.detach().requires_grad_() for t in (q, k, v)]
        same = [t.clone(memory_format=torch.contiguous_format).requires_grad_() for t in (q, k, v)]
        a, b = (LA.gated_delta_rule(*t, g, beta) for t in (rows, same))
        da, db = torch.autograd.grad(a, rows, up), torch.autograd.grad(b, same, up.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(da, db))
        s1, s2 = torch.ones(1, hv, d, d, device="cuda"), torch.ones(1, hv, d, d, device="cuda")
        with torch.no_grad():
            assert torch.equal(LA.gated_delta_rule_step(q, k, v, g, beta, s1), LA.gated_delta_rule_step(*same, g, beta, s2))
        assert torch.equal(s1, s2)
    x, up, w = odd(1, d), odd(1, d), randn(gen, d, 4, dtype=BF16)
    xs = [x.detach().requires_grad_(), x.clone(memory_format=torch.contiguous_format).requires_grad_()]
    y = [LA.causal_conv1d(t, w) for t in xs]
    dx = [torch.autograd.grad(t, u, up)[0] for t, u in zip(y, xs)]
    assert torch.equal(*y) and torch.equal(*dx)
    w1, w2 = (torch.ones(1, d, 3, device="cuda", dtype=BF16) for _ in range(2))
    with torch.no_grad():
        assert torch.equal(LA.causal_conv1d_step(x, w1, w), LA.causal_conv1d_step(xs[1], w2, w))
    assert torch.equal(w1, w2)


def test_bad_slots_where_no_kernel_covers_the_step():
    """fp32 rows take the PyTorch form, which reads the slots: it refuses what the kernel would leave out."""
    gen = torch.Generator(device="cuda").manual_seed(13)
    q, k, v = (randn(gen, 2, 1, 16) for _ in range(3))
    g, x, w = torch.zeros(2, 1, device="cuda"), randn(gen, 2, 12), randn(gen, 12, 4)
    pool, win = randn(gen, 3, 1, 16, 16), randn(gen, 3, 12, 3)
    kept = pool.clone(), win.clone()
    for bad in ([1, 1], [0, 3], [2 ** 32, 0]):
        idx = torch.tensor(bad, device="cuda")
        with pytest.raises(ValueError, match="state_indices"):
            LA.gated_delta_rule_step(q, k, v, g, g + 1, pool, state_indices=idx)
        with pytest.raises(ValueError, match="state_indices"):
            LA.causal_conv1d_step(x, win, w, state_indices=idx)
    assert torch.equal(pool, kept[0]) and torch.equal(win, kept[1])
    idx = torch.tensor([2, -1], device="cuda")
    o = LA.gated_delta_rule_step(q, k, v, g, g + 1, pool, state_indices=idx)
    assert o[0].any() and not o[1].any() and torch.equal(pool[:2], kept[0][:2])
    with pytest.raises(ValueError, match="whole"):
        LA.causal_conv1d_step(x, win, w, state_indices=idx.float())


@pytest.mark.parametrize("strong", [-30.0, -8.0])
def test_gated_delta_rule_resets_among_mild_decays(strong):
    """The gradient of a reset is next to nothing, and what comes back is the rounding of the terms that cancel in it: o . do
    and v . dv of the tokens behind it, each off by up to 4 * 2^-17 of itself, independently, so their 2-norm. The gradient
    of a rate that multiplies all decays weighs these with g."""
    q, k, v, g, beta, do, cu = make([250], 2, 4, 128, 128, 21, decay=0.05)
    hit = torch.rand(250, 4, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.06
    g[hit] = strong
    ins = [t.requires_grad_() for t in (q, k, v, g, beta)]
    got = torch.autograd.grad(LA.gated_delta_rule(*ins, cu_seqlens=cu), ins, do)
    rins = [t.detach().double().requires_grad_() for t in ins]
    ro, _ = oracle(*rins, [0, 250])
    want = torch.autograd.grad((ro * do.double()).sum(), rins)
    terms = ((ro * do.double()).sum(-1).square() + (rins[2] * want[2]).sum(-1).square()).sum(0).sqrt()
    lim = 4 * 2.0 ** -17 * terms
    off = (got[3].double() - want[3]).abs()
    assert (torch.where(hit, off, 0.0) <= lim).all(), (off[hit].max(), lim)
    rate = (g.detach().double() * (got[3].double() - want[3])).sum(0).abs()
    assert (rate <= lim * g.detach().double().norm(dim=0)).all(), (rate, lim)
    assert rel(got[3], want[3]) < 4 * 2.0 ** -17


def test_gated_delta_rule_long_memory():
    """Heads as training leaves some: decays near one over thousands of tokens, where a state is the sum of hundreds."""
    check([2100], 1, 2, decay=1e-3)


@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
def test_gated_delta_rule_gradients_of_strided_rows(dk, dv):
    """q, k and v as the layer cuts them out of the convolution's rows, and an upstream gradient laid out otherwise."""
    gen = torch.Generator(device="cuda").manual_seed(14)
    T, hk, hv = 150, 2, 4
    rows = randn(gen, T, 2 * hk * dk + hv * dv, dtype=BF16).requires_grad_()
    g, beta = -torch.rand(T, hv, device="cuda"), torch.rand(T, hv, device="cuda")
    cu = torch.tensor([0, 70, 150], device="cuda")
    up = randn(gen, hv, T, dv, dtype=BF16).transpose(0, 1)
    cut = lambda x: (x[:, :hk * dk].view(T, hk, dk), x[:, hk * dk:2 * hk * dk].view(T, hk, dk), x[:, 2 * hk * dk:].view(T, hv, dv))  # noqa: E731
    o = LA.gated_delta_rule(*cut(rows), g, beta, cu_seqlens=cu)
    got = torch.autograd.grad(o, rows, up)[0]
    whole = [t.detach().contiguous().requires_grad_() for t in cut(rows)]
    want = torch.autograd.grad(LA.gated_delta_rule(*whole, g, beta, cu_seqlens=cu), whole, up.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(cut(got), want))


def test_gated_delta_rule_without_gradients_gives_the_same_bits():
    q, k, v, g, beta, _, cu = make([100, 0, 130], 2, 4, 128, 128, 16)
    s0 = torch.randn(3, 4, 128, 128, device="cuda")
    with torch.no_grad():
        a = LA.gated_delta_rule(q, k, v, g, beta, cu_seqlens=cu, initial_state=s0, output_final_state=True)
    b = LA.gated_delta_rule(q.requires_grad_(), k, v, g, beta, cu_seqlens=cu, initial_state=s0, output_final_state=True)
    assert b[0].requires_grad and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gated_delta_rule_does_not_read_what_memory_held():
    """Another call's buffers, and buffers full of NaN, where this call's come to lie."""
    q, k, v, g, beta, do, cu = make([1, 2, 63, 64, 65, 130], 2, 4, 128, 128, 17)
    other = make([200, 125], 2, 4, 128, 128, 18)

    def run(q, k, v, g, beta, do, cu):
        ins = [t.detach().requires_grad_() for t in (q, k, v, g, beta)]
        o, last = LA.gated_delta_rule(*ins, cu_seqlens=cu, output_final_state=True)
        return [o.detach(), last.detach(), *torch.autograd.grad(o, ins, do)]

    want = run(q, k, v, g, beta, do, cu)
    run(*other)
    got = run(q, k, v, g, beta, do, cu)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for fill in (float("nan"), 3e38):
        del got
        junk = [torch.full((n,), fill, device="cuda") for n in (1 << 25, 1 << 23, 1 << 21, 1 << 19, 1 << 17) * 3]
        del junk
        got = run(q, k, v, g, beta, do, cu)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
