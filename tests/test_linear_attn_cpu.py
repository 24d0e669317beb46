"""Linear-attention operators on the CPU: the PyTorch forms with states, shared heads and single tokens, and refusals."""
import pytest
import torch

from loongforge_b200.ops import linear_attn as LA


def make(T=90, hk=2, hv=4, dk=16, dv=8, seed=0):
    torch.manual_seed(seed)
    q, k, v = torch.randn(T, hk, dk), torch.randn(T, hk, dk), torch.randn(T, hv, dv)
    return q, k, v, -torch.rand(T, hv), torch.rand(T, hv)


def test_shared_key_heads_equal_repeated_ones():
    q, k, v, g, beta = make()
    rq, rk = q.repeat_interleave(2, 1), k.repeat_interleave(2, 1)
    assert torch.equal(LA.gated_delta_rule(q, k, v, g, beta), LA.gated_delta_rule(rq, rk, v, g, beta))
    assert torch.equal(LA.gated_delta_rule_recurrent(q, k, v, g, beta), LA.gated_delta_rule_recurrent(rq, rk, v, g, beta))


def test_states_carry_a_sequence_over_and_steps_continue_it():
    q, k, v, g, beta = make()
    whole, last = LA.gated_delta_rule(q, k, v, g, beta, output_final_state=True)
    first, mid = LA.gated_delta_rule(q[:50], k[:50], v[:50], g[:50], beta[:50], output_final_state=True)
    second, end = LA.gated_delta_rule(q[50:], k[50:], v[50:], g[50:], beta[50:], initial_state=mid, output_final_state=True)
    # fp32 sums of some hundred terms of order one, in another order
    assert torch.allclose(torch.cat([first, second]), whole, atol=1e-4) and torch.allclose(end, last, atol=1e-4)
    pool = torch.zeros(3, 4, 16, 8)
    pool[1] = mid[0]
    steps = [LA.gated_delta_rule_step(*(t[i:i + 1] for t in (q, k, v, g, beta)), pool, state_indices=[1]) for i in range(50, 90)]
    assert torch.allclose(torch.cat(steps), whole[50:], atol=1e-4) and torch.allclose(pool[1], last[0], atol=1e-4)
    assert not pool[0].any() and not pool[2].any()


def test_rows_outside_the_sequences_and_empty_ones():
    q, k, v, g, beta = make()
    s0 = torch.randn(3, 4, 16, 8)
    o, last = LA.gated_delta_rule(q, k, v, g, beta, cu_seqlens=[10, 40, 40, 70], initial_state=s0, output_final_state=True)
    assert o.shape == v.shape and not o[:10].any() and not o[70:].any() and o[10:70].any()
    assert torch.equal(last[1], s0[1])
    x = torch.randn(20, 6)
    w = torch.randn(6, 4)
    y = LA.causal_conv1d(x, w, cu_seqlens=[2, 9, 15])
    assert y.shape == x.shape and not y[:2].any() and not y[15:].any()
    assert torch.allclose(y[2:15], LA.causal_conv1d(x[2:15], w, cu_seqlens=[0, 7, 13]))


def test_conv_steps_continue_a_sequence():
    torch.manual_seed(1)
    x, w, b = torch.randn(12, 6), torch.randn(6, 4), torch.randn(6)
    want = LA.causal_conv1d(x, w, b)
    state = torch.zeros(2, 6, 3)
    state[1] = x[5:8].t()
    for t in range(8, 12):
        y = LA.causal_conv1d_step(x[t:t + 1], state, w, b, state_indices=torch.tensor([1]))
        assert torch.allclose(y[0], want[t], atol=1e-5)
    assert torch.equal(state[1], x[9:12].t()) and not state[0].any()


def test_step_padding_rows_touch_nothing():
    q, k, v, g, beta = make(T=3)
    pool = torch.randn(2, 4, 16, 8)
    kept = pool.clone()
    o = LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=[-1, 1, -1])
    assert not o[0].any() and not o[2].any() and o[1].any()
    assert torch.equal(pool[0], kept[0]) and not torch.equal(pool[1], kept[1])


@pytest.mark.parametrize("bad", [[0], [0, 50, 40, 90], [-1, 90], [0, 91], torch.tensor([0, 100])])
def test_bad_boundaries_are_refused(bad):
    q, k, v, g, beta = make()
    with pytest.raises(ValueError, match="cu_seqlens"):
        LA.gated_delta_rule(q, k, v, g, beta, cu_seqlens=bad)
    with pytest.raises(ValueError, match="cu_seqlens"):
        LA.causal_conv1d(torch.randn(90, 6), torch.randn(6, 4), cu_seqlens=bad)


def test_bad_shapes_are_refused():
    q, k, v, g, beta = make()
    s = torch.zeros(90, 4, 16, 8)
    for args in ((q, k[:, :1], v, g, beta), (q, k, v[:80], g, beta), (q, k, v[:, :3], g[:, :3], beta[:, :3]), (q, k, v, g[:, :1], beta),
                 (q, k, v, g, beta.t()), (q[0], k[0], v, g, beta)):
        with pytest.raises(ValueError):
            LA.gated_delta_rule(*args)
        with pytest.raises(ValueError):
            LA.gated_delta_rule_step(*args, s)
    for state in (torch.zeros(2, 4, 16, 8), torch.zeros(1, 4, 8, 16), torch.zeros(1, 4, 16, 8, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="initial_state"):
            LA.gated_delta_rule(q, k, v, g, beta, initial_state=state)


def test_bad_slots_and_states_are_refused():
    q, k, v, g, beta = make(T=3)
    pool = torch.zeros(4, 4, 16, 8)
    for idx in ([0, 1], [0, 1, 4], [2, 1, 2], torch.tensor([3, 3, 3])):
        with pytest.raises(ValueError, match="state_indices"):
            LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=idx)
    with pytest.raises(ValueError, match="slots"):
        LA.gated_delta_rule_step(q, k, v, g, beta, pool[:2])
    with pytest.raises(ValueError, match="contiguous"):
        LA.gated_delta_rule_step(q, k, v, g, beta, torch.zeros(4, 4, 8, 16).transpose(2, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        LA.gated_delta_rule_step(q.requires_grad_(), k, v, g, beta, pool)
    x, w = torch.randn(3, 6), torch.randn(6, 4)
    for st in (torch.zeros(3, 6, 4), torch.zeros(3, 5, 3), torch.zeros(3, 6, 3, dtype=torch.float64)):
        with pytest.raises(ValueError, match="state"):
            LA.causal_conv1d_step(x, st, w)
    with pytest.raises(ValueError, match="activation"):
        LA.causal_conv1d(x, w, activation="relu")
    with pytest.raises(ValueError):
        LA.causal_conv1d(x, w[:5])
    with pytest.raises(ValueError, match="bias"):
        LA.causal_conv1d(x, w, torch.zeros(5))


def test_numbers_that_are_not_whole_are_refused():
    q, k, v, g, beta = make(T=3)
    pool, x, w = torch.zeros(4, 4, 16, 8), torch.randn(3, 6), torch.randn(6, 4)
    for idx in (torch.tensor([0.0, 1.0, 2.0]), torch.tensor([0.5, 1.5, 2.5], dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="state_indices must be whole"):
            LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=idx)
        with pytest.raises(ValueError, match="state_indices must be whole"):
            LA.causal_conv1d_step(x, torch.zeros(3, 6, 3), w, state_indices=idx)
    for cu in (torch.tensor([0.0, 3.0]), torch.tensor([0.0, 1.5, 3.0])):
        with pytest.raises(ValueError, match="cu_seqlens must be whole"):
            LA.gated_delta_rule(q, k, v, g, beta, cu_seqlens=cu)
        with pytest.raises(ValueError, match="cu_seqlens must be whole"):
            LA.causal_conv1d(x, w, cu_seqlens=cu)
    with pytest.raises(TypeError):
        LA.gated_delta_rule_step(q, k, v, g, beta, pool, state_indices=[0, 1.5, 2])
    with pytest.raises(TypeError):
        LA.causal_conv1d(x, w, cu_seqlens=[0, 1.5, 3])
