"""Linear-attention layer: prompts and single tokens through its cache give what one pass over the row gives."""
import pytest
import torch


def layer(device="cpu", dtype=torch.float32, **ov):
    from loongforge_b200.models.hybrid import GatedDeltaNet
    from loongforge_b200.models.registry import get_model_config
    from loongforge_b200.parallel import state as ps

    ps.destroy_model_parallel()
    ps.initialize_model_parallel(ps.ParallelDims())
    cfg = get_model_config("tiny-qwen3-next", params_dtype=dtype, **ov)
    torch.manual_seed(0)
    return cfg, GatedDeltaNet(cfg, "decoder.layers.0.self_attention", device=device)


def decode_against_forward(cfg, net, device, dtype, tol):
    from loongforge_b200.models.transformer import PackedSeqParams

    torch.manual_seed(1)
    lens, more = [9, 1, 70], 6  # a prompt shorter than the convolution's window among them
    rows = [torch.randn(n + more, cfg.hidden_size, dtype=dtype).to(device) for n in lens]
    cu = torch.tensor([0] + [n + more for n in lens]).cumsum(0).to(device=device, dtype=torch.int32)
    with torch.no_grad():
        want = net(torch.cat(rows), packed=PackedSeqParams(cu_seqlens=cu)).split([n + more for n in lens])
    cache = net.new_cache(5)
    slots = [3, 0, 4]
    pcu = torch.tensor([0] + lens).cumsum(0).to(device=device, dtype=torch.int32)
    first = net.prefill(torch.cat([r[:n] for r, n in zip(rows, lens)]), cache, slots, cu_seqlens=pcu).split(lens)
    got = [[f] for f in first]
    idx = torch.tensor(slots + [-1], device=device, dtype=torch.int32)  # a padding row at the end of the batch
    for t in range(more):
        x = torch.stack([r[n + t] for r, n in zip(rows, lens)] + [torch.zeros(cfg.hidden_size, dtype=dtype, device=device)])
        y = net.step(x, cache, slots=idx)
        for i in range(3):
            got[i].append(y[i:i + 1])
    for g, w in zip(got, want):
        g = torch.cat(g).float()
        assert (g - w.float()).norm() < tol * w.float().norm()
    for c in cache:
        assert not c[1].any() and not c[2].any() and c[0].any()


def test_linear_attention_layer_decodes_what_it_trains_on():
    cfg, net = layer()
    decode_against_forward(cfg, net, "cpu", torch.float32, 1e-4)


def test_prefill_refuses_a_wrong_number_of_slots():
    cfg, net = layer()
    with pytest.raises(ValueError, match="slots"):
        net.prefill(torch.randn(8, cfg.hidden_size), net.new_cache(4), [0], cu_seqlens=[0, 3, 8])


@pytest.mark.parametrize("slots", [[0, 0], [0, 4], [-1, 2], torch.tensor([1, 7])])
def test_prefill_refuses_slots_that_are_taken_twice_or_not_there(slots):
    cfg, net = layer()
    cache = net.new_cache(4)
    with pytest.raises(ValueError, match="slots"):
        net.prefill(torch.randn(8, cfg.hidden_size), cache, slots, cu_seqlens=[0, 3, 8])
    assert not cache[0].any() and not cache[1].any()


def test_positions_that_are_not_whole_numbers_keep_to_the_angle_table():
    from loongforge_b200.models.gpt import RotaryEmbedding
    from loongforge_b200.models.registry import get_model_config

    cfg = get_model_config("tiny-qwen3-next", position_embedding_type="mrope", mrope_section=[3, 3, 2], mrope_interleaved=True)
    r = RotaryEmbedding(cfg, 16).mrope(torch.rand(3, 20) * 9)
    assert r.axis_pos is None and r.freqs.shape == (20, 8)


def test_gated_attention_and_mrope_inputs_agree_on_the_angles():
    """The several-axis form of the rotary inputs names the same angles as the table beside it."""
    from loongforge_b200.models.gpt import RotaryEmbedding
    from loongforge_b200.models.registry import get_model_config

    for il, sec in ((True, [3, 3, 2]), (False, [2, 3, 3])):
        cfg = get_model_config("tiny-qwen3-next", position_embedding_type="mrope", mrope_section=sec, mrope_interleaved=il)
        r = RotaryEmbedding(cfg, 16).mrope(torch.randint(0, 1000, (3, 20)))
        ang = r.axis_pos.double()[r.axis.long()].t() * r.inv_freq.double()
        assert torch.allclose(ang.float(), r.freqs, rtol=2.0 ** -23, atol=0)


def test_prefill_refuses_slots_that_are_not_whole():
    cfg, net = layer()
    cache = net.new_cache(4)
    for slots in ([0, 1.5], torch.tensor([0.0, 1.0])):
        with pytest.raises(TypeError):
            net.prefill(torch.randn(8, cfg.hidden_size), cache, slots, cu_seqlens=[0, 3, 8])
    assert not cache[0].any() and not cache[1].any()
