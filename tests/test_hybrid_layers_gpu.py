"""Hybrid layers on the kernels: decoding through the cache, and the fused query / key norm + rotation against the
separate passes in both attention layers, outputs and gradients."""
import pytest
import torch

from test_hybrid_decode_cpu import decode_against_forward, layer

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("d", [64, 128])
def test_linear_attention_layer_decodes_on_the_gpu(d):
    cfg, net = layer("cuda", BF16, linear_key_head_dim=d, linear_value_head_dim=d)
    # projections, norm and output round to bf16 in both orders: a handful of roundings of 2^-8 each
    decode_against_forward(cfg, net, "cuda", BF16, 6 * 2.0 ** -8)
    from loongforge_b200.ops import _ext
    _ext.check_status()


@pytest.mark.parametrize("kind", ["qwen3", "gated", "gated 3 axes"])
def test_attention_layers_fused_norm_and_rotation(kind, monkeypatch):
    from loongforge_b200.models import hybrid, transformer
    from loongforge_b200.models.gpt import RotaryEmbedding
    from loongforge_b200.models.registry import get_model_config
    from loongforge_b200.ops import _ext
    from loongforge_b200.parallel import state as ps

    ps.destroy_model_parallel()
    ps.initialize_model_parallel(ps.ParallelDims())
    ov = dict(params_dtype=BF16, kv_channels=64, qk_layernorm=True)
    if "axes" in kind:
        ov.update(position_embedding_type="mrope", mrope_section=[6, 5, 5], mrope_interleaved=True, rotary_percent=0.5)
    cfg = get_model_config("tiny-qwen3-next", **ov)
    cls = transformer.SelfAttention if kind == "qwen3" else hybrid.GatedAttention
    net = cls(cfg, "decoder.layers.3.self_attention", device="cuda",
              **({"fused_norm": False} if kind == "qwen3" else {}))
    torch.manual_seed(3)
    T = 150
    for p in (net.q_layernorm.weight, net.k_layernorm.weight):
        p.data.copy_(torch.randn_like(p) * 0.2 + 1 - net.q_layernorm.offset)
    rot = RotaryEmbedding(cfg, net.rot_dim)
    rotary = rot.mrope(torch.randint(0, 300, (3, T), device="cuda")) if "axes" in kind else rot.table(T, "cuda")
    x, up = torch.randn(T, cfg.hidden_size, device="cuda").to(BF16), torch.randn(T, cfg.hidden_size, device="cuda").to(BF16)

    def run():
        xi = x.clone().requires_grad_()
        params = list(net.parameters())
        y = net(xi, rotary, None)
        return [y.detach(), *torch.autograd.grad(y, [xi, *params], up)]

    calls = []
    from loongforge_b200.ops import functional as OF
    one = OF.qk_norm_rope
    monkeypatch.setattr(OF, "qk_norm_rope", lambda *a, **k: calls.append(1) or one(*a, **k))
    fused = run()
    assert calls
    monkeypatch.setattr(transformer, "fused_qk_applies", lambda *a, **k: False)
    monkeypatch.setattr(hybrid, "fused_qk_applies", lambda *a, **k: False)
    apart = run()
    assert len(calls) == 1
    _ext.check_status()
    # q and k are rounded once instead of twice (2^-8 each), which goes through a softmax of scores of order ten: up to
    # ten such roundings relative to the probabilities, and as many again in the gradients
    for a, b in zip(fused, apart):
        assert (a.float() - b.float()).norm() < 20 * 2.0 ** -8 * b.float().norm()


@pytest.mark.parametrize("d", [64, 128])
def test_linear_attention_layer_trains_on_the_gpu(d, monkeypatch):
    """Outputs and gradients of the layer over a packed row, on the kernels and with the delta rule and the convolution in
    their PyTorch form on the same GPU, which differ by roundings to bf16."""
    from loongforge_b200.models.transformer import PackedSeqParams
    from loongforge_b200.ops import _ext
    from loongforge_b200.ops import linear_attn as LA

    cfg, net = layer("cuda", BF16, linear_key_head_dim=d, linear_value_head_dim=d)
    torch.manual_seed(5)
    lens = [70, 1, 130]
    x, up = (torch.randn(sum(lens), cfg.hidden_size, device="cuda").to(BF16) for _ in range(2))
    cu = torch.tensor([0] + lens).cumsum(0).to(device="cuda", dtype=torch.int32)

    def run():
        xi = x.clone().requires_grad_()
        params = list(net.parameters())
        y = net(xi, packed=PackedSeqParams(cu_seqlens=cu))
        return [y.detach(), *torch.autograd.grad(y, [xi, *params], up)]

    _ext.reset_launch_count()
    on = run()
    assert _ext.launch_count() >= 8  # convolution 1 + 2, delta rule 3 + 3 and their neighbours
    _ext.check_status()
    monkeypatch.setattr(LA, "gated_delta_rule_native", lambda *a: False)
    monkeypatch.setattr(LA, "_conv_native", lambda *a: False)
    off = run()
    # the convolution's sum and its activation are rounded apart in the PyTorch form, q, k and v once more each; projections,
    # norm and gates round in both: a handful of roundings of 2^-8, as in decoding, twice over on the way back
    for n, a, b in zip(["y", "x"] + [n for n, _ in net.named_parameters()], on, off):
        assert (a.float() - b.float()).norm() < 12 * 2.0 ** -8 * b.float().norm(), (n, (a.float() - b.float()).norm() / b.float().norm())
