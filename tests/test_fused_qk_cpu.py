"""When the attention layers take query / key norms and rotation as one kernel."""
import pytest
import torch


@pytest.mark.parametrize("gated", [False, True])
def test_watched_norms_are_called(gated, monkeypatch, tmp_path):
    """The one-pass kernel takes the weights of the norms: a module with hooks on it is called instead, so that what
    watches it (statistics, dumps) sees every tensor."""
    from loongforge_b200.models import hybrid, transformer
    from loongforge_b200.models.registry import get_model_config
    from loongforge_b200.ops import functional as OF
    from loongforge_b200.parallel import state as ps
    from loongforge_b200.runtime.profiling import TensorInspector

    ps.destroy_model_parallel()
    ps.initialize_model_parallel(ps.ParallelDims())
    cfg = get_model_config("tiny-qwen3-next", params_dtype=torch.float32, qk_layernorm=True)
    cls = hybrid.GatedAttention if gated else transformer.SelfAttention
    net = cls(cfg, "decoder.layers.3.self_attention", device="cpu", **({} if gated else {"fused_norm": False}))
    monkeypatch.setattr(OF, "qk_norm_rope_supported", lambda *a, **k: True)  # as for bf16 on a GPU
    calls = []
    one = OF.qk_norm_rope
    monkeypatch.setattr(OF, "qk_norm_rope", lambda *a, **k: calls.append(1) or one(*a, **k))
    x = torch.randn(12, cfg.hidden_size)
    rotary = transformer.RotaryInputs(freqs=OF.rope_freqs(torch.arange(12), net.rot_dim, 1e4))
    want = net(x, rotary, None)
    assert len(calls) == 1
    for name in ("q_layernorm", "k_layernorm"):
        seen = TensorInspector(net, [name], str(tmp_path / f"{name}.jsonl"))
        y = net(x, rotary, None)
        y.sum().backward()
        assert len(calls) == 1 and {r["kind"] for r in seen.records} == {"fwd", "bwd"}
        assert torch.allclose(y, want, atol=1e-5)  # the same in fp32 but for the order of sums
        for h in seen.handles:
            h.remove()
        assert torch.equal(net(x, rotary, None), want)
        calls.pop()
