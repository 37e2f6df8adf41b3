"""What FusedLlamaStep takes of a model (host logic, no GPU)."""
import pytest
import torch

from serving_engine_b200.e2e import random_llama
from serving_engine_b200.llama_step import FusedLlamaStep


class Norm(torch.nn.Module):
    """RMSNorm of a head by scale(weight), with its roundings as common models have them."""

    def __init__(self, weight, eps, scale=lambda w: w, centre=False):
        super().__init__()
        self.weight, self.eps, self.scale, self.centre = torch.nn.Parameter(weight), eps, scale, centre

    def forward(self, x):
        y = x.float()
        y = y - y.mean(-1, keepdim=True) if self.centre else y
        y = y * (y.square().mean(-1, keepdim=True) + self.eps).rsqrt()
        return self.scale(self.weight) * y.to(x.dtype)


def model_with(**kw):
    model = random_llama("tiny", 0, torch.bfloat16, "cpu")
    d = model.config.hidden_size // model.config.num_attention_heads
    w = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(0))).bfloat16()
    for layer in model.model.layers:
        layer.self_attn.q_norm = Norm(w, **{"eps": model.config.rms_norm_eps, **kw})
        layer.self_attn.k_norm = Norm(w.flip(0), model.config.rms_norm_eps)
    return model


def test_head_norms_that_are_taken():
    step = FusedLlamaStep(model_with())
    assert all(layer["qn"] is not None and layer["kn"] is not None for layer in step.layers)
    step = FusedLlamaStep(random_llama("tiny", 0, torch.bfloat16, "cpu"))
    assert all(layer["qn"] is None and layer["kn"] is None for layer in step.layers)


@pytest.mark.parametrize("kw", [{"scale": lambda w: 1 + w}, {"centre": True}, {"eps": 1e-2},
                                {"scale": lambda w: w * w.numel() ** 0.5}])
def test_head_norms_that_are_refused(kw):
    """One by 1 + weight, a LayerNorm, another eps, another factor: qk_norm_rope_append would answer wrongly."""
    with pytest.raises(ValueError, match="not an RMSNorm"):
        FusedLlamaStep(model_with(**kw))


def test_head_norms_over_all_heads_are_refused():
    model = random_llama("tiny", 0, torch.bfloat16, "cpu")
    model.model.layers[0].self_attn.q_norm = Norm(torch.ones(model.config.hidden_size).bfloat16(), 1e-6)
    with pytest.raises(ValueError, match="norm weights"):
        FusedLlamaStep(model)
