"""The gated linear layer and the Muon optimizer, as far as they go without a GPU."""
import pytest
import torch

from elman_b200 import ladder_lm
from elman_b200.gated_linear import GatedLinearElman
from elman_b200.train_step import FlatGradients, FlatMuon, hidden_matrices


def test_level_and_parameters():
    assert ladder_lm.get_ladder_level("gated_linear") is GatedLinearElman
    model = ladder_lm.LadderLM(vocab_size=64, dim=24, depth=2, level="gated_linear", expansion=1.5)
    names = {k.split(".", 2)[2] for k in model.state_dict() if k.startswith("layers.")}
    assert names == {"in_proj.weight", "in_proj.bias", "out_proj.weight"}
    assert model.layers[0].in_proj.weight.shape == (108, 24) and model.layers[0].d_inner == 36
    for bad in ("gated", 7, "7"):
        with pytest.raises(ValueError, match="gated_linear"):
            ladder_lm.get_ladder_level(bad)
    with pytest.raises(ValueError, match="convolution"):
        GatedLinearElman(8, use_conv=True)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        GatedLinearElman(8)(torch.zeros(1, 2, 8))
    layer = torch.nn.Linear(4, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        FlatMuon(FlatGradients([list(layer.parameters())]), [layer.weight])


def test_reset_is_refused_by_the_other_levels():
    model = ladder_lm.LadderLM(vocab_size=64, dim=16, depth=1, level=1)
    with pytest.raises(ValueError, match="gated_linear"):
        model(torch.zeros(1, 3, dtype=torch.long), reset=torch.zeros(1, 3, dtype=torch.bool))


def test_hidden_matrices_are_the_layers_own():
    model = ladder_lm.LadderLM(vocab_size=64, dim=16, depth=2, level=1)
    mats = hidden_matrices(model)
    assert all(p.dim() == 2 for p in mats) and all(p is not model.embedding.weight for p in mats)
    assert len(mats) == 2 * 4       # in_proj, W_x, W_h, out_proj
    model.layers[0].out_proj.weight.requires_grad_(False)
    assert len(hidden_matrices(model)) == 7
    assert hidden_matrices(torch.nn.Linear(2, 2)) == []
