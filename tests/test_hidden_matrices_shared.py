"""Layers that are one and the same, or share a matrix, give Muon that matrix once."""
from elman_b200.ladder_lm import LadderLM
from elman_b200.train_step import hidden_matrices


def test_a_shared_layer_counts_once():
    model = LadderLM(vocab_size=64, dim=16, depth=3, level="gated_linear")
    assert len(hidden_matrices(model)) == 6
    model.layers[2] = model.layers[0]
    model.layers[1].out_proj.weight = model.layers[0].out_proj.weight
    mats = hidden_matrices(model)
    assert [id(p) for p in mats] == [id(p) for p in (model.layers[0].in_proj.weight, model.layers[0].out_proj.weight,
                                                     model.layers[1].in_proj.weight)]
