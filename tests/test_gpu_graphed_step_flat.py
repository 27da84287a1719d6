"""A captured step with a flat optimizer, and no reducer named, takes that optimizer's own: every replay starts from zeroed
gradients."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200.ladder_lm import LadderLM, zipf_tokens
from elman_b200.train_step import FlatAdamW, FlatMuon, GraphedTrainStep, hidden_matrices, make_gradient_reducer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["muon", "adamw"])
def test_replays_do_not_add_up_gradients(kind):
    batches = [zipf_tokens(2, 65, seed=k).cuda() for k in range(4)]
    runs = []
    for named in (True, False):
        torch.manual_seed(5)
        model = LadderLM(vocab_size=256, dim=64, depth=2, level="gated_linear").cuda()
        red = make_gradient_reducer(model)
        opt = FlatMuon(red, hidden_matrices(model), lr=0.01) if kind == "muon" else FlatAdamW(red, lr=1e-3)
        step = GraphedTrainStep(model, opt, batches[0], max_grad_norm=1.0, warmup_steps=2, reducer=red if named else None)
        losses = [float(step(tok)) for tok in batches]
        runs.append((losses, red.flat.clone()))
        step.graph = None
        red.close()
    (a, ga), (b, gb) = runs
    assert all(abs(x - y) < 1e-3 * abs(x) for x, y in zip(a, b)), (a, b)
    assert float((ga - gb).norm()) < 1e-2 * float(ga.norm())
    assert _lib.device_status()[0] == 0
