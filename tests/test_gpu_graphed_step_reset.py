"""Packed documents in a captured training step: every replay takes its own reset mask."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200.ladder_lm import LadderLM, zipf_tokens
from elman_b200.train_step import FlatMuon, GraphedTrainStep, hidden_matrices, make_gradient_reducer

pytestmark = pytest.mark.gpu


def test_captured_steps_follow_eager_ones_on_packed_documents():
    batches = [zipf_tokens(3, 130, seed=60 + k).cuda() for k in range(4)]
    masks = [(torch.rand(3, 130, generator=torch.Generator().manual_seed(k)) < 0.1).cuda() for k in range(4)]

    def make():
        torch.manual_seed(9)
        model = LadderLM(vocab_size=256, dim=64, depth=2, level="gated_linear").cuda()
        red = make_gradient_reducer(model)
        return model, red, FlatMuon(red, hidden_matrices(model), lr=0.01, adamw_lr=1e-3)

    model, red, opt = make()
    eager, without = [], []
    for tok, reset in [(batches[0], masks[0])] * 2 + list(zip(batches, masks)):
        red.zero()
        with torch.no_grad():
            without.append(float(model(tok, return_loss=True)))
        loss = model(tok, return_loss=True, reset=reset)
        loss.backward()
        red.finish()
        opt.step(grad_scale=red.clip_coef(1.0)[0])
        eager.append(float(loss.detach()))
    red.close()
    del loss
    model, red, opt = make()
    step = GraphedTrainStep(model, opt, batches[0], warmup_steps=2, reducer=red, example_reset=masks[0])
    graphed = [float(step(tok, reset)) for tok, reset in zip(batches, masks)]
    # the same kernels on the same numbers; sums of the embedding's gradient may be ordered otherwise
    assert all(abs(a - b) < 1e-4 * abs(a) for a, b in zip(eager[2:], graphed)), (eager, graphed)
    assert any(abs(a - b) > 1e-3 * abs(a) for a, b in zip(eager[2:], without[2:]))
    for bad in (None, masks[0][:, :-1]):
        with pytest.raises(ValueError, match="reset"):
            step(batches[0], bad)
    step.graph = None
    red.close()
    model, red, opt = make()
    step = GraphedTrainStep(model, opt, batches[0], warmup_steps=2, reducer=red)
    with pytest.raises(ValueError, match="without a reset mask"):
        step(batches[0], masks[0])
    step.graph = None
    red.close()
    assert _lib.device_status()[0] == 0
