"""The gated linear layer, its autograd node and LadderLM's level "gated_linear"; the Muon step; both together in a
captured training step and in generation."""
import pytest
import torch
import torch.nn.functional as F

from elman_b200 import _lib, fused_ops
from elman_b200 import hasty_pytorch_lib as H
from elman_b200.gated_linear import GatedLinearElman
from elman_b200.ladder_lm import LadderLM, zipf_tokens
from elman_b200.train_step import FlatGradients, FlatMuon, GraphedTrainStep, hidden_matrices, make_gradient_reducer

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-4, torch.bfloat16: 2e-2}     # the layers' tolerances elsewhere


def rel(a, b):
    return float((a.detach().double().cpu() - b.double().cpu()).norm() / b.double().norm())


def definition(fcz, h0, reset):
    """[T,B,3d] -> y, h_last in the dtype given."""
    f, c, z = fcz.chunk(3, dim=-1)
    h, hs = h0, []
    for t in range(fcz.shape[0]):
        p = h if reset is None else torch.where(reset[t].unsqueeze(-1), torch.zeros_like(h), h)
        h = p + torch.sigmoid(-f[t]) * (c[t] - p)
        hs.append(h)
    return torch.stack(hs) * F.silu(z), h


@pytest.mark.parametrize("T,B,d", [(1, 2, 24), (9, 3, 64), (130, 2, 33), (300, 1, 64)])
@pytest.mark.parametrize("with_reset", [False, True])
def test_gradients_are_those_of_differences(T, B, d, with_reset):
    """Directional derivatives of the definition by central differences in float64 (off by less than 1e-9) against the
    kernel's fp32 gradients."""
    g = torch.Generator().manual_seed(T)
    fcz, h0 = torch.randn(T, B, 3 * d, generator=g).cuda(), torch.randn(B, d, generator=g).cuda()
    reset = (torch.rand(T, B, generator=g) < 0.05).cuda() if with_reset else None
    wy, wh = torch.randn(T, B, d, generator=g), torch.randn(B, d, generator=g)
    x, s = fcz.clone().requires_grad_(True), h0.clone().requires_grad_(True)
    y, h = fused_ops.gated_linear(x, s, reset)
    ((y * wy.cuda()).sum() + (h * wh.cuda()).sum()).backward()
    cpu_reset = None if reset is None else reset.cpu()

    def loss(a, b):
        yy, hh = definition(a, b, cpu_reset)
        return (yy * wy.double()).sum() + (hh * wh.double()).sum()

    for k in range(3):
        vx, vs = torch.randn(T, B, 3 * d, generator=g).double(), torch.randn(B, d, generator=g).double()
        e = 1e-5
        a, b = fcz.double().cpu(), h0.double().cpu()
        want = (loss(a + e * vx, b + e * vs) - loss(a - e * vx, b - e * vs)) / (2 * e)
        gx, gs = x.grad.double().cpu(), s.grad.double().cpu()
        got = (gx * vx).sum() + (gs * vs).sum()
        # the gradients are 4e-6 off norm-wise, in no direction in particular
        assert abs(float(got - want)) < 2e-5 * float((gx.norm() ** 2 + gs.norm() ** 2).sqrt()), k


def test_node_accepts_what_autograd_hands_it():
    """Broadcast gradients, a missing gradient of either output, no gradient for h0, batch-major input."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 40, 3 * 16, generator=g).cuda().requires_grad_(True)        # batch-major
    y, h = fused_ops.gated_linear(x.transpose(0, 1))
    (grad,) = torch.autograd.grad(y.sum(), x, retain_graph=True)
    (grad_h,) = torch.autograd.grad(h.sum(), x)
    ref = x.detach().cpu().double().requires_grad_(True)
    yy, hh = definition(ref.transpose(0, 1), torch.zeros(2, 16, dtype=torch.float64), None)
    assert rel(grad, torch.autograd.grad(yy.sum(), ref, retain_graph=True)[0]) < 2e-5
    assert rel(grad_h, torch.autograd.grad(hh.sum(), ref)[0]) < 2e-5
    assert grad.is_contiguous()
    with pytest.raises(RuntimeError, match="3 \\* dim"):
        fused_ops.gated_linear(torch.zeros(3, 2, 10, device="cuda"))
    with pytest.raises(RuntimeError, match="float32"):
        fused_ops.gated_linear(torch.zeros(3, 2, 9, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="bool"):
        fused_ops.gated_linear(torch.zeros(3, 2, 9, device="cuda"), None, torch.zeros(3, 2, device="cuda"))
    with pytest.raises(RuntimeError, match="shape"):
        fused_ops.gated_linear(torch.zeros(3, 2, 9, device="cuda"), None, torch.zeros(2, 3, device="cuda", dtype=torch.bool))
    with pytest.raises(RuntimeError, match="not supported"):
        fused_ops.gated_linear(torch.zeros(3, 2, 9, device="cuda", dtype=torch.float16))


def test_second_derivatives_are_refused():
    x = torch.randn(20, 2, 3 * 16, device="cuda", requires_grad=True)
    y, _ = fused_ops.gated_linear(x)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_gradient_slices_that_overlap_are_refused():
    x = torch.zeros(70, 2, 8, device="cuda")
    saved = H.gated_linear_forward(True, x, x, x)[2]
    one = torch.empty_like(x)
    with pytest.raises(_lib.ElmanB200Error, match="overlap"):
        H.gated_linear_backward(x, x, x, saved, x, out=(one, one, torch.empty_like(x)))
    rows = torch.empty(70, 2, 20, device="cuda")
    with pytest.raises(_lib.ElmanB200Error, match="overlap"):
        H.gated_linear_backward(x, x, x, saved, x, out=(rows[..., :8], rows[..., 6:14], torch.empty_like(x)))


def test_flat_muon_with_a_parameter_of_no_elements():
    """The empty parameter lies between others; the step is that of the same model without it."""
    def run(empty):
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((5,), (8, 12), (7,))]
        if empty:
            ps.insert(1, torch.nn.Parameter(torch.empty(0, device="cuda")))
        grads = FlatGradients([ps])
        opt = FlatMuon(grads, [p for p in ps if p.dim() == 2])
        for p in ps:
            p.grad.fill_(0.5)
        opt.step()
        return [p.detach() for p in ps if p.numel() > 0]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


def test_python_entry_refuses_on_the_device():
    x = torch.zeros(70, 2, 8, device="cuda")
    y, h, saved = H.gated_linear_forward(True, x, x, x)
    with pytest.raises(RuntimeError, match="dense channels"):
        H.gated_linear_forward(False, x.transpose(0, 2).contiguous().transpose(0, 2), x, x)
    with pytest.raises(RuntimeError, match="shape"):
        H.gated_linear_forward(False, x, x[:3], x)
    with pytest.raises(RuntimeError, match="training=True"):
        H.gated_linear_backward(x, x, x, x.new_empty(0), x)
    with pytest.raises(RuntimeError, match="saved has shape"):
        H.gated_linear_backward(x, x, x, saved[:1], x)
    with pytest.raises(RuntimeError, match="share storage"):
        H.gated_linear_backward(x, x, x, saved, x, out=(x, torch.empty_like(x), torch.empty_like(x)))
    big = torch.zeros(70, 2, 8, device="cuda")
    with pytest.raises(_lib.ElmanB200Error, match="overlap"):
        H.gated_linear_backward(x, x, x, saved, x, out=(big[:1].expand(70, 2, 8), torch.empty_like(x), torch.empty_like(x)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,expansion", [(64, 1.0), (48, 1.5)])
def test_layer_against_its_definition(dim, expansion, dtype):
    torch.manual_seed(5)
    layer = GatedLinearElman(dim, expansion=expansion).cuda().to(dtype)
    x = torch.randn(3, 90, dim, device="cuda").to(dtype).requires_grad_(True)
    h0 = torch.randn(3, layer.d_inner, device="cuda")
    reset = torch.rand(3, 90, device="cuda") < 0.03
    out, h = layer(x, h0, reset)
    w = torch.randn_like(out)
    (out * w).sum().backward()
    ref = {k: v.detach().double().cpu().requires_grad_(True) for k, v in layer.named_parameters()}
    xr = x.detach().double().cpu().requires_grad_(True)
    fcz = xr @ ref["in_proj.weight"].T + ref["in_proj.bias"]
    yy, hh = definition(fcz.transpose(0, 1), h0.double().cpu(), reset.t().cpu())
    want = yy.transpose(0, 1) @ ref["out_proj.weight"].T
    (want * w.double().cpu()).sum().backward()
    assert out.dtype == dtype and h.dtype == torch.float32
    assert rel(out, want.detach()) < TOL[dtype] and rel(h, hh.detach()) < TOL[dtype]
    assert rel(x.grad, xr.grad) < TOL[dtype]
    for k, v in layer.named_parameters():
        assert rel(v.grad, ref[k].grad) < TOL[dtype], k


def test_generation_token_by_token_is_the_whole_sequence():
    torch.manual_seed(6)
    model = LadderLM(vocab_size=256, dim=64, depth=3, level="gated_linear").cuda().bfloat16().eval()
    tok = zipf_tokens(2, 50, seed=1).cuda()
    with torch.no_grad():
        whole = model(tok)
        states, steps = None, []
        for t in range(50):
            logits, (states, _) = model(tok[:, t:t + 1], return_prev_hiddens=True, prev_hiddens=states)
            steps.append(logits)
    assert all(s.dtype == torch.float32 for s in states)
    assert rel(torch.cat(steps, 1), whole) < TOL[torch.bfloat16]


def test_reset_separates_packed_documents():
    torch.manual_seed(7)
    model = LadderLM(vocab_size=256, dim=64, depth=2, level="gated_linear").cuda()
    tok = zipf_tokens(1, 60, seed=2).cuda()
    reset = torch.zeros(1, 60, dtype=torch.bool, device="cuda")
    reset[0, 25] = True
    with torch.no_grad():
        both, second = model(tok, reset=reset), model(tok[:, 25:])
    assert rel(both[:, 25:], second) < TOL[torch.float32]
    assert float(model(tok, return_loss=True, reset=reset)) > 0
    with pytest.raises(ValueError, match="gated_linear"):
        LadderLM(vocab_size=256, dim=64, depth=1, level=1).cuda()(tok, reset=reset)


# ------------------------------------------------------------------ Muon

def muon_reference(p, g, mom, lr, mu, nesterov, wd, steps=5):
    a, b, c = H.NEWTON_SCHULZ_COEFFICIENTS
    mom += (1 - mu) * (g - mom)
    u = g + mu * (mom - g) if nesterov else mom
    X = u / (u.norm() + 1e-7)
    for _ in range(steps):
        A = X @ X.T
        X = a * X + (b * A + c * A @ A) @ X
    p *= 1 - lr * wd
    p -= lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * X


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.a = torch.nn.Linear(40, 72)
        self.b = torch.nn.Linear(72, 72)
        self.c = torch.nn.Linear(72, 40)
        self.d = torch.nn.Linear(40, 72)
        self.e = torch.nn.Linear(72, 9)


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_flat_muon_follows_its_definition(dtype, nesterov):
    torch.manual_seed(3)
    net = Net().cuda().to(dtype)
    grads = FlatGradients([list(net.e.parameters()) + list(net.d.parameters()),
                           [p for m in (net.a, net.b, net.c) for p in m.parameters()]])
    mats = [net.a.weight, net.b.weight, net.c.weight, net.d.weight]
    lr, mu, wd = 0.03, 0.9, 0.1
    opt = FlatMuon(grads, mats, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, adamw_lr=3e-3, betas=(0.9, 0.95))
    rest = [p for p in net.parameters() if all(p is not m for m in mats)]
    twin = [p.detach().clone().requires_grad_(True) for p in rest]
    adam = torch.optim.AdamW(twin, lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0)
    ref = [p.detach().double().clone() for p in mats]
    start = [p.clone() for p in ref]
    moms = [torch.zeros_like(p) for p in ref]
    scale = torch.tensor(0.5, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    for it in range(4):
        for p in grads.params:
            p.grad.copy_(torch.randn(p.shape, generator=gen, device="cuda"))
        for p, r, m in zip(mats, ref, moms):
            muon_reference(r, 0.5 * p.grad.double(), m, lr, mu, nesterov, wd)
        for p, t in zip(rest, twin):
            t.grad = (0.5 * p.grad).to(t.dtype)
        opt.step(grad_scale=scale)
        adam.step()
        if dtype == torch.bfloat16:        # the parameters' own rounding is not what is compared
            for p, r in zip(mats, ref):
                assert rel(p, r) < 2 ** -7
                r.copy_(p.double())
    for p, r, s in zip(mats, ref, start):
        # fp32: the moves, four of them, each 2e-5 off at most, and the rounding of p (2^-24 of it, p about four moves)
        assert rel(p, r) < (2 ** -7 if dtype == torch.bfloat16 else 1e-5)
        if dtype == torch.float32:
            assert rel(p.double() - s, r - s) < 5e-5
    for (m, n, offsets, momentum) in opt.groups:
        assert momentum.dtype == torch.float32 and momentum.shape == (offsets.numel(), m, n)
    assert sorted((m, n, o.numel()) for m, n, o, _ in opt.groups) == [(40, 72, 1), (72, 40, 2), (72, 72, 1)]
    for p, t in zip(rest, twin):
        assert rel(p, t.detach()) < (2e-5 if dtype == torch.float32 else 2e-2)
    assert grads.check_views() and _lib.device_status()[0] == 0


def test_flat_muon_state_round_trip_and_refusals():
    torch.manual_seed(4)

    def make():
        net = Net().cuda()
        grads = FlatGradients([list(net.parameters())])
        return net, grads, FlatMuon(grads, [net.a.weight, net.b.weight])

    net, grads, opt = make()
    for p in grads.params:
        p.grad.normal_()
    opt.step()
    other, grads2, opt2 = make()
    with torch.no_grad():
        grads2.flat_params.copy_(grads.flat_params)
    grads2.flat.copy_(grads.flat)
    opt2.load_state_dict(opt.state_dict())
    opt.step()
    opt2.step()
    assert torch.equal(grads.flat_params, grads2.flat_params)
    with pytest.raises(ValueError, match="2-D"):
        FlatMuon(grads, [net.a.bias])
    with pytest.raises(ValueError, match="2-D"):
        FlatMuon(grads, [other.a.weight])
    with pytest.raises(ValueError, match="more than once"):
        FlatMuon(grads, [net.a.weight, net.a.weight])
    with pytest.raises(RuntimeError, match="grad_scale"):
        opt.step(grad_scale=torch.ones((), device="cuda", dtype=torch.float64))


@pytest.mark.parametrize("level", ["gated_linear", 1])
def test_captured_training_with_muon_follows_the_eager_one(level):
    """The whole of it: layers, loss, gradients in flat buffers, clipping, Muon and AdamW, captured and replayed."""
    batches = [zipf_tokens(4, 129, seed=300 + k).cuda() for k in range(4)]

    def make():
        torch.manual_seed(29)
        model = LadderLM(vocab_size=256, dim=128, depth=2, level=level, r_h_mode="none").cuda().bfloat16()
        red = make_gradient_reducer(model)
        return model, red, FlatMuon(red, hidden_matrices(model), lr=0.01, adamw_lr=1e-3)

    model, red, opt = make()
    eager = []
    for tok in [batches[0]] * 3 + batches:
        red.zero()
        loss = model(tok, return_loss=True)
        loss.backward()
        red.finish()
        opt.step(grad_scale=red.clip_coef(1.0)[0])
        eager.append(float(loss.detach()))
    red.close()
    model, red, opt = make()
    step = GraphedTrainStep(model, opt, batches[0], max_grad_norm=1.0, warmup_steps=3, reducer=red)
    graphed = [float(step(tok)) for tok in batches]
    assert _lib.device_status()[0] == 0 and red.check_views()
    assert float(opt.step_count[0]) == 3 + len(batches)
    assert all(abs(a - b) < 2e-2 * abs(a) for a, b in zip(eager[3:], graphed)), (eager, graphed)
    step.graph = None
    red.close()
