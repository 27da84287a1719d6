"""The gated linear recurrence (elman_gated_linear_*) against its definition in 64 bits: forward, gradients,
document resets, strided inputs, chained calls, generation."""
import pytest
import torch

from elman_b200 import _lib
from elman_b200 import hasty_pytorch_lib as H

pytestmark = pytest.mark.gpu

# Outputs are rounded once from fp32: half a step of the type, eps / 2 relative.  The fp32 arithmetic before it
# adds its own part: the gates come from __expf, whose argument scaling leaves |f| 2^-24 relative (|f| < 12 in the
# inputs below: 7e-7), and the state is a convex combination of values with such weights, so 4e-6 covers states
# and gradients norm-wise (about six such factors); with bf16 outputs that is below half a step, which the
# norm-wise error cannot exceed.
TOL = {torch.float32: 4e-6, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2 + 4e-6}
STATE_TOL = 4e-6


def reference(f, c, z, h0, reset, dy=None, dh=None):
    """The definition, step by step in float64, and its gradients by autograd."""
    T, B, d = f.shape
    leaves = [t.detach().double().cpu().requires_grad_(True) for t in (f, c, z)]
    h0 = (torch.zeros(B, d, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()).requires_grad_(True)
    fd, cd, zd = leaves
    h, hs = h0, []
    for t in range(T):
        u = torch.sigmoid(-fd[t])
        p = h if reset is None else torch.where(reset[t].cpu().unsqueeze(-1), torch.zeros_like(h), h)
        h = p + u * (cd[t] - p)
        hs.append(h)
    y = torch.stack(hs) * torch.nn.functional.silu(zd) if T else fd
    if dy is None:
        return y.detach(), h.detach()
    loss = (y * dy.double().cpu()).sum() + (0 if dh is None else (h * dh.double().cpu()).sum())
    return [y.detach(), h.detach()] + [g for g in torch.autograd.grad(loss, leaves + [h0])]


def rel(a, b):
    a, b = a.detach().double().cpu(), b.double()
    assert a.shape == b.shape and torch.isfinite(a).all()
    norm = b.norm()
    return float((a - b).norm() / norm) if norm > 0 else float(a.norm())


def make(T, B, d, dtype, seed=0, packed=False, batch_major=False, reset=None, h0=True):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = rnd(T, B, 3 * d)
    x[..., :d] += 4 * torch.rand(d, generator=g)
    x = x.to(dtype).cuda()
    if batch_major:
        x = x.transpose(0, 1).contiguous().transpose(0, 1)
    parts = list(x.chunk(3, dim=-1))
    if not packed:
        parts = [p.transpose(0, 1).contiguous().transpose(0, 1) if batch_major else p.contiguous() for p in parts]
    marks = None if reset is None else (torch.rand(T, B, generator=g) < reset).cuda()
    return dict(f=parts[0], c=parts[1], z=parts[2], h0=rnd(B, d).cuda() if h0 else None, reset=marks,
                dy=rnd(T, B, d).to(dtype).cuda(), dh=rnd(B, d).cuda())


def check(s, dtype, use_dh=True):
    f, c, z, h0, reset, dy = (s[k] for k in ("f", "c", "z", "h0", "reset", "dy"))
    dh = s["dh"] if use_dh else None
    want = reference(f, c, z, h0, reset, dy, dh)
    y, h, saved = H.gated_linear_forward(True, f, c, z, h0, reset)
    grads = H.gated_linear_backward(f, c, z, saved, dy, dh, reset)
    y2, h2, none = H.gated_linear_forward(False, f, c, z, h0, reset)
    assert torch.equal(y, y2) and torch.equal(h, h2) and none.numel() == 0
    got = [y, h] + grads
    names = ["y", "h_last", "df", "dc", "dz", "dh0"]
    for name, g, w in zip(names, got, want):
        tol = STATE_TOL if name in ("h_last", "dh0") else TOL[dtype]
        assert rel(g, w) < tol, (name, rel(g, w), tol)
    assert _lib.device_status()[0] == 0


SHAPES = [(1, 1, 1), (1, 3, 40), (2, 1, 257), (7, 2, 64), (8, 2, 64), (9, 1, 66), (63, 2, 96), (64, 1, 33), (65, 3, 130), (127, 1, 64),
          (128, 2, 62), (129, 1, 1), (200, 5, 101), (1000, 2, 48), (2100, 1, 70), (300, 40, 256)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,B,d", SHAPES)
def test_against_definition(T, B, d, dtype):
    check(make(T, B, d, dtype, seed=T + d), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed,batch_major", [(True, False), (True, True), (False, True)])
@pytest.mark.parametrize("T,B,d", [(70, 3, 40), (150, 4, 37), (5, 2, 64), (260, 1, 128)])
def test_strided_inputs(T, B, d, packed, batch_major, dtype):
    s = make(T, B, d, dtype, seed=5, packed=packed, batch_major=batch_major, reset=0.02)
    check(s, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed,batch_major", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("T,B,d,reset", [(9, 2, 64, None), (64, 1, 120, 0.05), (129, 3, 128, None), (200, 2, 1000, 0.01), (2100, 2, 120, None),
                                         (5000, 1, 64, 0.002), (4097, 1, 60, None), (300, 9, 1280, None)])
def test_rows_on_16_bytes(T, B, d, reset, packed, batch_major, dtype):
    """The shapes whose rows TMA copies: whole and ragged channel groups, one tile and several groups of them."""
    check(make(T, B, d, dtype, seed=T, packed=packed, batch_major=batch_major, reset=reset), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed,batch_major", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("T,B,d,reset", [(9, 2, 63, None), (112, 1, 62, 0.05), (113, 3, 61, None), (200, 2, 1001, 0.01), (2100, 2, 126, None),
                                         (5000, 1, 55, 0.002), (300, 9, 1279, None), (130, 2, 118, 0.02)])
def test_rows_of_any_alignment(T, B, d, reset, packed, batch_major, dtype):
    """The shapes whose rows are copied one by one: starts on 4 and on 2 bytes, changing from row to row."""
    check(make(T, B, d, dtype, seed=T, packed=packed, batch_major=batch_major, reset=reset), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_tensors_off_their_16_byte_boundary(shift, dtype):
    """The same values from storages that start elsewhere, and outputs that leave their neighbours alone."""
    T, B, d = 150, 2, 128
    s = make(T, B, d, dtype, seed=12)
    def moved(t):
        room = torch.full((t.numel() + 64,), float("nan"), device="cuda", dtype=dtype)
        room[16 + shift:16 + shift + t.numel()] = t.reshape(-1)
        return room[16 + shift:16 + shift + t.numel()].view(t.shape)
    f, c, z, dy = (moved(s[k]) for k in ("f", "c", "z", "dy"))
    y, h, saved = H.gated_linear_forward(True, f, c, z, s["h0"])
    want = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])
    tol = TOL[dtype]
    assert rel(y, want[0].cpu()) < 2 * tol and rel(h, want[1].cpu()) < 2 * STATE_TOL
    outs = [torch.full((T * B * d + 64,), 7.0, device="cuda", dtype=dtype) for _ in range(3)]
    views = tuple(o[16 + shift:16 + shift + T * B * d].view(T, B, d) for o in outs)
    H.gated_linear_backward(f, c, z, saved, dy, out=views)
    ref = H.gated_linear_backward(s["f"], s["c"], s["z"], want[2], s["dy"])
    for o, v, r in zip(outs, views, ref):
        assert rel(v, r.cpu()) < 2 * tol
        assert (o[:16 + shift] == 7).all() and (o[16 + shift + T * B * d:] == 7).all()


@pytest.mark.parametrize("T,d", [(200, 128), (200, 62), (200, 24)])
def test_expanded_inputs(T, d):
    """Inputs broadcast over time or batch (stride 0): full gradients come back."""
    s = make(T, 3, d, torch.float32, seed=13)
    f, c, z = s["f"][:1].expand(T, 3, d), s["c"][:, :1].expand(T, 3, d), s["z"]
    y, h, saved = H.gated_linear_forward(True, f, c, z, s["h0"])
    g = H.gated_linear_backward(f, c, z, saved, s["dy"], s["dh"])
    y2, h2, saved2 = H.gated_linear_forward(True, f.contiguous(), c.contiguous(), z, s["h0"])
    g2 = H.gated_linear_backward(f.contiguous(), c.contiguous(), z, saved2, s["dy"], s["dh"])
    for a, b in zip([y, h] + g, [y2, h2] + g2):
        assert rel(a, b.cpu()) < 2 * TOL[torch.float32]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 62, 61, 20])
def test_calls_on_two_streams_at_once(d, dtype):
    """Long chains in several launches that share the device: none waits for another's blocks."""
    sets = [make(3000, 4, d, dtype, seed=40 + k, reset=0.001) for k in range(3)]
    want = [[t.clone() for t in H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                out = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])
                got.append(out + H.gated_linear_backward(s["f"], s["c"], s["z"], out[2], s["dy"], s["dh"], s["reset"]))
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out[:3], want[k % 3]))
        assert all(torch.equal(a, b) for a, b in zip(out[3:], got[k % 3][3:]))
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("share", [0.01, 0.3, 1.0])
@pytest.mark.parametrize("T,B,d", [(3, 2, 16), (200, 3, 65), (1500, 1, 64)])
def test_resets(T, B, d, share, dtype):
    check(make(T, B, d, dtype, seed=9, reset=share), dtype, use_dh=share != 0.3)


@pytest.mark.parametrize("T", [1, 30, 700])
def test_reset_drops_a_state_that_is_not_finite(T):
    """Nothing of the state before a reset is read: not inf, not NaN; what precedes the reset keeps it."""
    s = make(T, 2, 64, torch.float32, seed=3)
    s["reset"] = torch.zeros(T, 2, dtype=torch.bool, device="cuda")
    cut = T // 2
    s["reset"][cut, 0] = True
    s["h0"][0] = float("inf")
    s["h0"][0, ::2] = float("nan")
    y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])
    want_y, want_h = reference(s["f"], s["c"], s["z"], s["h0"], s["reset"])
    assert torch.isfinite(h).all() and torch.isfinite(y[cut:]).all() and torch.isfinite(y[:, 1]).all()
    assert rel(h, want_h) < STATE_TOL and rel(y[cut:], want_y[cut:]) < TOL[torch.float32]
    assert not torch.isfinite(y[:cut, 0]).any()
    # and no gradient crosses it backwards, not even one that is not finite
    s["dy"][cut:, 0] = float("nan")
    s["dh"][0] = float("inf")
    s["h0"].zero_()
    y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])
    df, dc, dz, dh0 = H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"], s["dh"], s["reset"])
    assert torch.isfinite(dh0).all() and torch.isfinite(df[:cut]).all() and torch.isfinite(dc[:cut]).all()


def test_nan_gate_reaches_everything_after_it_and_nothing_before():
    s = make(400, 1, 64, torch.bfloat16, seed=4)
    s["f"][150, 0, 7] = float("nan")
    y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])
    bad = torch.isnan(y[:, 0])
    assert bad[150:, 7].all() and not bad[:150].any() and bad.sum() == 250 and torch.isnan(h[0, 7])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_extreme_gates(dtype):
    """Gates that are open, shut, or beyond exp's range; silu far out on both sides."""
    T, d = 300, 64
    f = torch.tensor([-1e4, -90.0, -20.0, 0.0, 15.0, 60.0, 100.0, 1e4]).repeat(8).expand(T, 1, d).to(dtype).cuda().contiguous()
    c = torch.randn(T, 1, d, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    z = torch.linspace(-120, 120, T).view(T, 1, 1).expand(T, 1, d).to(dtype).cuda().contiguous()
    h0 = torch.randn(1, d, generator=torch.Generator().manual_seed(2)).cuda()
    dy = torch.randn(T, 1, d, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    s = dict(f=f, c=c, z=z, h0=h0, reset=None, dy=dy, dh=torch.randn(1, d, generator=torch.Generator().manual_seed(6)).cuda())
    check(s, dtype)


def test_memory_of_many_steps_is_kept_in_fp32():
    """Gates of 1e-6: the state must move by u (c - p), which 1 - u in fp32 would lose."""
    T, d = 5000, 64
    f = torch.full((T, 1, d), 13.8, device="cuda", dtype=torch.float32)
    c, z = torch.ones_like(f), torch.ones_like(f)
    y, h, _ = H.gated_linear_forward(False, f, c, z, None)
    _, want = reference(f, c, z, None, None)
    # every step adds about 1e-6 to a state below 5e-3, rounded to 2^-24 of it: 5000 roundings of 3e-10, at worst
    # all one way, 1.5e-6 absolute = 3e-4; at random 4e-6; the gate itself is off by 13.8 * 2^-24 < 1e-6
    assert rel(h, want) < 1e-4


@pytest.mark.parametrize("cuts", [[1] * 10, [64, 64, 72], [3, 130, 67]])
def test_chained_calls_are_the_whole_sequence(cuts):
    T = sum(cuts)
    s = make(T, 3, 80, torch.float32, seed=8, reset=0.02)
    y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])
    whole = H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"], s["dh"], s["reset"])
    state, parts, t0 = s["h0"], [], 0
    for n in cuts:
        at = slice(t0, t0 + n)
        out = H.gated_linear_forward(True, s["f"][at], s["c"][at], s["z"][at], state, s["reset"][at])
        parts.append((at, out))
        state, t0 = out[1], t0 + n
    assert rel(torch.cat([o[0] for _, o in parts]), y.cpu()) < 2 * TOL[torch.float32]
    assert rel(state, h.cpu()) < 2 * STATE_TOL
    dh, pieces = s["dh"], []
    for at, out in reversed(parts):
        *g, dh = H.gated_linear_backward(s["f"][at], s["c"][at], s["z"][at], out[2], s["dy"][at], dh, s["reset"][at])
        pieces.insert(0, g)
    for k in range(3):
        assert rel(torch.cat([p[k] for p in pieces]), whole[k].cpu()) < 2 * TOL[torch.float32]
    assert rel(dh, whole[3].cpu()) < 2 * STATE_TOL


def test_two_runs_give_the_same_bits():
    s = make(3000, 2, 200, torch.bfloat16, seed=11, reset=0.001)
    runs = []
    for _ in range(3):
        y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"], s["reset"])
        runs.append([y, h] + H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"], s["dh"], s["reset"]))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_empty_sequence_and_empty_batch():
    f = torch.empty(0, 2, 8, device="cuda")
    h0 = torch.randn(2, 8, device="cuda")
    y, h, saved = H.gated_linear_forward(True, f, f, f, h0)
    assert y.shape == (0, 2, 8) and torch.equal(h, h0)
    *g, dh0 = H.gated_linear_backward(f, f, f, saved, f, h0)
    assert torch.equal(dh0, h0) and all(t.shape == (0, 2, 8) for t in g)
    y, h, saved = H.gated_linear_forward(True, *[torch.empty(4, 0, 8, device="cuda")] * 3)
    assert y.shape == (4, 0, 8) and h.shape == (0, 8)


def test_gradients_go_into_the_slices_of_one_buffer_and_nowhere_else():
    s = make(90, 2, 48, torch.bfloat16, seed=2, packed=True)
    y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])
    want = H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"])
    buf = torch.full((90, 3, 5 * 48), 7.0, device="cuda", dtype=torch.bfloat16)
    got = H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"],
                                  out=tuple(buf[:, :2, k * 48:(k + 1) * 48] for k in (1, 2, 3)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert (buf[:, 2] == 7).all() and (buf[..., :48] == 7).all() and (buf[..., 4 * 48:] == 7).all()


def test_offsets_beyond_32_bits():
    """A batch-major slice of a buffer of more than 2^31 elements: the last rows lie past 32-bit offsets."""
    T, B, d = 20, 3, 64
    room = torch.empty(3, 1_200_000_000, device="cuda", dtype=torch.bfloat16)      # 7.2 GB
    s = make(T, B, d, torch.bfloat16, seed=6)
    view = lambda k: room.as_strided((T, B, d), (3 * d, room.stride(0), 1), k * d)  # noqa: E731
    for k, name in enumerate(("f", "c", "z")):
        view(k).copy_(s[name])
    y, h, saved = H.gated_linear_forward(True, view(0), view(1), view(2), s["h0"])
    want = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])
    assert all(torch.equal(a, b) for a, b in zip((y, h, saved), want))
    far = room.as_strided((T, B, d), (150_000_000, d, 1), 0)
    far.copy_(s["f"])
    assert torch.equal(H.gated_linear_forward(False, far, s["c"], s["z"], s["h0"])[1], h)


def test_captured_calls_on_another_stream_share_a_pool():
    """Two graphs captured into one memory pool, replayed in turn with new inputs."""
    a, b = make(700, 2, 64, torch.bfloat16, seed=20), make(900, 1, 96, torch.bfloat16, seed=21)
    pool, graphs, outs = None, [], []
    side = torch.cuda.Stream()

    def call(s):
        y, h, saved = H.gated_linear_forward(True, s["f"], s["c"], s["z"], s["h0"])
        return [y, h] + H.gated_linear_backward(s["f"], s["c"], s["z"], saved, s["dy"], s["dh"])

    with torch.cuda.stream(side):
        call(a), call(b)
    torch.cuda.synchronize()
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool, stream=side):
            outs.append(call(s))
        pool = g.pool()
        graphs.append(g)
    for seed in (30, 31):
        for s, g, out in zip((a, b), graphs, outs):
            T, B, d = s["f"].shape
            fresh = make(T, B, d, torch.bfloat16, seed=seed)
            for k in ("f", "c", "z", "h0", "dy", "dh"):
                s[k].copy_(fresh[k])
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(x, y) for x, y in zip(got, call(s)))
    del graphs
