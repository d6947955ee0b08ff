"""residual_norm, causal_conv and selective_scan as a block uses them together: forward, gradients, decoding from the
prompt's states, captured into graphs, on other streams and from two threads."""

import threading

import pytest
import torch

from boltz_lumi_amd import ops

pytestmark = pytest.mark.gpu

D, C, N, W, RANK = 64, 128, 16, 4, 8


def parameters(seed, device, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)

    def randn(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale + shift).to(device, dtype)

    return {"in": randn(D, 2 * C, scale=D ** -0.5), "conv": randn(C, W, scale=0.5), "conv_bias": randn(C, scale=0.1),
            "maps": randn(C, RANK + 2 * N, scale=C ** -0.5), "dt": randn(RANK, C, scale=RANK ** -0.5),
            "dt_bias": randn(C, scale=0.5, shift=-2.0), "A": -torch.rand(C, N, generator=g, dtype=torch.float64).add(0.1).to(
                device, dtype), "D": randn(C), "out": randn(C, D, scale=C ** -0.5), "y_weight": randn(D, scale=0.2, shift=1.0),
            "scale": randn(D, scale=0.1, shift=0.5), "weight": randn(D, scale=0.2, shift=1.0)}


def block(x, h, p, lengths=None, states=(None, None), keep=False, out_states=(None, None)):
    """One block on the stream x and its normalised rows h: (new stream, its normalised rows, last states)."""
    u, z = (h @ p["in"]).split([C, C], -1)
    carry = keep or out_states[0] is not None
    u = ops.causal_conv(u, p["conv"], p["conv_bias"], state=states[0], lengths=lengths, return_state=carry,
                        state_out=out_states[0])
    u, last_conv = u if carry else (u, None)
    dt, B, Cm = (u @ p["maps"]).split([RANK, N, N], -1)
    y = ops.selective_scan(u, dt @ p["dt"], p["A"], B.unsqueeze(2), Cm.unsqueeze(2), p["D"], z, p["dt_bias"],
                           state=states[1], lengths=lengths, return_state=carry, state_out=out_states[1])
    y, last_scan = y if carry else (y, None)
    r, h = ops.residual_norm(x, y @ p["out"], None, p["y_weight"], p["scale"], p["weight"])
    return r, h, (last_conv, last_scan)


def plain_block(x, h, p, lengths):
    """The same in elementary operations, for autograd in fp64."""
    b, t, _ = x.shape
    keep = (torch.arange(t, device=x.device) < lengths[:, None])[..., None]
    u, z = (h @ p["in"]).split([C, C], -1)
    rows = torch.cat([u.new_zeros(b, W - 1, C), u], 1)
    conv = p["conv_bias"] + sum(p["conv"][:, j] * rows[:, j:j + t] for j in range(W))
    u = conv * torch.sigmoid(conv) * keep
    dt, B, Cm = (u @ p["maps"]).split([RANK, N, N], -1)
    d = torch.log1p(torch.exp(dt @ p["dt"] + p["dt_bias"]))
    state, ys = u.new_zeros(b, C, N), []
    for i in range(t):
        state = torch.exp(d[:, i, :, None] * p["A"]) * state + (d[:, i] * u[:, i])[..., None] * B[:, i, None]
        ys.append((state * Cm[:, i, None]).sum(-1))
    y = (torch.stack(ys, 1) + p["D"] * u) * z * torch.sigmoid(z) * keep
    m = y @ p["out"]
    r = x + p["scale"] * m / (m.square().mean(-1, keepdim=True) + 1e-6).sqrt() * p["y_weight"]
    return r, r / (r.square().mean(-1, keepdim=True) + 1e-6).sqrt() * p["weight"]


def inputs(seed, b, t, device, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(b, t, D, generator=g, dtype=torch.float64).to(device, dtype) for _ in range(4)]


def test_two_blocks_and_their_gradients(gpu):
    """fp32, two blocks deep, ragged: results and gradients of every parameter within 1e-4 of the largest (each product
    and norm is within about 1e-6 of its terms, some twenty of them follow each other, over 45 tokens)."""
    lengths = torch.tensor([45, 20, 1], device=gpu)
    x, h, dr, dh = inputs(0, 3, 45, gpu)
    keep = (torch.arange(45, device=gpu) < lengths[:, None])[..., None]
    dr, dh = dr * keep, dh * keep
    layers = [{k: v.requires_grad_() for k, v in parameters(i, gpu).items()} for i in (1, 2)]

    def run(form, x, h, layers):
        for p in layers:
            x, h = form(x, h, p, lengths)[:2]
        return x, h

    leaves = [x.requires_grad_(), h.requires_grad_(), *(v for p in layers for v in p.values())]
    made = run(block, x, h, layers)
    grads = torch.autograd.grad(made, leaves, (dr, dh))
    exact = [v.detach().double().requires_grad_() for v in leaves]
    keys = list(layers[0])
    deep = [dict(zip(keys, exact[2 + i * len(keys):2 + (i + 1) * len(keys)])) for i in (0, 1)]
    want = run(plain_block, exact[0], exact[1], deep)
    expected = torch.autograd.grad(want, exact, (dr.double(), dh.double()))
    for name, a, w in zip(["r", "h", "dx", "dh", *keys, *keys], [*made, *grads], [*want, *expected]):
        assert (a - w).abs().max() <= 1e-4 * w.abs().max(), name


def test_prompt_and_decoding(gpu):
    """A prompt of ragged lengths leaves states; tokens one by one in place are then the longer sequence."""
    p = parameters(3, gpu)
    x, h, _, _ = inputs(4, 3, 40, gpu)
    prompt = torch.tensor([30, 9, 0], device=gpu)
    with torch.no_grad():
        whole = block(x, h, p, prompt + 10)
        _, _, states = block(x[:, :30], h[:, :30], p, prompt, keep=True)
        for i in range(10):
            at = (prompt + i)[:, None, None].expand(-1, 1, D)
            r, g, _ = block(x.gather(1, at), h.gather(1, at), p, states=states, out_states=states)
            assert (r - whole[0].gather(1, at)).abs().max() <= 1e-4
            assert (g - whole[1].gather(1, at)).abs().max() <= 1e-4


def test_captured_steps(gpu):
    """A decoding step in place, captured: every replay moves the states on as an eager step does, other work between."""
    p = parameters(5, gpu)
    x, h, _, _ = inputs(6, 4, 8, gpu)
    with torch.no_grad():
        eager = [torch.randn(4, W - 1, C, device=gpu), torch.randn(4, C, N, device=gpu)]
        states = [s.clone() for s in eager]
        first = [s.clone() for s in eager]
        now = [x[:, :1].clone(), h[:, :1].clone()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(*now, p, states=states, out_states=states)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r, g, _ = block(*now, p, states=states, out_states=states)
        for s, f in zip(states, first):
            s.copy_(f)
        for i in range(8):
            now[0].copy_(x[:, i:i + 1])
            now[1].copy_(h[:, i:i + 1])
            graph.replay()
            want = block(x[:, i:i + 1].contiguous(), h[:, i:i + 1].contiguous(), p, states=eager, out_states=eager)
            torch.cuda.synchronize()
            assert torch.equal(r, want[0]) and torch.equal(g, want[1])
            assert all(torch.equal(a, b) for a, b in zip(states, eager))


@pytest.mark.parametrize("t", [5, 700])
def test_captured_training_step(gpu, t):
    """Forward and backward captured, its leaves made inside, replayed on new inputs between eager steps."""
    p = parameters(7, gpu)
    lengths = torch.tensor([t, t // 2], device=gpu)

    def step(x, h, dr, dh):
        leaves = [v.detach().requires_grad_() for v in (x, h, *p.values())]
        r, g, _ = block(leaves[0], leaves[1], dict(zip(p, leaves[2:])), lengths)
        return [r.detach(), g.detach(), *torch.autograd.grad((r, g), leaves, (dr, dh))]

    held = inputs(8, 2, t, gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step(*held)
    for seed in range(4):
        new = inputs(20 + seed, 2, t, gpu)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new)
        torch.cuda.synchronize()
        # the library's products may choose other kernels under capture: the operators' own bits are tested below
        for a, w in zip(made, want):
            assert (a - w).abs().max() <= 1e-4 * w.abs().max() + 1e-6


def one_of_each(seed, gpu):
    """The three operators on their own, forward and backward: results of fixed bits."""
    g = torch.Generator().manual_seed(seed)
    u, dt, z = (torch.randn(2, 300, 40, generator=g).to(gpu) for _ in range(3))
    B, Cm = (torch.randn(2, 300, 1, 16, generator=g).to(gpu) for _ in range(2))
    A, w = -torch.rand(40, 16, generator=g).to(gpu), torch.randn(40, 4, generator=g).to(gpu)
    gate = torch.randn(2, 1, 40, generator=g).to(gpu)
    leaves = [v.requires_grad_() for v in (u, dt, z, B, Cm, A, w, gate)]

    def run():
        c = ops.causal_conv(u, w)
        y, last = ops.selective_scan(c, dt, A, B, Cm, z=z, return_state=True)
        r, h = ops.residual_norm(u, y, gate)
        total = (r, h, last)
        back = [torch.ones_like(t) for t in total]
        return [*(t.detach() for t in total), *torch.autograd.grad(total, leaves, back)]

    return run


def test_same_bits_every_time(gpu):
    run = one_of_each(0, gpu)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_other_streams(gpu):
    runs = [one_of_each(s, gpu) for s in (1, 2)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in runs], [None, None]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            for _ in range(5):
                got[i] = runs[i]()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_two_threads(gpu):
    runs = [one_of_each(s, gpu) for s in (3, 4)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = runs[i]()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
