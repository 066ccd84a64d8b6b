"""The operators around a mixer as a model uses them: a whole block of the framework's own layers (norm, projections, short
convolution, gates, Gated DeltaNet, gated norm, output projection, norm, gated feed-forward block), in training, in decoding,
captured into graphs and on several streams at once, and sizes whose offsets pass 32 bits."""

import math

import pytest
import torch

from jax_linear_attention_b200 import layers, ops

pytestmark = pytest.mark.gpu

D, H, K, F = 256, 4, 64, 520  # model width, heads, head size, feed-forward width


def _weights(dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def mat(out, depth):
        return (torch.randn(out, depth, generator=gen, device="cuda") / math.sqrt(depth)).to(dtype)

    w = dict(qkv=mat(3 * H * K, D), z=mat(H * K, D), ab=mat(2 * H, D), out=mat(D, H * K), gate=mat(F, D), up=mat(F, D), down=mat(D, F))
    for n in ("n1", "n2"):
        w[n] = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
    w["n3"] = 1 + 0.1 * torch.randn(K, generator=gen, device="cuda")
    w["conv"] = 0.5 * torch.randn(3 * H * K, 4, generator=gen, device="cuda")
    w["a_log"], w["dt"] = torch.zeros(H, device="cuda"), torch.full((H,), -2.0, device="cuda")
    w["qkv_b"] = 0.1 * torch.randn(3 * H * K, generator=gen, device="cuda")
    return w


def block(x, stream, w, conv=None, state=None):
    """``(branch output, stream, conv state, state)``: the next block's norm adds the branch output to the stream."""
    B, T, _ = x.shape
    n, stream = layers.rms_norm(x, w["n1"], residual=stream)
    qkv, conv = layers.short_conv(layers.linear(n, w["qkv"], w["qkv_b"]), w["conv"], state=conv)
    q, k, v = (t.reshape(B, T, H, K) for t in qkv.split(H * K, -1))
    ab = layers.linear(n, w["ab"])
    g, beta = layers.gate_prologue(ab[..., :H].contiguous(), w["a_log"], w["dt"], ab[..., H:].contiguous())
    o, state = ops.linear_attention("gated_deltanet", q, k, v, g=g, beta=beta, use_qk_l2norm=True, initial_state=state,
                                    output_final_state=True)
    z = layers.linear(n, w["z"]).reshape(B, T, H, K)
    o = layers.gated_rms_norm(o, z, w["n3"])
    y = layers.linear(o.reshape(B, T, H * K), w["out"])
    n, stream = layers.rms_norm(y, w["n2"], residual=stream)
    return layers.linear(layers.gated_linear(n, w["gate"], w["up"]), w["down"]), stream, conv, state


def reference(x, stream, w):
    """The same in 64 bits."""
    B, T, _ = x.shape

    def norm(t, weight):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * weight

    stream = stream + x
    n = norm(stream, w["n1"])
    c = n @ w["qkv"].t() + w["qkv_b"]
    c = torch.nn.functional.pad(c, (0, 0, 3, 0))
    c = torch.nn.functional.silu(sum(c[:, i:i + T] * w["conv"][:, i] for i in range(4)))
    q, k, v = (t.reshape(B, T, H, K) for t in c.split(H * K, -1))
    q, k = (t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    ab = n @ w["ab"].t()
    g = -torch.exp(w["a_log"]) * torch.nn.functional.softplus(ab[..., :H] + w["dt"])
    beta = torch.sigmoid(ab[..., H:])
    state, o = torch.zeros(B, H, K, K, dtype=x.dtype, device=x.device), []
    for t in range(T):
        state = state * torch.exp(g[:, t])[..., None, None]
        delta = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhk,bhkv->bhv", k[:, t], state))
        state = state + torch.einsum("bhk,bhv->bhkv", k[:, t], delta)
        o.append(torch.einsum("bhk,bhkv->bhv", q[:, t] * K ** -0.5, state))
    o = norm(torch.stack(o, 1), w["n3"]) * torch.nn.functional.silu((n @ w["z"].t()).reshape(B, T, H, K))
    stream = stream + o.reshape(B, T, H * K) @ w["out"].t()
    n = norm(stream, w["n2"])
    return (torch.nn.functional.silu(n @ w["gate"].t()) * (n @ w["up"].t())) @ w["down"].t(), stream


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return float((a - b).norm() / b.norm())


# Sixteen roundings to 16 bits lie between a block's input and its output (and as many again on a gradient's way back), each at
# most half a step, on values that add up to no more than what they are relative to: 16 half steps, and 32 for gradients. The
# mixer's own kernels are held to 1e-2 in bf16 by their tests, about three half steps: counted among them.
@pytest.mark.parametrize("dtype, T", [(torch.bfloat16, 100), (torch.float16, 100), (torch.bfloat16, 1100)])
def test_block_training(dtype, T):
    w = _weights(dtype)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, s, dy, ds = (torch.randn(2, T, D, generator=gen, device="cuda").to(dtype) for _ in range(4))
    leaves = {"x": x, "s": s, **w}
    for t in leaves.values():
        t.requires_grad_()
    y, stream, _, _ = block(x, s, w)
    got = torch.autograd.grad([y, stream], list(leaves.values()), [dy, ds])
    wide = {n: t.detach().double().requires_grad_() for n, t in leaves.items()}
    ry, rs = reference(wide["x"], wide["s"], wide)
    want = torch.autograd.grad([ry, rs], list(wide.values()), [dy.double(), ds.double()])
    half = torch.finfo(dtype).eps / 2
    assert _rel(y, ry) <= 16 * half and _rel(stream, rs) <= 16 * half
    for name, a, b in zip(leaves, got, want):
        assert a.dtype == leaves[name].dtype and _rel(a, b) <= 32 * half, (name, _rel(a, b), 32 * half)


@torch.no_grad()
def test_block_decoding_follows_the_prompt():
    w = _weights(torch.bfloat16)
    x, s = (torch.randn(3, 70, D, device="cuda").bfloat16() for _ in range(2))
    y, stream, _, final = block(x, s, w)
    conv = torch.zeros(3, 3, 3 * H * K, device="cuda", dtype=torch.bfloat16)
    state, steps = torch.zeros(3, H, K, K, device="cuda"), []
    for t in range(70):
        yt, st, conv, state = block(x[:, t:t + 1], s[:, t:t + 1], w, conv, state)
        steps.append((yt, st))
    # both are 16 half steps from the exact values
    assert _rel(torch.cat([a for a, _ in steps], 1), y) <= 32 * 2.0 ** -8
    assert _rel(torch.cat([b for _, b in steps], 1), stream) <= 32 * 2.0 ** -8
    assert _rel(state, final) <= 32 * 2.0 ** -8


@torch.no_grad()
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_eight_bit_projections_behind_the_norm(rows):
    gen = torch.Generator(device="cuda").manual_seed(2)
    x, s = (torch.randn(rows, D, generator=gen, device="cuda").bfloat16() for _ in range(2))
    n = 1 + 0.1 * torch.randn(D, generator=gen, device="cuda")
    w, up = (torch.randn(F, D, generator=gen, device="cuda") / 16 for _ in range(2))
    (wq, ws), (uq, us) = (((m / sc[:, None]).to(torch.float8_e4m3fn), sc) for m, sc in ((m, m.abs().amax(1) / 448) for m in (w, up)))
    q, scale, stream = layers.rms_norm(x, n, residual=s, out_dtype=torch.float8_e4m3fn)
    y = layers.linear(q, wq, x_scale=scale, weight_scale=ws)
    h = layers.gated_linear(q, wq, uq, x_scale=scale, gate_scale=ws, up_scale=us)
    t = x.double() + s.double()
    e = t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * n.double()
    # every value of both operands is off by half a step of e4m3 at most (2^-4; 2^-10 of a row's scale where subnormal, far
    # less): a product by 2^-3 of its terms, which add up to no more than the terms' norms
    g, u = e @ w.double().t(), e @ up.double().t()
    off = 2.0 ** -3 * (e.abs() @ w.abs().double().t()) + 1e-2
    assert bool(((y.double() - g).abs() <= off + 2.0 ** -8 * g.abs()).all())
    assert _rel(y, g) <= 2.0 ** -3 and _rel(h, torch.nn.functional.silu(g) * u) <= 2.0 ** -2
    assert _rel(stream, t) <= 2.0 ** -8


def test_decoding_step_captured_and_replayed():
    w = _weights(torch.float16)
    x, s = torch.randn(5, 1, D, device="cuda").half(), torch.randn(5, 1, D, device="cuda").half()
    conv, state = torch.zeros(5, 3, 3 * H * K, device="cuda", dtype=torch.float16), torch.randn(5, H, K, K, device="cuda")
    with torch.no_grad():
        block(x, s, w, conv, state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, s, w, conv, state)
        for seed in range(3):
            torch.manual_seed(seed)
            x.copy_(torch.randn_like(x)), s.copy_(torch.randn_like(s)), state.copy_(torch.randn_like(state))
            graph.replay()
            for a, b in zip(out, block(x, s, w, conv, state)):
                assert bool((a == b).all())


@pytest.mark.parametrize("rows", [30, 2100, 8300])
def test_training_step_captured_and_replayed(rows):
    def step(x, w, up, n, b, dy):
        leaves = [x, w, up, n, b]
        h = layers.gated_linear(layers.rms_norm(x, n), w, up)
        y = layers.linear(layers.linear(h, up.t(), activation="silu"), w, b, activation="gelu")
        return torch.autograd.grad(y, leaves, dy)

    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, 64, generator=gen, device="cuda").bfloat16().requires_grad_()
    w, up = ((torch.randn(72, 64, generator=gen, device="cuda") / 8).bfloat16().requires_grad_() for _ in range(2))
    n, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(72, device="cuda", requires_grad=True)
    dy = torch.randn(rows, 72, generator=gen, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, w, up, n, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, up, n, b, dy)
    for seed in range(2):
        torch.manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn_like(x)), dy.copy_(torch.randn_like(dy))
        graph.replay()
        for a, c in zip(out, step(x, w, up, n, b, dy)):
            assert bool((a == c).all())


@pytest.mark.parametrize("op", ["rms_norm", "linear", "gated_linear"])
def test_capture_while_an_eager_graph_lives(op):
    """The leaves' gradients would be handed over on the eager graph's stream, outside of the capture: refused, until that
    graph is gone or where it is another leaf's."""
    x, w = (torch.randn(64, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    n = torch.ones(64, device="cuda", requires_grad=True)
    second = n if op == "rms_norm" else w
    call = {"rms_norm": lambda: layers.rms_norm(x, n), "linear": lambda: layers.linear(x, w),
            "gated_linear": lambda: layers.gated_linear(x, w, w)}[op]

    def step(leaves):
        y = call()
        return torch.autograd.grad(y, leaves, torch.ones_like(y))

    want = step([x, second])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([x, second])
    torch.cuda.synchronize()
    alive = call()
    for leaves in ([x, second], [second]):
        with pytest.raises(RuntimeError, match="eager autograd graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                step(leaves)
    del alive
    alive = second * 2 if op == "rms_norm" else second + 1  # of the second leaf only
    for leaves, at in (([x], 0), ([x, second], None)):
        if at is None:
            del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(leaves)
        graph.replay()
        assert all(bool((a == b).all()) for a, b in zip(out, want))


def test_two_streams_at_once():
    w = [_weights(torch.bfloat16, seed) for seed in range(2)]
    x = [torch.randn(2, 600, D, device="cuda").bfloat16() for _ in range(2)]
    s = [torch.randn(2, 600, D, device="cuda").bfloat16() for _ in range(2)]
    with torch.no_grad():
        want = [block(x[i], s[i], w[i])[:2] for i in range(2)]
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    got[i] = block(x[i], s[i], w[i])[:2]
        torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(bool((p == q).all()) for p, q in zip(a, b))


@pytest.mark.parametrize("rows", [3, 100, 2100, 8300])
def test_kernels_that_overlap_see_what_was_written_before(rows):
    """Blocks of a kernel start while the one before still runs: every input, weights and scales among them, is written by the
    kernel just before, torch's or one of these."""
    def chain(wait):
        torch.manual_seed(5)
        x = torch.randn(rows, 512, device="cuda").bfloat16()
        w, up, down = ((torch.randn(512, 512, device="cuda") / 23).bfloat16() for _ in range(3))
        n, b = torch.ones(512, device="cuda"), torch.zeros(512, device="cuda")
        seen = []
        for i in range(30):
            n.add_(0.01), wait()
            y, x = layers.rms_norm(x, n, residual=x)
            wait(), w.mul_(0.999), wait()
            h = layers.gated_linear(y, w, up)
            wait(), b.add_(0.01), wait()
            x = layers.linear(h, down, b, residual=x, activation="silu")
            wait(), up.copy_(down), wait()
            q, scale = layers.rms_norm(x, n, out_dtype=torch.float8_e4m3fn)
            wait()
            wq, ws = w.to(torch.float8_e4m3fn), torch.full((512,), 1 / (i + 1), device="cuda")
            z = layers.linear(q, wq, x_scale=scale, weight_scale=ws)
            wait(), x.copy_(z + x), wait()
            seen.append(x.clone())
        leaf = x.clone().requires_grad_()
        y = layers.linear(layers.rms_norm(leaf, n), w, b, activation="gelu")
        wait()
        seen += torch.autograd.grad(y, [leaf], x)
        return seen

    def still():
        torch.cuda.synchronize()

    for a, c in zip(chain(lambda: None), chain(still)):
        assert bool((a == c).all())


def test_two_host_threads_at_once():
    import threading

    w = _weights(torch.bfloat16)
    for t in w.values():
        t.requires_grad_()
    data = [[torch.randn(2, rows, D, device="cuda").bfloat16() for _ in range(2)] for rows in (40, 500)]
    leaves = [w[n] for n in ("qkv", "gate", "up", "down", "n1")]

    def step(x, s):
        y, stream, _, _ = block(x, s, w)
        return [y.detach(), *torch.autograd.grad(y, leaves, stream.detach())]

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    got[i] = step(*data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as err:  # noqa: BLE001 (shown by the assertion below)
            errors.append(err)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(want, got):
        # (the layers around these operators add gradients up with atomics: equal to a rounding, not to the bit)
        assert bool((a[0] == b[0]).all()) and all(_rel(q, p) <= 2.0 ** -7 for p, q in zip(a[1:], b[1:]))


def test_one_tensor_for_several_arguments():
    x = torch.randn(64, 64, device="cuda").bfloat16().requires_grad_()
    n, dy = torch.ones(64, device="cuda"), torch.randn(64, 64, device="cuda").bfloat16()
    a, b = (x.detach().clone().requires_grad_() for _ in range(2))
    for call in (lambda p, q: layers.linear(p, q), lambda p, q: layers.rms_norm(p, n, residual=q)[0]):
        one, = torch.autograd.grad(call(x, x), [x], dy)
        two = torch.autograd.grad(call(a, b), [a, b], dy)
        assert bool((one == two[0] + two[1]).all())
    c = x.detach().clone().requires_grad_()
    for call in (lambda p, q, r: layers.linear(p, q, residual=r, activation="silu"), lambda p, q, r: layers.gated_linear(p, q, r)):
        one, = torch.autograd.grad(call(x, x, x), [x], dy)
        three = torch.autograd.grad(call(a, b, c), [a, b, c], dy)
        # three terms, added two by two in whatever order: two roundings of half a step each, of sums no larger than all terms'
        size = sum(t.double().abs() for t in three)
        assert bool(((one.double() - sum(t.double() for t in three)).abs() <= 2 * 2.0 ** -8 * size).all())
    y, stream = layers.rms_norm(x, n, residual=x)
    assert bool((stream == 2 * x).all())


def test_offsets_beyond_32_bits():
    rows, dim = 1_100_000, 2048  # 2.25e9 elements
    x = torch.randn(rows, dim, device="cuda", dtype=torch.bfloat16)
    w = 1 + 0.1 * torch.randn(dim, device="cuda")
    y, stream = layers.rms_norm(x, w, residual=x)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        a, b = layers.rms_norm(x[part], w, residual=x[part])
        assert bool((y[part] == a).all()) and bool((stream[part] == b).all())
    del y, stream
    small = x[:, :64]  # rows that lie 2048 elements apart
    m = (torch.randn(dim, 64, device="cuda") / 8).bfloat16()
    y = layers.linear(small, m, residual=x)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        a = layers.linear(small[part].contiguous(), m, residual=x[part].contiguous())
        assert _rel(y[part], a) <= 2.0 ** -8
    del y
    leaf, wm = small.detach().contiguous().requires_grad_(), m.clone().requires_grad_()
    y = layers.linear(leaf, wm, activation="silu")
    dx, = torch.autograd.grad(y, [leaf], x)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        p = leaf[part].detach().requires_grad_()
        d, = torch.autograd.grad(layers.linear(p, wm, activation="silu"), [p], x[part])
        assert _rel(dx[part], d) <= 2.0 ** -7


def test_second_derivatives_and_transforms_are_refused():
    x = torch.randn(8, 64, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(64, 64, device="cuda") / 8).bfloat16().requires_grad_()
    n = torch.ones(64, device="cuda", requires_grad=True)
    for y, leaves in ((layers.linear(x, w, activation="silu"), [x, w]), (layers.gated_linear(x, w, w), [x, w]),
                      (layers.rms_norm(x, n), [x, n])):
        g = torch.autograd.grad(y, leaves, torch.ones_like(y), create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated"):
            torch.autograd.grad(g[0].float().sum(), leaves)
    with torch.no_grad():
        a, b = x.detach(), w.detach()
        with pytest.raises(Exception):
            torch.func.vmap(lambda v: layers.linear(v, b))(a.view(2, 4, 64))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(a, torch.ones_like(a))
        for call in (lambda: layers.linear(dual, b), lambda: layers.gated_linear(dual, b, b), lambda: layers.rms_norm(dual, n.detach())):
            with pytest.raises(Exception):
                call()


def test_inference_mode_and_shared_weights():
    x = torch.randn(8, 64, device="cuda").bfloat16()
    w = (torch.randn(64, 64, device="cuda") / 8).bfloat16()
    with torch.no_grad():
        want = layers.linear(x, w), layers.gated_linear(x, w, w), layers.rms_norm(x, w[0])
    with torch.inference_mode():
        got = layers.linear(x, w), layers.gated_linear(x, w, w), layers.rms_norm(x, w[0])
    assert all(bool((a == b).all()) for a, b in zip(want, got))
    p = torch.nn.Parameter(w)  # one weight for both: its gradient is the sum of two
    a, b = w.clone().requires_grad_(), w.clone().requires_grad_()
    dy = torch.randn(8, 64, device="cuda").bfloat16()
    one, = torch.autograd.grad(layers.gated_linear(x, p, p), [p], dy)
    two = torch.autograd.grad(layers.gated_linear(x, a, b), [a, b], dy)
    assert bool((one == (two[0] + two[1])).all())
    lazy = torch.complex(torch.zeros(4, 64, device="cuda"), torch.randn(4, 64, device="cuda")).conj().imag  # a negated view
    assert lazy.is_neg() and bool((layers.rms_norm(lazy, torch.ones(64, device="cuda")) ==
                                   layers.rms_norm(lazy.clone(), torch.ones(64, device="cuda"))).all())
