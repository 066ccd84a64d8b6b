"""The norm and the products on streams that wait for one another: a kernel that may start while the one before it on its own stream still
runs has to wait for events of other streams all the same, eagerly and in captured graphs."""

import pytest
import torch

from jax_linear_attention_b200 import layers

pytestmark = pytest.mark.gpu


def _work(rows):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, r = (torch.randn(rows, 512, generator=gen, device="cuda").bfloat16() for _ in range(2))
    w, up = ((torch.randn(512, 512, generator=gen, device="cuda") / 23).bfloat16() for _ in range(2))
    return x, r, w, up, torch.ones(512, device="cuda")


def _chain(t, a, b, slow, steps):
    """Two streams that hand each other their results; ``slow``: cycles that a producer is held up for before it writes."""
    x, r, w, up, n = t
    seen = []
    p, q = x, r
    for i in range(steps):
        with torch.cuda.stream(b):  # this stream's last kernel is one of ours, and early to let the next one in
            own = layers.linear(q, w)
        with torch.cuda.stream(a):
            if slow:
                torch.cuda._sleep(slow)
            p = layers.gated_linear(layers.rms_norm(p, n), w, up) + 1
        ready = a.record_event()
        b.wait_event(ready)
        with torch.cuda.stream(b):
            q = layers.linear(p, up, residual=own, activation="silu")
        back = b.record_event()
        a.wait_event(back)
        with torch.cuda.stream(a):
            p, _ = layers.rms_norm(q, n, residual=p)
        seen += [p, q]
    b.wait_event(a.record_event())
    a.wait_event(b.record_event())
    return seen


@pytest.mark.parametrize("rows", [3, 100, 3000])
@torch.no_grad()
def test_events_between_streams(rows):
    t = _work(rows)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    one = torch.cuda.current_stream()
    want = _chain(t, one, one, 0, 6)
    torch.cuda.synchronize()
    for slow in (0, 200_000):
        got = _chain(t, a, b, slow, 6)
        torch.cuda.synchronize()
        assert all(bool((p == q).all()) for p, q in zip(got, want))


@pytest.mark.parametrize("rows", [3, 100, 3000])
@torch.no_grad()
def test_events_between_streams_in_a_graph(rows):
    t = _work(rows)
    one = torch.cuda.current_stream()
    want = _chain(t, one, one, 0, 4)
    torch.cuda.synchronize()
    for slow in (0, 200_000):
        a, b, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=a):
            b.wait_event(a.record_event())
            got = _chain(t, a, b, slow, 4)
        for _ in range(3):
            for g in got:
                g.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(bool((p == q).all()) for p, q in zip(got, want))


@torch.no_grad()
def test_copies_and_fills_between_the_kernels():
    """What is not a kernel stands between two of them: a copy from the host, a fill, a copy back."""
    x, _, w, _, n = _work(40)
    host, out = torch.randn(512).pin_memory(), torch.empty(40, 512, dtype=torch.bfloat16).pin_memory()
    copies = []
    for i in range(20):
        n.copy_(host, non_blocking=True)
        y = layers.rms_norm(x, n)
        z = layers.linear(y, w)
        y.zero_()
        copies.append(layers.linear(y, w))
        out.copy_(z, non_blocking=True)
        torch.cuda.current_stream().synchronize()
        want = layers.linear(layers.rms_norm(x, host.cuda()), w)
        assert bool((out.cuda() == want).all()) and not bool(copies[-1].any())
        host.copy_(torch.randn(512))
