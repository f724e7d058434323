"""The attention operator inside CUDA graphs: forward, decode forward and backward, captured
once and replayed on changed inputs, give what the same calls give outside."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Sq,Skv,causal", [(300, 300, True), (130, 257, False), (1, 500, True), (16, 700, False)])
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_forward_and_backward(Sq, Skv, causal, dt):
    from co_alibi_attn import co_alibi_attention, device_status
    Hq, Hkv, D = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dt)  # noqa: E731
    shapes = ((2, Hq, Sq, D), (2, Hkv, Skv, D), (2, Hkv, Skv, D), (2, Hq, Sq, D))
    inputs = [tuple(rand(*s) for s in shapes) for _ in range(2)]

    def step(q, k, v, do):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        o = co_alibi_attention(q, k, v, causal=causal)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [[t.clone() for t in step(*x)] for x in inputs]
        again = [t.clone() for t in step(*inputs[0])]
    torch.cuda.current_stream().wait_stream(side)
    repeats = [torch.equal(a, b) for a, b in zip(again, want[0])]  # (all but what atomics sum)
    static = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for x, expect in ((inputs[1], want[1]), (inputs[0], want[0])):
        for s, t in zip(static, x):
            s.copy_(t)
        graph.replay()
        for a, b, same in zip(out, expect, repeats):
            if same:
                assert torch.equal(a, b)
            else:
                assert (a.float() - b.float()).norm() <= 1e-3 * b.float().norm()
    assert device_status(reset=True) == 0


def test_a_capturing_stream_of_the_call():
    """Forward calls on an explicit stream under capture, beside ones that are not captured."""
    from co_alibi_attn import co_alibi_attention
    q, k, v = (torch.randn(1, 2, 90, 128, device="cuda").half() for _ in range(3))
    want = co_alibi_attention(q, k, v)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = co_alibi_attention(q, k, v)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(co_alibi_attention(q, k, v), want)
