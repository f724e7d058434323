"""Rotary positions of the training model: the tables are built once, not per layer and step."""
import pytest
import torch

from tests.test_gpt import oracle_attention


def _cfg(**kw):
    from co_alibi_gpt import GPTConfig
    return GPTConfig(**{**dict(n_layer=3, d_model=128, n_head=2, vocab=97, seq_len=24, rotary_dim=32), **kw})


def test_tables_are_built_once_and_grow(monkeypatch):
    from co_alibi_attn import serving
    from co_alibi_gpt import build
    made, real = [], serving.rotary_tables
    monkeypatch.setattr(serving, "rotary_tables", lambda dim, n, **kw: made.append((dim, n)) or real(dim, n, **kw))
    monkeypatch.setattr("co_alibi_gpt.model._rotary_cache", {})
    model, _ = build(_cfg(), "cpu", seed=1, dtype=torch.float32, attn_fn=oracle_attention)
    tok = torch.randint(0, 97, (2, 50), generator=torch.Generator().manual_seed(2))
    short = model(tok[:, :7])
    model(tok[:, :24], targets=tok[:, 1:25]).backward()
    assert made == [(32, 24)]
    full = model(tok)  # longer than the configuration's length
    assert len(made) == 2 and made[1][1] >= 50
    assert torch.allclose(full[:, :7], short, atol=1e-5)


@pytest.mark.gpu
def test_a_training_step_can_be_captured():
    from co_alibi_gpt import build
    model, _ = build(_cfg(), "cuda", seed=1, dtype=torch.float16)
    tok = torch.randint(0, 97, (2, 25), generator=torch.Generator().manual_seed(2)).cuda()

    def step():
        for p in model.parameters():
            p.grad = None
        loss = model(tok[:, :-1], targets=tok[:, 1:])
        loss.backward()
        return loss.detach(), [p.grad for p in model.parameters()]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = [step() for _ in range(2)][-1]
        want = want[0].clone(), [g.clone() for g in want[1]]
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grads = step()
    graph.replay()
    assert (loss - want[0]).abs() <= 2e-3
    for g, w in zip(grads, want[1]):
        assert (g.float() - w.float()).abs().max() <= 1e-2 * w.float().abs().max() + 1e-6


@pytest.mark.parametrize("rotary_dim", [-16, 8, 24, 33, 80])
def test_widths_that_the_cache_does_not_take_are_refused(rotary_dim):
    from co_alibi_gpt import CoALiBiGPT
    with pytest.raises(ValueError):
        CoALiBiGPT(_cfg(rotary_dim=rotary_dim), oracle_attention)
    CoALiBiGPT(_cfg(rotary_dim=64), oracle_attention)
