"""What the package builds on first use and keeps (slope tables, the status word, rotary
tables): usable in any mode whatever mode the first call ran in."""
import pytest
import torch


def _fresh(monkeypatch):
    from co_alibi_attn import co_alibi_attn as core
    from co_alibi_gpt import model
    monkeypatch.setattr(core, "_slope_cache", {})
    monkeypatch.setattr(core, "_status_cache", {})
    monkeypatch.setattr(model, "_rotary_cache", {})
    return core, model


def test_built_in_inference_mode_used_in_training(monkeypatch):
    core, model = _fresh(monkeypatch)
    cpu = torch.device("cpu")
    with torch.inference_mode():
        built = [core._api_slopes(6, 8.0, torch.float32, cpu), core._status_word(cpu), *model._rotary(16, 8, 5, cpu)]
    assert not any(t.is_inference() for t in built)
    x = torch.ones(6, requires_grad=True)
    (x * built[0]).sum().backward()  # saves the table
    assert torch.equal(x.grad, built[0])
    built[1].zero_()


@pytest.mark.gpu
def test_first_calls_in_inference_mode(monkeypatch):
    import co_alibi_attn
    _fresh(monkeypatch)
    q, k, v = (torch.randn(1, 2, 40, 64, device="cuda").half() for _ in range(3))
    with torch.inference_mode():
        o = co_alibi_attn.co_alibi_attention(q, k, v)
    assert co_alibi_attn.device_status(reset=True) == 0
    q2 = q.clone().requires_grad_()
    out = co_alibi_attn.co_alibi_attention(q2, k, v)
    out.sum().backward()
    assert torch.equal(out, o) and torch.isfinite(q2.grad).all()


@pytest.mark.gpu
def test_first_calls_inside_a_capture_are_refused(monkeypatch):
    import co_alibi_attn
    from co_alibi_attn import append_paged_kv, co_alibi_attention, paged_tree_attention
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    k, pages, table, lens = z(1, 2, 1, 64), z(3, 2, 16, 64), z(1, 1, dt=torch.int32), z(1, dt=torch.int32)
    x = z(1, 2, 40, 64)
    calls = (lambda: append_paged_kv(k, k, pages, pages.clone(), table, lens),
             lambda: paged_tree_attention(k, pages, pages, table, lens, slopes=z(2)),
             lambda: paged_tree_attention(k, pages, pages, table, lens),
             lambda: co_alibi_attention(x, x, x))
    for call in calls:
        core, _ = _fresh(monkeypatch)
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        assert not core._status_cache and not core._slope_cache
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graph.replay()
        assert co_alibi_attn.device_status(reset=True) == 0
