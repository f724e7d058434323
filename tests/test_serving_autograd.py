"""The serving operators beside autograd: no result drops its graph silently, and an append is
seen as a write of the pools."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _z(*s, dt=torch.float16):
    return torch.zeros(*s, dtype=dt, device="cuda")


def _append():
    return dict(k=_z(2, 2, 3, 64), v=_z(2, 2, 3, 64), k_pages=_z(3, 2, 16, 64), v_pages=_z(3, 2, 16, 64),
                page_table=_z(2, 1, dt=torch.int32), start=_z(2, dt=torch.int32), q=_z(2, 4, 3, 64))


def _attention():
    return dict(q=_z(2, 4, 1, 64), k_pages=_z(3, 2, 16, 64), v_pages=_z(3, 2, 16, 64),
                page_table=_z(2, 1, dt=torch.int32), ctx_lens=_z(2, dt=torch.int32), slopes=_z(4))


@pytest.mark.parametrize("name", ["k", "v", "q", "k_pages", "v_pages"])
def test_append_refuses_what_requires_grad(name):
    from co_alibi_attn import append_paged_kv
    args = _append()
    args[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        append_paged_kv(**args)
    with torch.no_grad():
        assert not append_paged_kv(**args).requires_grad


@pytest.mark.parametrize("name", ["q", "k_pages", "v_pages", "slopes"])
def test_attention_refuses_what_requires_grad(name):
    from co_alibi_attn import paged_tree_attention
    args = _attention()
    args[name].requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        paged_tree_attention(**args)
    with torch.no_grad():
        assert not paged_tree_attention(**args).requires_grad


def test_an_append_is_a_write_of_the_pools():
    from co_alibi_attn import append_paged_kv
    args = _append()
    base = torch.zeros(4, 2, 16, 64, dtype=torch.float16, device="cuda")
    args["k_pages"] = base[1:]  # a view writes its base
    w = torch.ones(4, 2, 16, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    loss = (base * w).sum()
    versions = base._version, args["v_pages"]._version
    append_paged_kv(**args)
    assert base._version > versions[0] and args["v_pages"]._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_in_inference_mode():
    from co_alibi_attn import append_paged_kv, paged_tree_attention
    with torch.inference_mode():
        append_paged_kv(**_append())
        paged_tree_attention(**_attention())
    args = _append()  # ordinary pools, written in inference mode
    with torch.inference_mode():
        append_paged_kv(**args)
