"""What the operators of the compiled binding do not differentiate is refused: dual inputs, as ``co_alibi_attention``
refuses them, rather than answered without their tangent, and pools that require grad.  On the CPU the binding itself,
which refuses before it looks for a device; on the GPU the calls."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _call(name, device, args):
    """The operator `name` with keywords `args`; by the binding (whose arguments go by position) on the CPU."""
    import co_alibi_attn
    if device == "cuda":
        return getattr(co_alibi_attn, name)(**args)
    from co_alibi_attn.serving import _native
    order = {"norm_rotate_qkv": ("qkv", "num_heads", "num_kv_heads", "q_weight", "k_weight", ("eps", 1e-6), "rotary", "start", "positions",
                                 ("interleaved", False), "status"),
             "append_paged_kv": ("k", "v", "k_pages", "v_pages", "page_table", "start", "count", "q", "rotary", ("interleaved", False), "positions",
                                 "status", "scales"),
             "paged_tree_attention": ("q", "k_pages", "v_pages", "page_table", "ctx_lens", "tree_mask", "sm_scale", "slopes", "status", "scales")}[name]
    args = {**args, "status": torch.zeros(1, dtype=torch.int32)}
    return getattr(_native(), name)(*(args.get(k, None) if isinstance(k, str) else args.get(*k) for k in order))


def _inputs(name, device, codes):
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
    if name == "norm_rotate_qkv":
        return dict(qkv=z(2, 3, 6, 64), num_heads=2, num_kv_heads=2, q_weight=z(64), k_weight=z(64), rotary=(z(4, 16, dt=torch.float32), z(4, 16, dt=torch.float32)))
    pool = lambda: z(3, 2, 16, 64, dt=torch.uint8).view(torch.float8_e4m3fn) if codes else z(3, 2, 16, 64)  # noqa: E731
    args = dict(k_pages=pool(), v_pages=pool(), page_table=z(2, 1, dt=torch.int32))
    if codes:
        args["scales"] = (z(3, 2, 1, dt=torch.float32), z(3, 2, 1, dt=torch.float32))
    if name == "append_paged_kv":
        return dict(**args, k=z(2, 2, 3, 64), v=z(2, 2, 3, 64), q=z(2, 4, 3, 64), start=z(2, dt=torch.int32))
    return dict(**args, q=z(2, 4, 1, 64), ctx_lens=z(2, dt=torch.int32), slopes=z(4))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name,dual,codes", [("norm_rotate_qkv", n, False) for n in ("qkv", "q_weight", "k_weight", "rotary")]
                         + [("append_paged_kv", n, c) for n in ("k", "v", "q") for c in (False, True)]
                         + [("paged_tree_attention", n, c) for n in ("q", "slopes") for c in (False, True)]
                         + [(op, "scales", True) for op in ("append_paged_kv", "paged_tree_attention")])
def test_dual_inputs_are_refused(name, dual, codes, device):
    args = _inputs(name, device, codes)
    with fwd.dual_level():
        make = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        args[dual] = (args[dual][0], make(args[dual][1])) if isinstance(args[dual], tuple) else make(args[dual])
        for ctx in (torch.enable_grad(), torch.no_grad()):
            with ctx, pytest.raises(RuntimeError, match="forward-mode"):
                _call(name, device, args)


@pytest.mark.gpu
def test_plain_calls_beside_dual_tensors():
    """Inputs without a tangent run inside a dual level, with their reverse-mode graph; so do detached ones."""
    import co_alibi_attn
    x = torch.randn(2, 3, 6, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    want, = torch.autograd.grad(co_alibi_attn.norm_rotate_qkv(x, 2, 2)[0].sum(), x)
    with fwd.dual_level():
        got, = torch.autograd.grad(co_alibi_attn.norm_rotate_qkv(x, 2, 2)[0].sum(), x)
        dual = fwd.make_dual(x.detach(), torch.ones_like(x))
        plain = fwd.unpack_dual(dual).primal
        assert torch.equal(co_alibi_attn.norm_rotate_qkv(plain, 2, 2)[0], co_alibi_attn.norm_rotate_qkv(x.detach(), 2, 2)[0])
    assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("name", ["k_pages", "v_pages", "k_scales", "v_scales"])
def test_reading_refuses_what_requires_grad(name, device):
    """As append and attention do; pools of codes are floating tensors to autograd."""
    import co_alibi_attn
    from co_alibi_attn.serving import _native
    z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
    t = {n: z(3, 2, 16, 64, dt=torch.uint8).view(torch.float8_e4m3fn) for n in ("k_pages", "v_pages")}
    t.update({n: z(3, 2, 1, dt=torch.float32) for n in ("k_scales", "v_scales")})
    t[name].requires_grad_()
    args = t["k_pages"], t["v_pages"], z(2, 1), z(2, 3), (t["k_scales"], t["v_scales"])
    with pytest.raises(RuntimeError, match="no_grad"):
        if device == "cuda":
            co_alibi_attn.read_paged_kv(*args)
        else:
            _native().read_paged_kv(*args, True, z(1))
    if device == "cuda":
        with torch.no_grad():
            assert not co_alibi_attn.read_paged_kv(*args)[0].requires_grad
