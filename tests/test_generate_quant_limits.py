"""Generation with normed heads and over a cache in 8 bits: the edges of the cache and of the arguments."""
import pytest
import torch

from tests.test_generate_quant import E4M3, _cfg, _model
from tests.test_quant_append import _tables


@pytest.mark.gpu
def test_small_values_of_a_float16_model_move_whole():
    """Accepted tokens keep their values where float16 has none for their codes."""
    from co_alibi_attn import append_paged_kv, read_paged_kv
    from co_alibi_gpt import generate as gen
    model = _model(_cfg())
    cache = gen.PagedCache(model, 2, 60, page_size=16, kv_dtype=E4M3)
    H, D, n = 2, 64, 40
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, H, n, D, generator=g).clamp(-1, 1) * 2.0 ** torch.randint(-9, 1, (2, H, n, D), generator=g)
    x[..., -1] = 2.0  # the same scale in every block (rotated elements are at most 2^0.5)
    x = (x * 2.0 ** -15).half().cuda()
    rotary = tuple(t.cuda() for t in _tables(n, 32))  # rotated keys enter the cache from float32
    for layer, (k, v) in enumerate(zip(cache.k, cache.v)):
        append_paged_kv(x, x, k, v, cache.table, cache.lens, rotary=rotary, **cache.of(layer))
    cache.lens += 22
    path = torch.tensor([[23, 26, 31, 39], [24, 25, 38, 22]], dtype=torch.int32).cuda()
    read = lambda layer, at: read_paged_kv(cache.k[layer], cache.v[layer], cache.table, at, cache.scales[layer])  # noqa: E731
    want = [read(layer, path) for layer in range(2)]
    assert float(want[0][0].abs().max()) == 2.0 ** -14 and (want[0][0].float() != want[0][0].half().float()).any()
    cache.move(path, torch.tensor([4, 2], dtype=torch.int32).cuda())
    at = cache.lens[:, None] + torch.arange(4, dtype=torch.int32).cuda()
    for layer in range(2):
        for got, expect in zip(read(layer, at), want[layer]):
            assert torch.equal(got[0], expect[0]) and torch.equal(got[1, :, :2], expect[1, :, :2])
