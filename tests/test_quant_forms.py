"""The 8-bit cache's append and read in the forms that their launches choose: many heads to a CTA, heads that do not
fill their warps, the longest batch."""
import pytest
import torch

from tests import _quant_ref as qr

f16, bf16 = torch.float16, torch.bfloat16


@pytest.mark.gpu
def test_as_many_tokens_as_an_int_counts():
    """All padding but one page's: an expanded row, so that nothing of the size is held."""
    import co_alibi_attn
    D, S = 64, (1 << 31) - 1
    row = torch.linspace(-2, 2, D, device="cuda").to(f16)
    x = row.expand(1, 1, S, D)
    codes = [qr.e4m3(torch.full((2, 1, 16, D), 0x7f, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    scales = tuple(torch.ones(2, 1, 1, device="cuda") for _ in range(2))
    table = torch.ones(1, 1, dtype=torch.int32, device="cuda")
    start, count = torch.full((1,), 3, dtype=torch.int32, device="cuda"), torch.full((1,), 13, dtype=torch.int32, device="cuda")
    co_alibi_attn.append_paged_kv(x, x, *codes, table, start, count=count, scales=scales)
    assert co_alibi_attn.device_status(reset=True) == 0
    want = qr.codes_of(row.cpu().double())
    for c in codes:
        got = c.view(torch.uint8).cpu()
        assert (qr.values_of(got[1, 0, 3:]) == qr.values_of(want)).all() and (got[0] == 0x7f).all() and (got[1, 0, :3] == 0x7f).all()
