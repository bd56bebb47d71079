"""Positions of kv8_append that the device reads: whatever number stands there, no table is read outside its rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from block_transformer_amd import ops  # noqa: E402
from block_transformer_amd.runtime import KV8Cache  # noqa: E402
from oracle import q8_ref as ref  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("pos", [31, 32, 1 << 30, 2 ** 31 - 9, 2 ** 31 - 3, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_far_behind_the_end(pos, dtype):
    """pos0 + t may lie behind the last 32-bit number: the queries of all those rows take the position table's last entry, nothing else
    of the cache changes behind its end."""
    B, heads, H, d, block, n, q_len = 2, 4, 2, 64, 16, 32, 7
    g = torch.Generator().manual_seed(pos & 1023)
    x = torch.randn(B, q_len, heads + 2 * H, d, generator=g).to(dtype)
    xg = x.to(DEV)
    kv = KV8Cache(1, B, H, n, d, dtype, DEV, block=block)[0]
    for t in kv:
        t.zero_()
    before = [t.clone() for t in kv]
    table = ops.rope_tables(100, 32, 10000.0, "cpu")
    entries = (torch.arange(n) * 3 + 1).int()
    got = ops.kv8_append(kv, xg[:, :, :heads], xg[:, :, heads:heads + H], xg[:, :, heads + H:], torch.tensor([pos], dtype=torch.int32, device=DEV),
                         rope=table.to(DEV), pos_table=entries.to(DEV))
    at = entries[(pos + torch.arange(q_len)).clamp(max=n - 1)].long()
    assert torch.equal(got.cpu(), ref.rope(x[:, :, :heads], at, table).to(dtype))
    if pos >= n:
        assert all(torch.equal(a, b) for a, b in zip(kv, before))
