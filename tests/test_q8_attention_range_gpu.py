"""attention_kv8 where every score that a query sees lies far below zero: the softmax only sees differences."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from block_transformer_amd import ops  # noqa: E402
from block_transformer_amd.runtime import KV8Cache  # noqa: E402

DEV = "cuda"


@pytest.mark.parametrize("n", [1, 5, 16, 17, 64, 200, 1100])
@pytest.mark.parametrize("n_split", [1, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e14, 1e16, 1e17])
def test_scores_far_below_zero(n, n_split, dtype, size):
    """q = -size, k = 2 size in every row but one, which has size: all scores are -size^2 sqrt(d) and twice that (1e28 .. 1e35, in
    natural units), the softmax is 1 at that row, and the result is its v -- a code times a scale, or the open block's row as it is."""
    B, heads, H, d, block = 2, 4, 2, 64, 16
    g = torch.Generator().manual_seed(n)
    k = torch.full((B, n, H, d), 2 * size)
    at = torch.randint(0, n, (B, H), generator=g)
    for b in range(B):
        for h in range(H):
            k[b, at[b, h], h] = size
    v = torch.randn(B, n, H, d, generator=g)
    q = torch.full((B, 1, heads, d), -size)
    kv = KV8Cache(1, B, H, n, d, dtype, DEV, block=block)[0]
    ops.kv8_append(kv, None, k.to(dtype).to(DEV), v.to(dtype).to(DEV), 0)
    rows = ops.kv8_read(kv, n)[1]
    out = ops.attention_kv8(q.to(dtype).to(DEV), kv, n - 1, n_split=n_split)
    want = torch.stack([rows[b, h // (heads // H), at[b, h // (heads // H)]] for b in range(B) for h in range(heads)]).view(B, 1, heads, d)
    # one weight of 1 and none beside it: the row's v, rounded to dtype as kv8_read does it, up to a few roundings of fp32 before that
    u = torch.finfo(dtype).eps / 2
    assert ((out - want).abs().double() <= (2 * u + 8 * 2 ** -24) * want.abs().double() + 1e-6 * float(v.abs().max())).all()
