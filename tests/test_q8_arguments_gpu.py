"""Calls of the 8-bit operators that their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from block_transformer_amd import ops  # noqa: E402
from block_transformer_amd._lib import BtError  # noqa: E402
from block_transformer_amd.runtime import KV8Cache  # noqa: E402
from oracle import q8_ref as ref  # noqa: E402

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("K", [1, 5, 13, 515, 2047])
@pytest.mark.parametrize("M", [1, 5, 3000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_of_large_constant_rows(M, K, dtype):
    """What a lane holds behind the row's end does not count: (0 - mean) * rstd may leave fp32 there.  The rows are one power of two, so that
    sums, mean and differences are exact whatever their order: the LayerNorm of such a row is its bias, to the last bit."""
    x = torch.full((M, K), 2.0 ** (126 - K.bit_length()), dtype=dtype)
    g = torch.Generator().manual_seed(K)
    w, b = torch.randn(K, generator=g).to(dtype), torch.randn(K, generator=g).to(dtype)
    c, s = ops.quantize_rows(x.to(DEV), w.to(DEV), b.to(DEV), eps=1e-12)
    want, scale = ref.quantize_rows(b[None])
    assert (s.cpu().double() == scale).all()
    assert (c.cpu()[:, :K].double() == want).all() and not c[:, K:].any()


def test_quantised_rows_say_how_many_columns_they_have():
    x, w = torch.randn(3, 515, device=DEV), torch.randn(8, 520, device=DEV)
    cx, cw = ops.quantize_rows(x), ops.quantize_rows(w)
    assert cx[0].columns == 515 and cw[0].columns == 520
    for rows in (x, cx):
        with pytest.raises(BtError, match="515 columns, the weight 520"):
            ops.linear_q8(rows, cw, dtype=F32)
    assert torch.equal(ops.linear_q8(x, ops.quantize_rows(w[:, :515])), ops.linear_q8(cx, ops.quantize_rows(w[:, :515]), dtype=F32))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_with_a_rotary_table_of_no_columns(dtype):
    """rope_tables(n, 0): nothing is rotated, q comes back as it is."""
    B, H, d, n = 2, 2, 32, 20
    x = torch.randn(B, n, 3, H, d, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    a, b = (KV8Cache(1, B, H, n, d, dtype, DEV)[0] for _ in range(2))
    for t in a + b:
        t.zero_()
    q = x[:, :, 0]
    none = ops.rope_tables(64, 0, 10000.0, DEV)
    assert ops.kv8_append(a, q, x[:, :, 1], x[:, :, 2], 0, rope=none) is q
    assert ops.kv8_append(b, q, x[:, :, 1], x[:, :, 2], 0) is q
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_attention_with_one_mask_for_all_sequences():
    """mask.expand(B, n): a batch stride of 0."""
    B, H, d, n = 3, 2, 64, 100
    x = torch.randn(B, n, 2, H, d, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    kv = KV8Cache(1, B, H, n, d, BF16, DEV)[0]
    ops.kv8_append(kv, None, x[:, :, 0], x[:, :, 1], 0)
    mask = (torch.arange(n, device=DEV) % 3 != 0)[None]
    for m in (mask, mask.to(torch.uint8)):
        got = ops.attention_kv8(x[:, -1:, 0], kv, n - 1, mask=m.expand(B, n))
        assert torch.equal(got, ops.attention_kv8(x[:, -1:, 0], kv, n - 1, mask=m.repeat(B, 1)))


@pytest.mark.parametrize("back_to", [70, 65, 64, 48, 16, 0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_taken_back(back_to, dtype):
    """Inside the open block (64 .. 70) or to the start of any block: the cache is that of the rows that stayed and those that came."""
    B, H, d, n = 2, 2, 64, 71
    x = torch.randn(B, 2 * n, 2, H, d, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    a, b = (KV8Cache(1, B, H, 2 * n, d, dtype, DEV)[0] for _ in range(2))
    ops.kv8_append(a, None, x[:, :n, 0], x[:, :n, 1], 0)
    ops.kv8_append(a, None, x[:, n:, 0], x[:, n:, 1], back_to)
    rows = torch.cat([x[:, :back_to], x[:, n:]], 1)
    ops.kv8_append(b, None, rows[:, :, 0], rows[:, :, 1], 0)
    for s, t in zip(ops.kv8_read(a, back_to + n), ops.kv8_read(b, back_to + n)):
        assert torch.equal(s, t)
    q = x[:, :1, 0]
    assert torch.equal(ops.attention_kv8(q, a, back_to + n - 1), ops.attention_kv8(q, b, back_to + n - 1))
