"""What attention_kv8 keeps of small probabilities, of scales that differ and of queries with outliers.

It multiplies what the cache stands for (code times scale, or the open block's row) with q and with the probabilities in the arithmetic of
an fp32 attention: every q and every probability enters with all its bits, products are exact, sums are fp32.  So a result is off by a few
2^-24 of sum_j p_j |v_j|, however small the p_j are that make it up, beside what the scores are off: their sums are off by about 2^-24 of
sum |q_i k_i| / sqrt(d) (a rounding at every step of the sum, errors of both signs), and a probability by a factor of as much.  In the
2-norm that is below 2e-5 for scores up to a hundred or so; a bf16 result is rounded once more, half a step: 2^-8 at most, and 2e-5 before
it moves that rounding by at most as much again."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from block_transformer_amd import ops  # noqa: E402
from block_transformer_amd.runtime import KV8Cache  # noqa: E402
from oracle import q8_ref as ref  # noqa: E402

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def rnd(*shape, seed, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def attend(k, v, q, block, dtype, mask=None, n_split=0, before=None):
    """(result, oracle) of q over rows k, v [B, n, H, d]; `before` changes the cache first and returns (k, v) in float64 as the cache then
    stands for them, given what it stood for."""
    B, n, H, d = k.shape
    kv, want = KV8Cache(1, B, H, n, d, dtype, DEV, block=block)[0], ref.Cache(B, H, d, block, dtype)
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    ops.kv8_append(kv, None, k.to(DEV), v.to(DEV), 0)
    want.append(k, v)
    rows = want.rows("k")[0], want.rows("v")[0]
    if before:
        rows = before(kv, *rows)
    out = ops.attention_kv8(q.to(DEV), kv, n - q.shape[1], mask=None if mask is None else mask.to(DEV), n_split=n_split)
    return out.cpu().double(), ref.attention(q, *rows, n - q.shape[1], mask)


def close(out, y, dtype, more=0.0):
    off = float((out - y).norm() / y.norm())
    assert off <= 2e-5 + more + (2 ** -8 if dtype == BF16 else 0), off


@pytest.mark.parametrize("gap", [10, 12, 14, 17, 18, 30])
@pytest.mark.parametrize("n", [16, 48, 64, 70, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_small_probabilities_beside_a_row_that_takes_all_but_has_no_value(gap, n, dtype):
    """An attention sink: one row's score is `gap` above the others and its v is 0, so the result is what rows of e^-gap each say."""
    d, block = 64, 16
    k, v, q = rnd(1, n, 1, d, seed=n, scale=0.2), rnd(1, n, 1, d, seed=n + 1), torch.zeros(1, 1, 1, d)
    q[..., 0] = 8.0
    k[..., 0] = 0
    k[0, 0, 0, 0], v[0, 0] = float(gap), 0.0
    k[0, 1:16] = 0                                # (they share the first row's scale)
    out, y = attend(k, v, q, block, dtype)
    close(out, y, dtype)


@pytest.mark.parametrize("block,n", [(16, 64), (16, 100), (32, 64), (64, 130)])
@pytest.mark.parametrize("large", [1e2, 1e4, 1e6])
@pytest.mark.parametrize("gap", [0, 12, 40])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_block_of_large_values_with_little_or_no_weight(block, n, large, gap, dtype):
    """The rows of one block have `large` times the others' values, at e^-gap of their weight: where that is next to nothing the result is
    what the others say, to their own precision."""
    d, H = 64, 2
    k, v, q = rnd(2, n, H, d, seed=n, scale=0.2), rnd(2, n, H, d, seed=n + 1), torch.zeros(2, 1, 2 * H, d)
    q[..., 0] = 8.0
    k[..., 0] = 0
    first = 0 if n < 2 * block else block
    k[:, first:first + block, :, 0] = -float(gap)
    v[:, first:first + block] *= large
    out, y = attend(k, v, q, block, dtype)
    close(out, y, dtype)


@pytest.mark.parametrize("outlier", [20.0, 200.0, 2e4, 1e6])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_queries_with_an_outlier_that_meets_no_key(outlier, d, dtype):
    """One channel of q is far larger than the rest, and the keys have nothing there: the scores are what the rest says."""
    n, H = 150, 2
    k, v, q = rnd(1, n, H, d, seed=d), rnd(1, n, H, d, seed=d + 1), rnd(1, 2, H, d, seed=d + 2, scale=2.0)
    k[..., d // 2 + 3] = 0
    q[..., d // 2 + 3] = 2.0 * outlier
    out, y = attend(k, v, q, 16, dtype)
    close(out, y, dtype)


@pytest.mark.parametrize("d,block", [(32, 64), (64, 32), (128, 16)])
@pytest.mark.parametrize("q_scale", [1e-3, 1.0, 8.0, 40.0])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_flat_and_peaked(d, block, q_scale, dtype):
    """Up to scores of 40 times a normal number: a step of fp32 at the sum of magnitudes comes to the 2e-5."""
    n = 330
    k, v, q = rnd(2, n, 2, d, seed=d), rnd(2, n, 2, d, seed=d + 1), rnd(2, 1, 4, d, seed=d + 2, scale=q_scale)
    out, y = attend(k, v, q, block, dtype)
    size = float((q.abs().double()[:, 0, :, None] * k.abs().double().transpose(1, 2).repeat_interleave(2, 1)).sum(-1).max()) / math.sqrt(d)
    close(out, y, dtype, 2 * 2 ** -24 * size)


@pytest.mark.parametrize("n_split", [1, 3, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_that_differ_from_block_to_block(n_split, dtype):
    """Every block has its own size, over twelve orders of magnitude in v and two in k; some rows masked."""
    B, n, H, d, block = 2, 530, 2, 128, 32
    k, v, q = rnd(B, n, H, d, seed=1), rnd(B, n, H, d, seed=2), rnd(B, 1, 4, d, seed=3)
    size = torch.arange(n) // block
    v *= (10.0 ** (size * 7 % 13 - 6).double()).float()[None, :, None, None]
    k *= (10.0 ** (size * 5 % 3 - 1).double()).float()[None, :, None, None]
    mask = (torch.rand(B, n, generator=torch.Generator().manual_seed(4)) < 0.8).to(torch.uint8)
    out, y = attend(k, v, q, block, dtype, mask, n_split)
    top = float((q.abs().double()[:, 0, :, None] * k.abs().double().transpose(1, 2).repeat_interleave(2, 1)).sum(-1).max()) / math.sqrt(d)
    close(out, y, dtype, 2 * 2 ** -24 * top)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e20, 1e30, 1e37])
def test_queries_of_any_size(size, dtype):
    """q of any size against keys of the other: the scores are ordinary, and nothing on the way to them leaves fp32."""
    n, d = 90, 64
    k, v, q = rnd(1, n, 2, d, seed=6) / size, rnd(1, n, 2, d, seed=7), rnd(1, 1, 2, d, seed=8) * size
    q, k = q.clamp(-3e38, 3e38), k.clamp(-3e38, 3e38)
    out, y = attend(k[:, :80], v[:, :80], q, 16, dtype)      # (no open block)
    close(out, y, dtype)
