"""8-bit serving without a GPU: what the entry points refuse (arguments are checked before anything is launched), the cache's shapes, and
the oracle's own definitions."""
import ctypes

import pytest
import torch

from block_transformer_amd import _lib, ops
from block_transformer_amd._lib import BtError
from block_transformer_amd.runtime import KV8Cache
from oracle import q8_ref as ref

P = 0x1000      # a pointer that is never followed


def refused(rc, text, status=-1):
    assert rc == status, rc
    assert text.encode() in _lib.lib().bt_last_error(), _lib.lib().bt_last_error()


def test_quant_rows_refusals():
    f = _lib.lib().bt_quant_rows
    ok = dict(dtype=1, M=4, K=100, x=P, ldx=100, ln_w=None, ln_b=None, eps=1e-5, codes=P, ldc=112, scales=P, stream=None)

    def call(**kw):
        return f(*dict(ok, **kw).values())

    refused(call(dtype=2), "dtype")
    refused(call(K=0), "shape")
    refused(call(M=-1), "shape")
    refused(call(x=None), "null")
    refused(call(scales=None), "null")
    refused(call(ln_w=P), "ln_w and ln_b")
    refused(call(ldx=99), "row stride")
    refused(call(ldc=100), "round_up")
    refused(call(ldc=120), "round_up")
    refused(call(codes=P + 8), "round_up")
    assert call(M=0) == 0


def test_linear_q8_refusals():
    f = _lib.lib().bt_linear_q8
    ok = dict(dtype=1, M=4, N=8, K=128, A=P, lda=128, a_scale=P, W=P, ldw=128, w_scale=P, bias=None, residual=None, ldr=0, out=P, ldo=8, act=0,
              scratch=None, scratch_bytes=0, stream=None)

    def call(**kw):
        return f(*dict(ok, **kw).values())

    refused(call(dtype=3), "dtype")
    refused(call(N=0), "shape")
    refused(call(K=120), "multiple of 16")
    refused(call(K=131072, lda=131072, ldw=131072), "multiple of 16 up to 131056")
    refused(call(w_scale=None), "null")
    refused(call(lda=136), "16-byte granular")
    refused(call(ldw=112), "16-byte granular")
    refused(call(A=P + 4), "16-byte granular")
    refused(call(ldo=7), "row stride")
    refused(call(residual=P, ldr=7), "row stride")
    refused(call(ldo=1 << 26), "too large")
    refused(call(act=2), "act")
    refused(call(scratch=P + 8, scratch_bytes=64), "scratch")
    assert call(M=0) == 0
    assert _lib.lib().bt_linear_q8_scratch_bytes(1, 1, 16) >= 0


def cache(**kw):
    c = _lib.bt_kv8_cache(16, 2, 64, 3, 64, P, P, P, P, P, P)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


ROWS = _lib.bt_kv8_rows(P, 1024, 128, 64)
CACHE_REFUSALS = [(dict(struct_size=8), "struct_size"), (dict(block=48), "block"), (dict(head_dim=96), "head_dim"), (dict(n_max=72), "n_max"),
                  (dict(n_max=0), "n_max"), (dict(kv_heads=0), "kv_heads"), (dict(k_scale=None), "null"), (dict(v_codes=P + 4), "aligned")]


def test_append_refusals():
    f = _lib.lib().bt_kv8_append
    ok = dict(dtype=1, cache=cache(), q_len=1, heads=2, q=ROWS, q_out=ROWS, k=ROWS, v=ROWS, pos0_dev=None, pos0_host=0, pos_table=None, rot=16,
              cos=P, sin=P, max_pos=64, stream=None)

    def call(**kw):
        return f(*dict(ok, **kw).values())

    for kw, text in CACHE_REFUSALS:
        refused(call(cache=cache(**kw)), text)
    refused(call(dtype=5), "dtype")
    refused(call(cache=None), "null cache")
    refused(call(q_len=0), "q_len")
    refused(call(rot=15), "rotary")
    refused(call(rot=66), "rotary")
    refused(call(cos=None), "tables")
    refused(call(rot=0), "nothing to rotate")
    refused(call(q_out=None), "q_out")
    refused(call(heads=0), "heads")
    refused(call(k=None), "null k")
    refused(call(v=_lib.bt_kv8_rows(P, 1024, 130, 64)), "v must be 16-byte")
    refused(call(pos0_host=64), "overflow")
    refused(call(pos0_host=-1), "overflow")
    refused(call(pos0_host=60, q_len=5), "overflow")
    refused(call(pos0_host=20, max_pos=20), "beyond the tables")
    assert call(cache=cache(batch=0)) == 0


def test_read_refusals():
    f = _lib.lib().bt_kv8_read
    for kw, text in CACHE_REFUSALS:
        refused(f(1, cache(**kw), 10, 0, 1, P, P, None), text)
    for n, first, count in ((65, 0, 1), (10, -1, 1), (10, 4, 7), (10, 0, -1), (-1, 0, 0)):
        refused(f(1, cache(), n, first, count, P, P, None), "range")
    refused(f(1, cache(), 10, 0, 1, P + 2, P, None), "aligned")
    assert f(1, cache(), 10, 10, 0, P, P, None) == 0 and f(1, cache(), 10, 0, 5, None, None, None) == 0


def test_attention_refusals():
    f = _lib.lib().bt_attention_kv8
    ok = dict(dtype=1, cache=cache(), q_len=1, heads=4, q=ROWS, pos0_dev=None, pos0_host=10, mask=None, mask_ld=0, out=P, ldo=256, n_split=1,
              ws=None, ws_bytes=0, stream=None)

    def call(**kw):
        return f(*dict(ok, **kw).values())

    for kw, text in CACHE_REFUSALS:
        refused(call(cache=cache(**kw)), text)
    refused(call(q_len=-1), "q_len")
    refused(call(heads=5), "share")
    refused(call(q=_lib.bt_kv8_rows(P + 2, 0, 0, 0)), "q must be 16-byte")
    refused(call(out=None), "output")
    refused(call(ldo=248), "output")
    refused(call(pos0_host=64), "overflow")
    refused(call(mask=P, mask_ld=10), "mask")
    refused(call(mask=P, mask_ld=63, pos0_dev=P), "mask")
    refused(call(n_split=0), "n_split")
    refused(call(n_split=2), "workspace", -3)
    need = _lib.lib().bt_attention_kv8_workspace_bytes(3, 1, 4, 64, 2)
    refused(call(n_split=2, ws=P, ws_bytes=need - 1), "workspace", -3)
    refused(call(n_split=2, ws=P + 4, ws_bytes=need), "workspace", -3)
    assert call(cache=cache(batch=0)) == 0


def test_split_count_depends_on_its_arguments_alone_and_is_bounded():
    f = _lib.lib().bt_attention_kv8_split_count
    for batch in (1, 2, 7, 64, 1000):
        for n in (1, 16, 64, 100, 1000, 32773, 1 << 20):
            s = f(batch, 4, 2, 1, n)
            assert s == f(batch, 4, 2, 1, n) and 1 <= s <= max(1, -(-n // 64))


def test_tensor_level_refusals():
    """Checked before the library is called; CPU tensors are refused as everywhere."""
    x, w = torch.zeros(3, 40), (torch.zeros(8, 48, dtype=torch.int8), torch.zeros(8))
    with pytest.raises(BtError, match="GPU memory"):
        ops.quantize_rows(x)
    with pytest.raises(BtError, match="ln_w and ln_b"):
        ops.quantize_rows(x, torch.ones(40))
    with pytest.raises(BtError, match="LayerNorm weight"):
        ops.quantize_rows(x, torch.ones(41), torch.ones(41))
    with pytest.raises(BtError, match="empty"):
        ops.quantize_rows(x[:, :0])
    with pytest.raises(BtError, match="unit inner stride"):
        ops.quantize_rows(x.T)
    codes = (torch.zeros(3, 48, dtype=torch.int8), torch.zeros(3))
    with pytest.raises(BtError, match="which dtype"):
        ops.linear_q8(codes, w)
    with pytest.raises(BtError, match="not supported"):
        ops.linear_q8(codes, w, dtype=torch.float16)
    with pytest.raises(BtError, match="columns"):
        ops.linear_q8(torch.zeros(3, 49), w)
    with pytest.raises(BtError, match="columns"):
        ops.linear_q8((torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)), w, dtype=torch.float32)
    with pytest.raises(BtError, match="int8 codes"):
        ops.linear_q8((torch.zeros(3, 48), torch.zeros(3)), w, dtype=torch.float32)
    with pytest.raises(BtError, match="one contiguous scale"):
        ops.linear_q8((codes[0], torch.zeros(2)), w, dtype=torch.float32)
    with pytest.raises(BtError, match="bias"):
        ops.linear_q8(codes, w, torch.zeros(7))
    with pytest.raises(BtError, match="bias"):
        ops.linear_q8(codes, w, torch.zeros(8), dtype=torch.bfloat16)
    with pytest.raises(BtError, match="residual"):
        ops.linear_q8(codes, w, residual=torch.zeros(3, 9), dtype=torch.float32)
    with pytest.raises(BtError, match="activation"):
        ops.linear_q8(codes, w, act="relu", dtype=torch.float32)
    with pytest.raises(BtError, match="GPU memory"):
        ops.linear_q8(codes, w, dtype=torch.float32)


def test_cache_level_refusals():
    c = KV8Cache(2, 3, 4, 70, 32, torch.bfloat16, "cpu", block=32)
    assert len(c) == 2 and c.n_max == 96 and c.block == 32
    assert [tuple(t.shape) for t in c[1]] == [(3, 4, 96, 32), (3, 4, 3, 32, 32), (3, 4, 3), (3, 4, 3), (3, 4, 32, 32), (3, 4, 32, 32)]
    with pytest.raises(BtError, match="block"):
        KV8Cache(1, 1, 1, 16, 32, torch.bfloat16, "cpu", block=24)
    with pytest.raises(BtError, match="not supported"):
        KV8Cache(1, 1, 1, 16, 32, torch.float16, "cpu")
    kv, q = c[0], torch.zeros(3, 1, 4, 32, dtype=torch.bfloat16)
    with pytest.raises(BtError, match="GPU memory"):
        ops.attention_kv8(q, kv, 0)
    with pytest.raises(BtError, match="k_scale"):
        ops.attention_kv8(q, kv[:2] + (kv[2][:, :, :2],) + kv[3:], 0)
    with pytest.raises(BtError, match="v_tail"):
        ops.attention_kv8(q, kv[:5] + (kv[5].float(),), 0)
    with pytest.raises(BtError, match="k_codes"):
        ops.attention_kv8(q, (kv[0].transpose(0, 1).contiguous().transpose(0, 1),) + kv[1:], 0)
    with pytest.raises(BtError, match="q must be"):
        ops.attention_kv8(q.float(), kv, 0)
    with pytest.raises(BtError, match="q must be"):
        ops.attention_kv8(q[:2], kv, 0)
    with pytest.raises(BtError, match="cannot share"):
        ops.attention_kv8(q[:, :, :3], kv, 0)
    with pytest.raises(BtError, match="unit inner stride"):
        ops.attention_kv8(torch.zeros(3, 1, 32, 4, dtype=torch.bfloat16).transpose(2, 3), kv, 0)
    with pytest.raises(BtError, match="mask must be"):
        ops.attention_kv8(q, kv, 0, mask=torch.ones(3, 8))
    with pytest.raises(BtError, match="too short"):
        ops.attention_kv8(q, kv, 8, mask=torch.ones(3, 8, dtype=torch.uint8))
    with pytest.raises(BtError, match="one int32"):
        ops.attention_kv8(q, kv, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(BtError, match="4 heads"):
        ops.kv8_append(kv, None, q[:, :, :2], q[:, :, :2], 0)
    with pytest.raises(BtError, match="k must be"):
        ops.kv8_append(kv, None, q[..., :16], q, 0)
    with pytest.raises(BtError, match="no rows"):
        ops.kv8_append(kv, None, q[:, :0], q[:, :0], 0)
    with pytest.raises(BtError, match="range|rows"):
        ops.kv8_read(kv, 97)
    with pytest.raises(BtError, match="range|rows"):
        ops.kv8_read(kv, 10, first=5, count=6)


def test_oracle_codes():
    """Half steps go to the even code, a quotient beside one to its own side; blocks ignore what is not finite."""
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5]])
    c, s = ref.quantize_rows(x)
    assert s.item() == 1.0 and c.tolist() == [[127, 0, 2, 2, 0, -2, 126]]
    c, s = ref.block_values(torch.tensor([[254.0, float("inf")], [float("nan"), -3.0]]), torch.float32)
    assert float(s) == 2.0 and c.tolist() == [[127, 127], [0, -2]]


def test_oracle_attention_is_softmax_attention():
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(2, 3, 4, 8, generator=g), torch.randn(2, 2, 9, 8, generator=g).double(), torch.randn(2, 2, 9, 8, generator=g).double()
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(1, 2), k.repeat_interleave(2, 1), v.repeat_interleave(2, 1),
                                                           attn_mask=torch.arange(9) <= torch.arange(6, 9)[:, None])
    assert (ref.attention(q, k, v, 6) - want.transpose(1, 2)).abs().max() < 1e-12


def test_structs_match_the_header():
    assert ctypes.sizeof(_lib.bt_kv8_cache) == 80 and ctypes.sizeof(_lib.bt_kv8_rows) == 32
