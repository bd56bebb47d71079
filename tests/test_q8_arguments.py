"""Calls of the 8-bit operators that are refused, and that nothing else depends on: without a GPU."""
import importlib.util

import pytest
import torch

from block_transformer_amd import _lib, ops
from block_transformer_amd._lib import BtError
from block_transformer_amd.runtime import KV8Cache


def weight(columns, rows=8):
    w = torch.zeros(rows, (columns + 15) // 16 * 16, dtype=torch.int8), torch.zeros(rows)
    w[0].columns = columns                # as quantize_rows leaves it
    return w


def test_linear_q8_of_another_number_of_columns():
    """515 and 520 columns both take 528 codes: their product would mean nothing."""
    with pytest.raises(BtError, match="x has 515 columns, the weight 520"):
        ops.linear_q8(torch.zeros(3, 515), weight(520))
    with pytest.raises(BtError, match="x has 515 columns, the weight 520"):
        ops.linear_q8(weight(515, 3), weight(520), dtype=torch.float32)
    with pytest.raises(BtError, match="GPU memory"):      # (refused for the device alone)
        ops.linear_q8(torch.zeros(3, 520), weight(520))
    with pytest.raises(BtError, match="GPU memory"):
        ops.linear_q8(weight(520, 3), weight(520), dtype=torch.float32)
    with pytest.raises(BtError, match="GPU memory"):      # codes that do not say
        ops.linear_q8(torch.zeros(3, 515), (torch.zeros(8, 528, dtype=torch.int8), torch.zeros(8)))


def test_workspaces_whose_elements_share_memory():
    """An expanded tensor has more elements than memory: a kernel that took it by its size would write behind it."""
    thin = torch.zeros(1, dtype=torch.uint8).expand(1 << 20)
    with pytest.raises(BtError, match="scratch must be contiguous"):
        ops.linear_q8(weight(64, 3), weight(64), dtype=torch.float32, scratch=thin)
    kv, q = KV8Cache(1, 3, 4, 64, 32, torch.bfloat16, "cpu")[0], torch.zeros(3, 1, 4, 32, dtype=torch.bfloat16)
    for ws in (thin, torch.zeros(1 << 20, dtype=torch.uint8)[::2]):
        with pytest.raises(BtError, match="ws must be contiguous"):
            ops.attention_kv8(q, kv, 0, n_split=2, ws=ws)


def test_queries_that_are_written_over_each_other():
    kv, x = KV8Cache(1, 3, 4, 64, 32, torch.bfloat16, "cpu")[0], torch.zeros(3, 5, 4, 32, dtype=torch.bfloat16)
    rope = ops.rope_tables(64, 16, 10000.0, "cpu")
    wide = torch.zeros(3 * 5 * 4 * 32 + 64, dtype=torch.bfloat16)
    for q_out in (x[:1].expand(3, 5, 4, 32), x[:, :, :1].expand(3, 5, 4, 32), wide.as_strided((3, 5, 4, 32), (640, 128, 16, 1)),
                  wide.as_strided((3, 5, 4, 32), (512, 128, 32, 1))):
        with pytest.raises(BtError, match="q_out overlaps itself"):
            ops.kv8_append(kv, x, x, x, 0, rope=rope, q_out=q_out)
    fused = torch.zeros(3, 5, 12, 32, dtype=torch.bfloat16)
    for q_out in (x, fused[:, :, 4:8], fused.transpose(1, 2)[:, :4].transpose(1, 2), torch.zeros(5, 3, 4, 32, dtype=torch.bfloat16).transpose(0, 1)):
        with pytest.raises(BtError, match="GPU memory"):      # (refused for the device alone)
            ops.kv8_append(kv, x, x, x, 0, rope=rope, q_out=q_out)


def test_one_mask_row_for_all_sequences():
    """mask_ld = 0 is a row that all share; what lies between is too short.  (The last argument that is checked refuses the call.)"""
    p = 0x1000      # a pointer that is never followed
    cache = _lib.bt_kv8_cache(16, 2, 64, 3, 64, p, p, p, p, p, p)
    for ld, text in ((0, b"n_split"), (10, b"mask row too short"), (11, b"n_split")):
        rc = _lib.lib().bt_attention_kv8(1, cache, 1, 4, _lib.bt_kv8_rows(p, 1024, 128, 64), None, 10, p, ld, p, 256, 0, None, 0, None)
        assert rc == -1 and text in _lib.lib().bt_last_error()


def test_the_module_is_imported_on_a_torch_without_gpu_support(monkeypatch):
    """Such a build has no torch._C._cuda_*; calls are refused as on any machine without a GPU."""
    for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("block_transformer_amd.ops_again", ops.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    with pytest.raises(BtError, match="GPU memory"):
        again.quantize_rows(torch.zeros(3, 40))


def test_launches_of_more_threads_than_32_bits_count():
    """Such a grid would be cut or fail; the entry points say so.  (No pointer is followed.)"""
    p, lib = 0x1000, _lib.lib()

    def refused(rc, text):
        assert rc == -1 and text in lib.bt_last_error(), (rc, lib.bt_last_error())

    refused(lib.bt_quant_rows(1, 1 << 26, 16, p, 16, None, None, 1e-5, p, 16, p, None), b"too many")
    refused(lib.bt_quant_rows(1, 1 << 24, 8192, p, 8192, None, None, 1e-5, p, 8192, p, None), b"too many")
    refused(lib.bt_linear_q8(1, 1 << 21, 2, 16, p, 16, p, p, 1 << 23, p, None, None, 0, p, 2, 0, None, 0, None), b"too many")
    rows = _lib.bt_kv8_rows(p, 32, 32, 32)
    cache = lambda batch, n_max: _lib.bt_kv8_cache(16, 1, 32, batch, n_max, p, p, p, p, p, p)  # noqa: E731
    refused(lib.bt_kv8_append(1, cache(1 << 25, 16), 1, 1, None, None, rows, rows, None, 0, None, 0, None, None, 0, None), b"too many")
    refused(lib.bt_kv8_append(1, cache(1 << 22, 256), 200, 64, rows, rows, rows, rows, None, 0, None, 2, p, p, 256, None), b"too many")
    refused(lib.bt_kv8_read(1, cache(1 << 20, 1024), 1024, 0, 1024, p, p, None), b"too large")
    refused(lib.bt_attention_kv8(1, cache(1 << 26, 16), 1, 1, rows, None, 0, None, 0, p, 32, 1, None, 0, None), b"too large")
    refused(lib.bt_attention_kv8(1, cache(1 << 24, 16), 1, 1, rows, None, 0, None, 0, p, 32, 2, p, 1 << 60, None), b"too large")


def test_sizes_whose_products_leave_64_bits():
    """They would pass for small ones.  (No pointer is followed.)"""
    p, lib = 0x1000, _lib.lib()

    def refused(rc, text):
        assert rc in (-1, -3) and text in lib.bt_last_error(), (rc, lib.bt_last_error())

    rows = _lib.bt_kv8_rows(p, 32, 32, 32)
    cache = lambda batch, heads, n_max: _lib.bt_kv8_cache(16, heads, 32, batch, n_max, p, p, p, p, p, p)  # noqa: E731
    refused(lib.bt_kv8_read(1, cache(1, 1, 64), 10, 1 << 62, 1 << 62, p, p, None), b"out of range")
    refused(lib.bt_kv8_read(1, cache(1 << 62, 4, 64), 10, 0, 1, p, p, None), b"bad batch")
    refused(lib.bt_kv8_append(1, cache(1, 1, 64), 1 << 30, 1 << 30, rows, rows, rows, rows, p, 0, None, 2, p, p, 64, None), b"too many")
    refused(lib.bt_kv8_append(1, cache(1 << 20, 1, 64), 1 << 16, 1 << 28, rows, rows, rows, rows, p, 0, None, 2, p, p, 64, None), b"too many")
    refused(lib.bt_attention_kv8(1, cache(1 << 20, 1, 1 << 20), 1 << 19, 1 << 10, rows, None, 0, None, 0, p, 1 << 15, 1 << 30, p, 1 << 62, None),
            b"too large")
