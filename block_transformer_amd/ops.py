"""Tensor-level wrappers over the C-ABI single ops (one call = one or two HIP kernels on torch's current stream).

torch is used for device memory and streams only; no arithmetic runs in ATen here."""
from __future__ import annotations

import contextlib
import ctypes
import struct
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import check, current_stream, dtype_code, lib, ptr


def _rows(t: torch.Tensor):
    if t.dim() < 2 or t.stride(-1) != 1:
        raise _lib.BtError("expected a row-major tensor with unit inner stride")
    t2 = t.reshape(-1, t.shape[-1]) if t.is_contiguous() else t
    if t2.dim() != 2:
        raise _lib.BtError("non-contiguous input must be 2-D")
    return t2, t2.stride(0)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
           residual: Optional[torch.Tensor] = None, act: str = "none", out: Optional[torch.Tensor] = None,
           scratch: Optional[torch.Tensor] = None):
    """out = act(x @ weight.T + bias) + residual   (weight in nn.Linear layout [out_features, in_features]).
    ``scratch`` (any dtype, >= 2*M*N*4 bytes) lets skinny problems use the split-K weight-streaming path."""
    x2, lda = _rows(x)
    M, K = x2.shape
    if weight.dim() == 3:  # Conv1d(kernel_size=1) weight [out, in, 1]
        weight = weight[:, :, 0]
    N = weight.shape[0]
    if weight.shape[1] != K or not weight.is_contiguous():
        raise _lib.BtError(f"weight must be contiguous [N, K={K}], got {tuple(weight.shape)}")
    if out is None:
        out = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    o2, ldo = _rows(out)
    ldr = 0
    if residual is not None:
        r2, ldr = _rows(residual)
    a = _lib.BT_ACT_GELU if act == "gelu" else _lib.BT_ACT_NONE
    if scratch is None:
        check(lib().bt_linear(dtype_code(x.dtype), M, N, K, ptr(x2), lda, ptr(weight), ptr(bias), ptr(residual), ldr,
                              ptr(o2), ldo, a, current_stream()), "bt_linear")
    else:
        check(lib().bt_linear_ws(dtype_code(x.dtype), M, N, K, ptr(x2), lda, ptr(weight), ptr(bias), ptr(residual), ldr,
                                 ptr(o2), ldo, a, ptr(scratch), scratch.numel() * scratch.element_size(),
                                 current_stream()), "bt_linear_ws")
    return out


def stream_k_scratch(device) -> torch.Tensor:
    """Scratch for the stream-K GEMM path of bt_linear_ws / bt_qkv_rope_append / bt_linear2_ws (hand-off slabs + flag words; the
    entry points clear the flag words themselves, the sticky time-out word behind them is zeroed here and read by
    ``stream_k_check``)."""
    scratch = torch.empty(int(lib().bt_stream_k_scratch_bytes()), dtype=torch.uint8, device=device)
    check(lib().bt_stream_k_reset(ptr(scratch), scratch.numel(), current_stream()), "bt_stream_k_reset")
    return scratch


def stream_k_check(scratch: torch.Tensor) -> None:
    """Raise if a stream-K launch on ``scratch`` flagged a hand-off time-out since the last reset (synchronises)."""
    err = torch.zeros(1, dtype=torch.int32, device=scratch.device)
    check(lib().bt_stream_k_status(ptr(scratch), scratch.numel() * scratch.element_size(), ptr(err), current_stream()),
          "bt_stream_k_status")
    if int(err.item()) & _lib.BT_DEV_ERR_HANDOFF_TIMEOUT:
        check(lib().bt_stream_k_reset(ptr(scratch), scratch.numel() * scratch.element_size(), current_stream()), "bt_stream_k_reset")
        raise _lib.BtError("stream-K GEMM hand-off timed out: the results of the launches on this scratch are incomplete")


def linear2(x1: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, x2: torch.Tensor, w2: torch.Tensor, b2: torch.Tensor,
            residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, scratch: Optional[torch.Tensor] = None):
    """out = x1 @ w1.T + b1 + x2 @ w2.T + b2 + residual in one call (attention.dense + mlp.dense_4h_to_h of a parallel-residual
    layer); with ``scratch`` (stream_k_scratch) stacks above 256 rows run as ONE stream-K GEMM over K1 + K2."""
    a1, ld1 = _rows(x1)
    a2, ld2 = _rows(x2)
    M, K1 = a1.shape
    K2 = a2.shape[1]
    N = w1.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=x1.dtype, device=x1.device)
    o2, ldo = _rows(out)
    ldr = 0
    if residual is not None:
        _, ldr = _rows(residual)
    if scratch is None:
        check(lib().bt_linear2(dtype_code(x1.dtype), M, N, K1, ptr(a1), ld1, ptr(w1), ptr(b1), K2, ptr(a2), ld2, ptr(w2), ptr(b2),
                               ptr(residual), ldr, ptr(o2), ldo, current_stream()), "bt_linear2")
    else:
        check(lib().bt_linear2_ws(dtype_code(x1.dtype), M, N, K1, ptr(a1), ld1, ptr(w1), ptr(b1), K2, ptr(a2), ld2, ptr(w2), ptr(b2),
                                  ptr(residual), ldr, ptr(o2), ldo, ptr(scratch), scratch.numel() * scratch.element_size(),
                                  current_stream()), "bt_linear2_ws")
    return out


def layernorm(x, w1, b1, eps: float, w2=None, b2=None):
    """LN(x)*w1+b1 (and LN(x)*w2+b2 when w2 is given) in one pass."""
    x2, ldx = _rows(x)
    M, H = x2.shape
    o1 = torch.empty_like(x2 if x2.is_contiguous() else x2.contiguous())
    o2 = torch.empty_like(o1) if w2 is not None else None
    check(lib().bt_layernorm(dtype_code(x.dtype), M, H, ptr(x2), ldx, ptr(w1), ptr(b1), ptr(o1), H, ptr(w2), ptr(b2),
                             ptr(o2), H, float(eps), current_stream()), "bt_layernorm")
    o1 = o1.view(x.shape) if x.is_contiguous() else o1
    if o2 is None:
        return o1
    return o1, (o2.view(x.shape) if x.is_contiguous() else o2)


def embed_rows(ids: torch.Tensor, table: torch.Tensor, out: Optional[torch.Tensor] = None,
               row_zero: Optional[torch.Tensor] = None, rows_per_seq: int = 1):
    """out[r] = table[ids[r]] for the flattened ids (int64; contiguous, or 1-D with any stride — no copy is made)."""
    if ids.dtype != torch.int64:
        raise _lib.BtError("ids must be int64")
    if ids.dim() == 1:
        ids_stride = ids.stride(0) if ids.numel() > 1 else 1
    elif ids.is_contiguous():
        ids_stride = 1
    else:
        raise _lib.BtError("ids must be contiguous or 1-D strided")
    rows = ids.numel()
    vocab, width = table.shape
    if out is None:
        out = torch.empty(ids.shape + (width,), dtype=table.dtype, device=table.device)
    check(lib().bt_embed_rows(dtype_code(table.dtype), rows, width, ptr(ids), ids_stride, vocab, ptr(table), ptr(out),
                              width, ptr(row_zero), rows_per_seq, current_stream()), "bt_embed_rows")
    return out


def argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None):
    l2, ld = _rows(logits)
    M, V = l2.shape
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=logits.device)
    check(lib().bt_argmax(dtype_code(logits.dtype), M, V, ptr(l2), ld, ptr(out), out.stride(0) if out.dim() else 1,
                          current_stream()), "bt_argmax")
    return out


def logits_argmax(hid: torch.Tensor, weight: torch.Tensor, logits: torch.Tensor, store_logits: bool = True,
                  out: Optional[torch.Tensor] = None, ws: Optional[torch.Tensor] = None):
    """ids = argmax(hid @ weight.T) (greedy token step): the logits GEMM with the argmax in its epilogue where the persistent MFMA
    kernel applies (``logits`` is then only written when ``store_logits``), bt_linear + bt_argmax through ``logits`` otherwise."""
    h2, ldh = _rows(hid)
    M, K = h2.shape
    V = weight.shape[0]
    l2, ldl = _rows(logits)
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=hid.device)
    if ws is None:
        ws = torch.empty(max(int(lib().bt_logits_argmax_workspace_bytes(M, V)), 16), dtype=torch.uint8, device=hid.device)
    check(lib().bt_logits_argmax(dtype_code(hid.dtype), M, V, K, ptr(h2), ldh, ptr(weight), ptr(l2), ldl, int(bool(store_logits)),
                                 ptr(out), out.stride(0) if out.dim() else 1, ptr(ws), ws.numel() * ws.element_size(),
                                 current_stream()), "bt_logits_argmax")
    return out


def topk_sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 50, seed: int = 0,
                step: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, row0: int = 0):
    l2, ld = _rows(logits)
    M, V = l2.shape
    if out is None:
        out = torch.empty(M, dtype=torch.int64, device=logits.device)
    check(lib().bt_topk_sample(dtype_code(logits.dtype), M, V, ptr(l2), ld, float(temperature), int(top_k), int(seed),
                               ptr(step), int(row0), ptr(out), out.stride(0), current_stream()), "bt_topk_sample")
    return out


def rope_tables(max_pos: int, rot: int, base: float, device) -> torch.Tensor:
    """fp32 [2, max_pos, rot/2] cos/sin tables, built on the host once (angle = pos * base^(-2j/rot))."""
    inv_freq = 1.0 / (base ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot))
    freqs = torch.outer(torch.arange(max(max_pos, 1), dtype=torch.float32), inv_freq)
    return torch.stack([freqs.cos(), freqs.sin()]).contiguous().to(device)


# ---- 8-bit serving ----------------------------------------------------------------------------------------------------------------
_HERE = contextlib.nullcontext()
# the current stream's handle and the current device without the Python objects around them: together 5 us of a call that takes 10
# (a torch built without GPU support has neither name: nothing can be launched there, but importing this module is no launch)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
# bt_kv8_cache as bytes: a third of the time that its fields take one by one
_cache_bytes = struct.Struct("=I3i2q6Q").pack
_CACHE_SIZE = ctypes.sizeof(_lib.bt_kv8_cache)
_CONTIGUOUS = torch.contiguous_format


def _on(index: int, *tensors):
    """A context in which device `index` is the current one; every tensor (None: left out) has to live there."""
    if index < 0:
        raise _lib.BtError("libbt_hip operates on GPU memory only; got a CPU tensor (move the model/inputs to 'cuda')")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise _lib.BtError(f"all tensors must be on cuda:{index}, got one on {t.device}")
    return _HERE if index == _device() else torch.cuda.device(index)


def _at(t: Optional[torch.Tensor]):
    """Device pointer of a tensor that `_on` has seen (None -> NULL)."""
    return None if t is None else t.data_ptr()


def _flat(t: torch.Tensor):
    """(rows, columns, row stride) of a tensor of rows: 2-D with any row stride, or contiguous."""
    shape = t.shape
    if len(shape) == 2:
        M, K = shape
        ld, one = t.stride()
        if one == 1 or K == 1:
            return M, K, ld if M > 1 else K      # (the stride of a single row says nothing)
    elif len(shape) > 2 and t.is_contiguous():
        K = shape[-1]
        return t.numel() // K if K else 0, K, K
    raise _lib.BtError("expected rows with unit inner stride: 2-D, or contiguous")


def _expect(t: torch.Tensor, what: str, shape, dtype) -> None:
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise _lib.BtError(f"{what} must be contiguous {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def _flat_memory(t: Optional[torch.Tensor], what: str) -> None:
    """A workspace's bytes are counted by its elements: they have to lie one behind the other."""
    if t is not None and not t.is_contiguous():
        raise _lib.BtError(f"{what} must be contiguous")


def quantize_rows(x: torch.Tensor, ln_w: Optional[torch.Tensor] = None, ln_b: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(codes, scales) of the rows of ``x`` [..., K] -- of LayerNorm(x; ln_w, ln_b, eps) if weights are given -- in 8-bit integers with one
    scale per row: codes int8 [..., round_up(K, 16)] (zero behind column K), scales float32 [...].  Activations and weights alike:
    ``quantize_rows(weight)`` has one scale per output channel.  A row with an infinity or NaN in it gets scale NaN.  ``codes.columns`` is K
(views of the codes do not have it)."""
    M, K, ldx = _flat(x)
    if K == 0:
        raise _lib.BtError("rows are empty")
    if (ln_w is None) != (ln_b is None):
        raise _lib.BtError("LayerNorm needs ln_w and ln_b")
    for w in (ln_w, ln_b):
        if w is not None:
            _expect(w, "LayerNorm weight", (K,), x.dtype)
    Kp = (K + 15) // 16 * 16
    code, index = dtype_code(x.dtype), x.get_device()
    with _on(index, ln_w, ln_b):
        lead = (M,) if x.dim() == 2 else x.shape[:-1]      # (a plain tuple makes the cheaper call)
        codes = x.new_empty(lead + (Kp,), dtype=torch.int8)
        scales = x.new_empty(lead, dtype=torch.float32)
        check(lib().bt_quant_rows(code, M, K, x.data_ptr(), ldx, _at(ln_w), _at(ln_b), eps, codes.data_ptr(), Kp, scales.data_ptr(),
                                  _raw_stream(index)), "bt_quant_rows")
    codes.columns = K
    return codes, scales


def linear_q8(x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], weight: Tuple[torch.Tensor, torch.Tensor],
              bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None, act: str = "none",
              out: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None, scratch: Optional[torch.Tensor] = None):
    """out = act(x @ weight.T + bias) + residual in 8-bit integers with scales per token and per output channel.  ``x``: rows in fp32 or
    bf16 (quantised here) or the (codes, scales) that ``quantize_rows`` made of them; ``weight``: ``quantize_rows`` of the nn.Linear
    weight [N, K]; both have to have the same K (of codes that do not say theirs -- ``codes.columns`` -- only round_up(K, 16) is compared).
    The sum over K is exact; ``dtype`` (default: that of x, bias, residual or out, whichever is a float tensor) is the
    type of bias, residual and result.  ``scratch`` (any dtype, >= bt_linear_q8_scratch_bytes) is allocated when it is needed and not
    given."""
    wc, ws = weight
    columns = getattr(wc, "columns", None)
    if isinstance(x, torch.Tensor):
        dtype = dtype or x.dtype
        if (x.shape[-1] + 15) // 16 * 16 != wc.shape[-1] or columns not in (None, x.shape[-1]):
            raise _lib.BtError(f"x has {x.shape[-1]} columns, the weight {columns or wc.shape[-1]}")
        x = quantize_rows(x)
    xc, xs = x
    if columns is not None and getattr(xc, "columns", columns) != columns:
        raise _lib.BtError(f"x has {xc.columns} columns, the weight {columns}")
    if dtype is None:
        dtype = next((t.dtype for t in (out, residual, bias) if t is not None), None)
        if dtype is None:
            raise _lib.BtError("quantised x without bias, residual or out: say which dtype the result has")
    code = dtype_code(dtype)
    if xc.dtype != torch.int8 or wc.dtype != torch.int8 or xs.dtype != torch.float32 or ws.dtype != torch.float32:
        raise _lib.BtError("quantised operands are (int8 codes, float32 scales)")
    M, K, lda = _flat(xc)
    if wc.dim() != 2:
        raise _lib.BtError("weight codes must be [N, K]")
    N, Kw, ldw = _flat(wc)
    if Kw != K:
        raise _lib.BtError(f"codes of x have {K} columns, those of the weight {Kw}")
    if xs.numel() != M or ws.numel() != N or not xs.is_contiguous() or not ws.is_contiguous():
        raise _lib.BtError("one contiguous scale per row of codes is needed")
    if act not in ("none", "gelu"):
        raise _lib.BtError(f"unknown activation {act!r}")
    if bias is not None:
        _expect(bias, "bias", (N,), dtype)
    shape = (M, N) if xc.dim() == 2 else xc.shape[:-1] + (N,)
    ldr = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype:
            raise _lib.BtError(f"residual must be {dtype} {tuple(shape)}")
        ldr = _flat(residual)[2]
    _flat_memory(scratch, "scratch")
    index = xc.get_device()
    with _on(index, xs, wc, ws, bias, residual, out, scratch):
        if out is None:
            out = xc.new_empty(shape, dtype=dtype)
            ldo = N
        elif out.shape != shape or out.dtype != dtype:
            raise _lib.BtError(f"out must be {dtype} {tuple(shape)}")
        else:
            ldo = _flat(out)[2]
        if scratch is None:
            need = lib().bt_linear_q8_scratch_bytes(M, N, K)
            if need:
                scratch = torch.empty(need, dtype=torch.uint8, device=xc.device)
        check(lib().bt_linear_q8(code, M, N, K, xc.data_ptr(), lda, xs.data_ptr(), wc.data_ptr(), ldw, ws.data_ptr(), _at(bias),
                                 _at(residual), ldr, out.data_ptr(), ldo,
                                 _lib.BT_ACT_GELU if act == "gelu" else _lib.BT_ACT_NONE, _at(scratch),
                                 0 if scratch is None else scratch.numel() * scratch.element_size(), _raw_stream(index)), "bt_linear_q8")
    return out


def _kv8(kv: Sequence[torch.Tensor]):
    """(bt_kv8_cache, dtype code, B, H, n_max, d, dtype) of one layer of an 8-bit cache: (k_codes, v_codes, k_scale, v_scale, k_tail,
    v_tail)."""
    kc, vc, ks, vs, kt, vt = kv
    codes, tail, dtype = kc.shape, kt.shape, kt.dtype
    if len(codes) != 4 or len(tail) != 4:
        raise _lib.BtError("a layer of an 8-bit cache is (k_codes, v_codes, k_scale, v_scale, k_tail, v_tail), see runtime.KV8Cache")
    B, H, n_max, d = codes
    block = tail[2]
    if block == 0 or n_max % block:
        raise _lib.BtError(f"{n_max} rows are not a whole number of blocks of {block}")
    blocks = n_max // block
    scales = (B, H, blocks)
    if not (kc.dtype is vc.dtype is torch.int8 and ks.dtype is vs.dtype is torch.float32 and vt.dtype is dtype and
            ks.shape == scales and vs.shape == scales and vc.shape == (B, H, blocks, d, block) and tail == (B, H, block, d) and
            vt.shape == (B, H, d, block) and kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and
            kt.is_contiguous() and vt.is_contiguous()):      # (all at once: 3 us less than one by one, which then says what is wrong)
        _expect(kc, "k_codes", (B, H, n_max, d), torch.int8)
        _expect(vc, "v_codes", (B, H, blocks, d, block), torch.int8)
        _expect(ks, "k_scale", scales, torch.float32)
        _expect(vs, "v_scale", scales, torch.float32)
        _expect(kt, "k_tail", (B, H, block, d), dtype)
        _expect(vt, "v_tail", (B, H, d, block), dtype)
    cache = _lib.bt_kv8_cache.from_buffer_copy(_cache_bytes(_CACHE_SIZE, block, H, d, B, n_max, kc.data_ptr(), vc.data_ptr(),
                                                            ks.data_ptr(), vs.data_ptr(), kt.data_ptr(), vt.data_ptr()))
    return cache, dtype_code(dtype), B, H, n_max, d, dtype


def _kv8_rows(t: torch.Tensor, what: str, batch: int, q_len: int, d: int, dtype):
    """(bt_kv8_rows, heads) of rows [batch, q_len, heads, d] with any outer strides."""
    shape = t.shape
    if len(shape) != 4 or shape[0] != batch or shape[1] != q_len or shape[3] != d or t.dtype is not dtype:
        raise _lib.BtError(f"{what} must be {dtype} [{batch}, {q_len}, heads, {d}], got {t.dtype} {tuple(shape)}")
    sb, st, sh, one = t.stride()
    if one != 1:
        raise _lib.BtError(f"{what} must have unit inner stride")
    heads = shape[2]
    # (the stride of a single row says nothing)
    return _lib.bt_kv8_rows(t.data_ptr(), sb if batch > 1 else 0, st if q_len > 1 else 0, sh if heads > 1 else 0), heads


def _apart(t: torch.Tensor, what: str) -> None:
    """No two elements of rows [batch, q_len, heads, d] that are written may share a place."""
    extent = t.shape[3]
    for stride, n in sorted((t.stride(i), t.shape[i]) for i in range(3) if t.shape[i] > 1):
        if stride < extent:
            raise _lib.BtError(f"{what} overlaps itself: strides {t.stride()} of {tuple(t.shape)}")
        extent += stride * (n - 1)


def _pos0(pos0):
    if isinstance(pos0, torch.Tensor):
        if pos0.dtype != torch.int32 or pos0.numel() != 1:
            raise _lib.BtError("a device-side pos0 is one int32")
        return pos0.data_ptr(), 0
    return None, int(pos0)


def kv8_append(kv: Sequence[torch.Tensor], q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, pos0,
               rope: Optional[torch.Tensor] = None, pos_table: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None):
    """Append rows ``k``, ``v`` [B, q_len, kv_heads, d] (any outer strides: views of a fused projection) at row ``pos0`` (an int, or one
    int32 on the device) of one layer of an 8-bit cache (``runtime.KV8Cache``), rotating ``k`` and ``q`` [B, q_len, heads, d] by ``rope``
    (``rope_tables``) at positions pos0 + t or ``pos_table[pos0 + t]``.  Returns the rotated q -- in ``q_out`` (which may be q), new
    memory otherwise; q itself without ``rope`` or with one of no columns.  Blocks that fill up are quantised in the same call.
    (A device-side pos0 below 0 does nothing at all; rows at the cache's end and behind it are dropped.)"""
    cache, code, B, H, n_max, d, dtype = _kv8(kv)
    q_len = k.shape[1] if k.dim() == 4 else 0
    kr, k_heads = _kv8_rows(k, "k", B, q_len, d, dtype)
    vr, v_heads = _kv8_rows(v, "v", B, q_len, d, dtype)
    if k_heads != H or v_heads != H:
        raise _lib.BtError(f"k and v must have the cache's {H} heads")
    if q_len == 0:
        raise _lib.BtError("no rows to append")
    qr = qor = None
    heads = rot = max_pos = 0
    cos = sin = None
    if q is not None:
        qr, heads = _kv8_rows(q, "q", B, q_len, d, dtype)
    if q_out is not None and q_out.dim() == 4:
        _apart(q_out, "q_out")
    pos_dev, pos_host = _pos0(pos0)
    index = k.get_device()
    with _on(index, *kv, q, v, rope, pos_table, q_out, pos0 if pos_dev else None):
        if rope is not None:
            table = rope.shape
            if len(table) != 3 or table[0] != 2 or rope.dtype != torch.float32 or not rope.is_contiguous():
                raise _lib.BtError("rope must be contiguous float32 [2, max_pos, rot / 2] (rope_tables)")
            max_pos, rot = table[1], 2 * table[2]
        if rot:
            cos = rope.data_ptr()
            sin = cos + max_pos * table[2] * 4
            if q is not None:
                if q_out is None:
                    q_out = torch.empty_like(q, memory_format=_CONTIGUOUS)
                elif q_out.shape != q.shape:
                    raise _lib.BtError("q_out must have q's shape")
                qor = _kv8_rows(q_out, "q_out", B, q_len, d, dtype)[0]
        elif q_out is not None:
            raise _lib.BtError("q_out without rope: there is nothing to rotate q by")
        if pos_table is not None and (pos_table.dtype != torch.int32 or pos_table.dim() != 1 or not pos_table.is_contiguous() or
                                      pos_table.numel() < (n_max if pos_dev else pos_host + q_len)):
            raise _lib.BtError("pos_table must be contiguous int32 and hold an entry for every row")
        check(lib().bt_kv8_append(code, ctypes.byref(cache), q_len, heads if rot else 0, qr if rot else None, qor, kr, vr, pos_dev, pos_host,
                                  _at(pos_table), rot, cos, sin, max_pos, _raw_stream(index)), "bt_kv8_append")
    return q_out if rot else q


def kv8_read(kv: Sequence[torch.Tensor], n: int, first: int = 0, count: Optional[int] = None):
    """(k, v) [B, kv_heads, count, d]: rows [first, first + count) (default: to the end) of a layer of an 8-bit cache that holds ``n``
    rows, in the cache's dtype."""
    cache, code, B, H, n_max, d, _ = _kv8(kv)
    count = n - first if count is None else count
    if not 0 <= first <= first + count <= n <= n_max:
        raise _lib.BtError(f"rows [{first}, {first + count}) of {n} in a cache of {n_max}")
    index = kv[0].get_device()
    with _on(index, *kv):
        k = kv[4].new_empty(B, H, count, d)
        v = torch.empty_like(k)
        check(lib().bt_kv8_read(code, ctypes.byref(cache), n, first, count, k.data_ptr(), v.data_ptr(), _raw_stream(index)), "bt_kv8_read")
    return k, v


def attention_kv8(q: torch.Tensor, kv: Sequence[torch.Tensor], pos0, mask: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, n_split: int = 0, ws: Optional[torch.Tensor] = None):
    """softmax(q k^T / sqrt(d)) v over a layer of an 8-bit cache: row t of ``q`` [B, q_len, heads, d] (rotated, any outer strides; heads a
    multiple of the cache's) sees the rows j <= pos0 + t with mask[b, j] != 0 (uint8 or bool [B, >= n], one row expanded too); zeros where none
    is left.  The
    rows pos0 .. pos0 + q_len - 1 are in the cache already.  ``n_split``: workgroups that share a head's rows (0: chosen from the sizes;
    with a device-side pos0 from the cache's size); ``ws``: >= bt_attention_kv8_workspace_bytes, allocated when needed and not given."""
    cache, code, B, H, n_max, d, dtype = _kv8(kv)
    q_len = q.shape[1] if q.dim() == 4 else 0
    qr, heads = _kv8_rows(q, "q", B, q_len, d, dtype)
    if q_len == 0 or heads == 0 or heads % H:
        raise _lib.BtError(f"{heads} query heads cannot share {H} key/value heads ({q_len} rows)")
    pos_dev, pos_host = _pos0(pos0)
    mask_ld = 0
    if mask is not None:
        if mask.dim() != 2 or mask.shape[0] != B or mask.dtype not in (torch.uint8, torch.bool) or mask.stride(1) != 1:
            raise _lib.BtError(f"mask must be uint8 or bool [{B}, rows] with unit inner stride")
        mask_ld = mask.stride(0) if B > 1 else mask.shape[1]
        if mask.shape[1] < (n_max if pos_dev else pos_host + q_len):
            raise _lib.BtError("mask row too short")
    _flat_memory(ws, "ws")
    index = q.get_device()
    with _on(index, *kv, mask, out, ws, pos0 if pos_dev else None):
        if out is None:
            out = torch.empty_like(q, memory_format=_CONTIGUOUS)
        elif out.shape != (B, q_len, heads, d) or out.dtype != dtype or not out.is_contiguous():
            raise _lib.BtError(f"out must be contiguous {dtype} [{B}, {q_len}, {heads}, {d}]")
        if n_split <= 0:
            n_split = lib().bt_attention_kv8_split_count(B, H, heads // H, q_len, n_max if pos_dev else pos_host + q_len)
        if ws is None and n_split > 1:
            need = int(lib().bt_attention_kv8_workspace_bytes(B, q_len, heads, d, n_split))
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        check(lib().bt_attention_kv8(code, ctypes.byref(cache), q_len, heads, qr, pos_dev, pos_host, _at(mask), mask_ld, out.data_ptr(),
                                     heads * d, n_split, _at(ws), 0 if ws is None else ws.numel() * ws.element_size(), _raw_stream(index)),
              "bt_attention_kv8")
    return out
