"""8-bit serving on the GPU (quantize_rows, linear_q8, the 8-bit KV cache and its attention) against the float64 oracle.

Tolerances, derived here once.  u = finfo(dtype).eps / 2 is the largest relative error of one rounding (bf16 2^-8, fp32 2^-24).
* codes and scales have no tolerance: the definition fixes every bit.  Behind a LayerNorm in fp32 the value that is quantised is off by
  at most (K + 20) 2^-24 of the row's size, here below 1e-3 of a step beside the half step that rounding may take.
* linear: an exact integer, then fl(int), sa * sw, their product, + bias, (gelu), + residual: six roundings of 2^-24 relative to the
  sum of magnitudes, and one of the output type.
* attention: q in D digits is off by amax|q| / (2 Q) per element, Q = 127 * 256 (bf16) or 127 * 65536 (fp32), so a score by
  ds <= sqrt(d) amax|q| max|k| / (2 Q) + 2^-20 (1 + max|s|); a probability by a factor exp(+-2 ds), and by at most 1 / (2 P) of its
  64-row tile's largest from its own three digits, P = 127 * 65536: |error| <= max|v| (exp(2 ds) - 1 + 64 / P) + u |out|.  That is a
  worst case; in the 2-norm the digits' errors are independent and the result has to be within u + 3e-4 (bf16), 2e-5 (fp32)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from block_transformer_amd import ops  # noqa: E402
from block_transformer_amd.runtime import KV8Cache  # noqa: E402
from oracle import q8_ref as ref  # noqa: E402

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def rnd(*shape, seed=0, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- quantize_rows ----------------------------------------------------------------------------------------------------------
def check_codes(x, codes, scales):
    want, s = ref.quantize_rows(x)
    K = x.shape[1]
    assert codes.dtype == torch.int8 and codes.shape == (x.shape[0], (K + 15) // 16 * 16)
    assert torch.equal(scales.double().cpu(), s)
    assert torch.equal(codes.cpu()[:, :K].double(), want)
    assert not codes[:, K:].any()


@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 17), (5, 515), (4, 2048), (2, 8192), (3, 20001), (67, 64), (9, 1000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows(M, K, dtype):
    x = rnd(M, K, seed=M * K, dtype=dtype)
    check_codes(x, *ops.quantize_rows(x.to(DEV)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_ties_and_range(dtype):
    """Values on and beside the border between two codes, and rows at the ends of the type's range."""
    half = torch.arange(-127, 128).double() / 2            # amax 63.5: scale 0.5, every other value a tie
    rows = [half * 2, half * 2 * 3, half * 2 / 3, half * 1e-38, half * 1e-41, half * 5e36, torch.zeros(255, dtype=torch.float64),
            half + 1e-6, torch.arange(255).double() * 127 / 254 * 1.7]
    x = torch.stack(rows).to(F32).to(dtype)
    check_codes(x, *ops.quantize_rows(x.to(DEV)))
    y = x[:1].repeat(40, 1) * (1 + torch.arange(40)[:, None] * 2.0 ** -7).to(dtype)      # the scale moves against the ties
    check_codes(y, *ops.quantize_rows(y.to(DEV)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_strides_and_shapes(dtype):
    base = rnd(7, 300, seed=3, dtype=dtype).to(DEV)
    for x in (base[:, 1:290], base[::2, 8:264], base[:, :33]):
        check_codes(x.cpu(), *ops.quantize_rows(x))
    c, s = ops.quantize_rows(base.view(7, 3, 100))
    assert c.shape == (7, 3, 112) and s.shape == (7, 3)
    check_codes(base.view(21, 100).cpu(), c.view(21, 112), s.view(21))
    c, s = ops.quantize_rows(base[:0])
    assert c.shape == (0, 304) and s.shape == (0,)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_not_finite(dtype):
    x = rnd(5, 96, seed=4, dtype=dtype)
    clean = x.clone()
    x[1, 95], x[2, 0], x[4, 50] = float("nan"), float("inf"), float("-inf")
    c, s = ops.quantize_rows(x.to(DEV))
    assert torch.isnan(s.cpu()).tolist() == [False, True, True, False, True]
    assert not c[[1, 2, 4]].any()
    want, ws = ref.quantize_rows(clean)
    assert torch.equal(c.cpu()[[0, 3]].double(), want[[0, 3]]) and torch.equal(s.cpu()[[0, 3]].double(), ws[[0, 3]])


@pytest.mark.parametrize("M,K", [(3, 64), (2, 2048), (5, 515), (1, 9000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_rows_of_a_layernorm(M, K, dtype):
    x = rnd(M, K, seed=5, scale=2.0, dtype=dtype) + 1
    w, b = (rnd(K, seed=6, scale=0.2) + 1).to(dtype), rnd(K, seed=7, scale=0.2, dtype=dtype)
    c, s = ops.quantize_rows(x.to(DEV), w.to(DEV), b.to(DEV), eps=1e-5)
    y = ref.layernorm(x, w, b, 1e-5)
    s = s.double().cpu()
    assert ((s - y.abs().amax(1) / 127).abs() <= 1e-5 * s).all()
    assert ((c.cpu()[:, :K].double() - y / s[:, None]).abs() <= 0.5 + 1e-3).all()
    assert not c[:, K:].any()


def gelu_error(dtype):
    """erff's few ulps of fp32; for bf16 the epilogue's polynomial, 8.5e-6 relative for x > -6 (and below 8e-9 beyond, where |x| = size)."""
    return 2e-6 if dtype == F32 else 1e-5


# ---- linear_q8 --------------------------------------------------------------------------------------------------------------
def linear_case(M, N, K, dtype, seed=0, bias=True, residual=False, act="none"):
    g = torch.Generator().manual_seed(seed)
    Kp = (K + 15) // 16 * 16
    a, w = torch.zeros(M, Kp, dtype=torch.int8), torch.zeros(N, Kp, dtype=torch.int8)
    a[:, :K] = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8)
    w[:, :K] = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    sa, sw = torch.rand(M, generator=g) * 0.02 + 0.01, (torch.rand(N, generator=g) * 0.02 + 0.01) * K ** -0.5
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    r = torch.randn(M, N, generator=g).to(dtype) if residual else None
    acc = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    y, size = acc, acc.abs()
    if bias:
        y, size = y + b.double(), size + b.double().abs()
    if act == "gelu":
        y = ref.gelu(y)
    if residual:
        y, size = y + r.double(), size + r.double().abs()
    return (a, sa), (w, sw), b, r, y, half_step(dtype) * y.abs() + (6 * 2 ** -24 + (gelu_error(dtype) if act == "gelu" else 0)) * size + 1e-30


def cuda(v):
    return tuple(t.to(DEV) for t in v) if isinstance(v, tuple) else None if v is None else v.to(DEV)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (1, 6144, 2048), (2, 100, 40), (5, 192, 64), (16, 256, 1024), (17, 48, 128), (33, 1000, 515),
                                   (64, 512, 256), (77, 1001, 515), (128, 128, 64), (130, 260, 128), (257, 768, 384), (300, 520, 2048),
                                   (512, 512, 512), (1025, 264, 192), (256, 2048, 8192), (2049, 2304, 1024)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("variant", ["plain", "bias_gelu", "bias_res", "gelu_res"])
def test_linear_q8(M, N, K, dtype, variant):
    x, w, b, r, y, tol = linear_case(M, N, K, dtype, seed=M + N, bias="bias" in variant, residual="res" in variant,
                                     act="gelu" if "gelu" in variant else "none")
    out = ops.linear_q8(cuda(x), cuda(w), cuda(b), cuda(r), act="gelu" if "gelu" in variant else "none", dtype=dtype)
    assert out.dtype == dtype and out.shape == (M, N)
    assert ((out.cpu().double() - y).abs() <= tol).all()


@pytest.mark.parametrize("M,N,K", [(3500, 3650, 128), (4100, 3137, 256), (8197, 1616, 384), (1100, 12000, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("variant", ["bias_gelu", "bias_res"])
def test_linear_q8_many_tiles(M, N, K, dtype, variant):
    """Products of more tiles than the card has CUs, cut at both edges, of one step of K and more."""
    x, w, b, r, y, tol = linear_case(M, N, K, dtype, seed=M, residual="res" in variant, act="gelu" if "gelu" in variant else "none")
    out = ops.linear_q8(cuda(x), cuda(w), cuda(b), cuda(r), act="gelu" if "gelu" in variant else "none", dtype=dtype)
    assert ((out.cpu().double() - y).abs() <= tol).all()


@pytest.mark.parametrize("M,N,K", [(3900, 2040, 1024), (4000, 2048, 640), (5567, 2850, 640), (4100, 3144, 1024)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("variant", ["bias_gelu", "bias_res"])
def test_linear_q8_tall_tiles_and_cut_rows(M, N, K, dtype, variant):
    """Products of about as many 256 x 128 tiles as the card has CUs and twice that, whose last rows are no whole tile; once and onto
    itself."""
    x, w, b, r, y, tol = linear_case(M, N, K, dtype, seed=M, residual="res" in variant, act="gelu" if "gelu" in variant else "none")
    act = "gelu" if "gelu" in variant else "none"
    x, w, b, r = cuda(x), cuda(w), cuda(b), cuda(r)
    out = ops.linear_q8(x, w, b, r, act=act, dtype=dtype)
    assert ((out.cpu().double() - y).abs() <= tol).all()
    for _ in range(3):
        again = torch.empty(M + 1, N, dtype=dtype, device=DEV).fill_(7)
        ops.linear_q8(x, w, b, r, act=act, dtype=dtype, out=again[:M])
        assert torch.equal(again[:M], out) and (again[M] == 7).all()


@pytest.mark.parametrize("M", [1, 3, 40, 200])
def test_linear_q8_largest_sums(M):
    """Every product 127 * 127 (or -127 * 127): the sum is exact to the last bit right up to the K that is refused."""
    K, N = 131056, 48
    a, w = torch.full((M, K), 127, dtype=torch.int8, device=DEV), torch.full((N, K), 127, dtype=torch.int8, device=DEV)
    w[1::2] = -127
    w[2, 5] = 126
    one = torch.ones(max(M, N), device=DEV)
    out = ops.linear_q8((a, one[:M]), (w, one[:N]), dtype=F32).cpu()
    total = 127 * 127 * K
    assert (out[:, 0] == torch.tensor(total).float()).all() and (out[:, 1] == -torch.tensor(total).float()).all()
    assert (out[:, 2] == torch.tensor(total - 127).float()).all()


@pytest.mark.parametrize("M,N,K", [(9, 70, 64), (70, 136, 256), (600, 300, 256), (300, 2048, 512)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_q8_strides_and_untouched_memory(M, N, K, dtype):
    """Operands and results inside larger, oddly aligned buffers: nothing outside the result is written."""
    x, w, b, r, y, tol = linear_case(M, N, K, dtype, seed=8, residual=True)
    a = torch.full((M + 2, K + 48), 55, dtype=torch.int8, device=DEV)
    a[1:-1, 16:16 + K] = cuda(x[0])
    wc = torch.full((N + 3, K + 16), 99, dtype=torch.int8, device=DEV)
    wc[2:-1, 16:] = cuda(w[0])
    res = torch.zeros(M, N + 7, dtype=dtype, device=DEV)
    res[:, 3:3 + N] = cuda(r)
    out = torch.full((M + 2, N + 5), 7.0, dtype=dtype, device=DEV)
    ops.linear_q8((a[1:-1, 16:16 + K], cuda(x[1])), (wc[2:-1, 16:], cuda(w[1])), cuda(b), res[:, 3:3 + N], out=out[1:-1, 1:1 + N])
    assert ((out[1:-1, 1:1 + N].cpu().double() - y).abs() <= tol).all()
    out[1:-1, 1:1 + N] = 7.0
    assert (out == 7.0).all()


@pytest.mark.parametrize("M,N,K", [(5, 40, 32), (33, 70, 16), (100, 130, 48), (200, 72, 80), (257, 264, 336)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_q8_short_and_cut_steps_of_k(M, N, K, dtype):
    x, w, b, _, y, tol = linear_case(M, N, K, dtype, seed=K)
    assert ((ops.linear_q8(cuda(x), cuda(w), cuda(b)).cpu().double() - y).abs() <= tol).all()


@pytest.mark.parametrize("M,N,K", [(3, 264, 128), (200, 512, 256), (300, 2048, 4096), (3500, 3650, 128)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_q8_onto_its_own_residual(M, N, K, dtype):
    x, w, b, r, y, tol = linear_case(M, N, K, dtype, seed=12, residual=True)
    stream = cuda(r)
    assert ops.linear_q8(cuda(x), cuda(w), cuda(b), stream, out=stream) is stream
    assert ((stream.cpu().double() - y).abs() <= tol).all()


def test_linear_q8_of_float_rows_and_a_row_that_is_not_finite():
    x, w = rnd(6, 200, seed=9), rnd(50, 200, seed=10)
    x[2, 7] = float("nan")
    out = ops.linear_q8(x.to(DEV), ops.quantize_rows(w.to(DEV)))
    assert torch.isnan(out[2]).all() and torch.isfinite(out[[0, 1, 3, 4, 5]]).all()
    keep = [0, 1, 3, 4, 5]
    (cx, sx), (cw, sw) = ref.quantize_rows(x[keep]), ref.quantize_rows(w)
    y = (cx @ cw.T) * sx[:, None] * sw
    assert ((out.cpu()[keep].double() - y).abs() <= 7 * 2 ** -24 * y.abs()).all()
    assert ops.linear_q8(x[:0].to(DEV), ops.quantize_rows(w.to(DEV))).shape == (0, 50)


@pytest.mark.parametrize("M,N,K", [(1, 2048, 8192), (100, 2048, 8192), (256, 256, 4096), (513, 1024, 4096)])
def test_linear_q8_is_the_same_with_and_without_scratch_and_from_call_to_call(M, N, K):
    x, w, b, _, _, _ = linear_case(M, N, K, BF16, seed=11)
    x, w, b = cuda(x), cuda(w), cuda(b)
    none = torch.empty(0, dtype=torch.uint8, device=DEV)
    first = ops.linear_q8(x, w, b)
    for _ in range(3):
        assert torch.equal(ops.linear_q8(x, w, b), first)
    assert torch.equal(ops.linear_q8(x, w, b, scratch=none), first)


# ---- the cache --------------------------------------------------------------------------------------------------------------
def table(rot, n=4096):
    return ops.rope_tables(n, rot, 10000.0, "cpu")


def new_cache(B, H, n_max, d, dtype, block, fill=None):
    """A cache whose unused places hold `fill`: 77 and NaN, so that reading one of them shows."""
    c = KV8Cache(1, B, H, n_max, d, dtype, DEV, block=block)
    c.k_codes.fill_(77), c.v_codes.fill_(77)
    for t in (c.k_scale, c.v_scale, c.k_tail, c.v_tail):
        t.fill_(float("nan"))
    return c[0]


def same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all() if a.is_floating_point() else (a == b).all())


def check_cache(kv, want, n, block):
    """Codes and scales of the full blocks and the open block's rows, bit for bit; everything else as new_cache left it."""
    full = n // block
    kc, vc, ks, vs, kt, vt = (t.cpu() for t in kv)
    B, H = kc.shape[:2]
    for which, codes, scales, tail in (("k", kc.view(B, H, -1, block, kc.shape[3]), ks, kt), ("v", vc.transpose(3, 4), vs, vt.transpose(2, 3))):
        _, c, s = want.rows(which)
        rows = want.k if which == "k" else want.v
        if full:
            c = torch.stack(c).view(full, B, H, block, -1).permute(1, 2, 0, 3, 4)
            s = torch.stack(s).view(full, B, H).permute(1, 2, 0)
            assert torch.equal(scales[:, :, :full].double(), s), which
            assert torch.equal(codes[:, :, :full].double(), c), which
        assert (codes[:, :, full:] == 77).all() and scales[:, :, full:].isnan().all(), which
        open_rows = rows[:, :, full * block:]
        assert same(tail[:, :, :n - full * block], open_rows), which


CACHES = [(1, 1, 1, 32, 16, 8, F32), (2, 4, 2, 64, 16, 16, BF16), (2, 3, 3, 128, 32, 32, BF16), (1, 8, 1, 128, 64, 128, F32),
          (3, 2, 2, 64, 64, 10, BF16), (2, 2, 2, 32, 32, 6, F32)]


@pytest.mark.parametrize("B,heads,H,d,block,rot,dtype", CACHES)
@pytest.mark.parametrize("chunks", [(1,), (5, 1, 1), (16, 16), (64,), (70, 1, 60), (3, 130, 1, 1), (15, 1, 16, 33, 63), (200, 7)])
def test_append(B, heads, H, d, block, rot, dtype, chunks):
    kv, want, t = new_cache(B, H, 256, d, dtype, block), ref.Cache(B, H, d, block, dtype), table(rot)
    pos = 0
    for i, c in enumerate(chunks):
        x = rnd(B, c, heads + 2 * H, d, seed=100 * i + c, dtype=dtype)
        q, k, v = x[:, :, :heads], x[:, :, heads:heads + H], x[:, :, heads + H:]
        xg = x.to(DEV)
        got = ops.kv8_append(kv, xg[:, :, :heads], xg[:, :, heads:heads + H], xg[:, :, heads + H:], pos, rope=t.to(DEV))
        at = torch.arange(pos, pos + c)
        assert torch.equal(got.cpu(), ref.rope(q, at, t).to(dtype))
        assert torch.equal(xg.cpu(), x)                       # the rows themselves stay as they were
        want.append(k, v, at, t)
        pos += c
        check_cache(kv, want, pos, block)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_at_once_is_append_one_by_one(dtype):
    B, H, d, block, n = 3, 4, 64, 32, 107
    x = rnd(B, n, 2, H, d, seed=21, dtype=dtype).to(DEV)
    a, b = new_cache(B, H, n, d, dtype, block), new_cache(B, H, n, d, dtype, block)
    t = table(32).to(DEV)
    ops.kv8_append(a, None, x[:, :, 0], x[:, :, 1], 0, rope=t)
    for i in range(n):
        ops.kv8_append(b, None, x[:, i:i + 1, 0], x[:, i:i + 1, 1], i, rope=t)
    for one, two in zip(a[:4], b[:4]):
        assert same(one, two)
    for first, count in ((0, n), (5, 100), (96, 11), (n - 1, 1), (3, 0)):
        for one, two in zip(ops.kv8_read(a, n, first, count), ops.kv8_read(b, n, first, count)):
            assert one.shape == (B, H, count, d) and torch.equal(one, two)


def test_append_without_rotation_in_place_with_a_table_and_on_strided_rows():
    B, heads, H, d, block, n = 2, 4, 2, 64, 16, 40
    kv, want = new_cache(B, H, 64, d, BF16, block), ref.Cache(B, H, d, block, BF16)
    wide = rnd(B, n + 3, 3, heads, d + 8, seed=22, dtype=BF16).to(DEV)
    q, k, v = wide[:, 1:n + 1, 0, :, :d], wide[:, 1:n + 1, 1, ::2, 8:], wide[:, 2:n + 2, 2, 1:3, :d]
    assert ops.kv8_append(kv, q, k, v, 0) is q                # nothing to rotate by
    want.append(k.cpu(), v.cpu())
    check_cache(kv, want, n, block)
    t, pos_table = table(16), (torch.arange(64) * 7 % 50).int()
    at = pos_table[n:n + 1].long()
    q0, k0, v0 = (x.cpu().clone() for x in (q[:, :1], k[:, :1], v[:, :1]))
    one = q[:, :1]
    assert ops.kv8_append(kv, one, k[:, :1], v[:, :1], n, rope=t.to(DEV), pos_table=pos_table.to(DEV), q_out=one) is one
    want.append(k0, v0, at, t)
    check_cache(kv, want, n + 1, block)
    assert torch.equal(one.cpu(), ref.rope(q0, at, t).to(BF16))
    before = [x.clone() for x in kv]
    ops.kv8_append(kv, None, k[:, :1].expand(B, 1, H, d), v[:, :1], n, rope=t.to(DEV), pos_table=pos_table.to(DEV))     # the same row again
    assert all(same(a, b) for a, b in zip(kv, before))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_rows_that_are_not_finite(dtype):
    """One such row does not spoil the rows of its block; in the open block it stands as it came."""
    B, H, d, block = 1, 2, 32, 16
    x = rnd(B, 20, 2, H, d, seed=23, dtype=dtype)
    x[0, 3, 0, 0, 5], x[0, 3, 1, 0, 6], x[0, 9, 0, 1, 0], x[0, 18, 1, 1, 2] = (float(s) for s in ("inf", "nan", "-inf", "nan"))
    x[0, 0:16, 1, 1] = float("inf")                           # nothing finite in the block: scale 0
    kv, want = new_cache(B, H, 32, d, dtype, block), ref.Cache(B, H, d, block, dtype)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    want.append(x[:, :, 0], x[:, :, 1])
    check_cache(kv, want, 20, block)


def test_append_beyond_the_end_with_a_device_position():
    B, H, d, block = 2, 2, 32, 16
    x = rnd(B, 8, 2, H, d, seed=24, dtype=BF16)
    kv, want = new_cache(B, H, 32, d, BF16, block), ref.Cache(B, H, d, block, BF16)
    first = rnd(B, 28, 2, H, d, seed=25, dtype=BF16)
    ops.kv8_append(kv, None, first.to(DEV)[:, :, 0], first.to(DEV)[:, :, 1], 0)
    pos = torch.tensor([28], dtype=torch.int32, device=DEV)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], pos)
    want.append(torch.cat([first, x], 1)[:, :32, 0], torch.cat([first, x], 1)[:, :32, 1])
    check_cache(kv, want, 32, block)
    before = [t.clone() for t in kv]
    for p in (32, 1000, -1):
        ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], pos.fill_(p))
    assert all(same(a, b) for a, b in zip(kv, before))
    # the queries of rows that are dropped take the position table's last entry
    t, at = table(16), (torch.arange(32) * 5 % 31).int()
    q = ops.kv8_append(kv, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], pos.fill_(30), rope=t.to(DEV), pos_table=at.to(DEV))
    assert torch.equal(q.cpu(), ref.rope(x[:, :, 0], at[torch.arange(30, 38).clamp(max=31)].long(), t).to(BF16))


@pytest.mark.parametrize("B,heads,H,d,block,rot,dtype", CACHES)
@pytest.mark.parametrize("n", [1, 16, 63, 64, 150])
def test_read(B, heads, H, d, block, rot, dtype, n):
    kv, want = new_cache(B, H, n, d, dtype, block), ref.Cache(B, H, d, block, dtype)
    x = rnd(B, n, 2, H, d, seed=n, dtype=dtype)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    want.append(x[:, :, 0], x[:, :, 1])
    for first, count in ((0, n), (n // 2, n - n // 2), (n // 3, 1)):
        for got, which in zip(ops.kv8_read(kv, n, first, count), "kv"):
            y = want.rows(which)[0][:, :, first:first + count]
            assert ((got.cpu().double() - y).abs() <= (half_step(dtype) + 2 ** -24) * y.abs()).all()


# ---- attention --------------------------------------------------------------------------------------------------------------
def attention_case(B, heads, H, d, block, dtype, n, q_len, seed, q_scale=2.0):
    """A cache of n rows (unused places: 77 and NaN) and q."""
    kv, want = new_cache(B, H, n + 70, d, dtype, block), ref.Cache(B, H, d, block, dtype)
    x = rnd(B, n, 2, H, d, seed=seed, dtype=dtype)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    want.append(x[:, :, 0], x[:, :, 1])
    q = rnd(B, q_len, heads, d, seed=seed + 1, scale=q_scale, dtype=dtype)
    return kv, want.rows("k")[0], want.rows("v")[0], q


def check_attention(out, y, q, k, v, dtype):
    d = q.shape[3]
    Q, P = 127 * (256 if dtype == BF16 else 65536), 127 * 65536
    big = float(q.double().abs().max()), float(k.abs().nan_to_num(0, 0, 0).max()), float(v.abs().nan_to_num(0, 0, 0).max())
    ds = math.sqrt(d) * big[0] * big[1] / (2 * Q) + 2 ** -20 * (1 + math.sqrt(d) * big[0] * big[1])
    off = (out.cpu().double() - y).abs()
    assert (off <= big[2] * (math.expm1(2 * ds) + 64 / P) + half_step(dtype) * y.abs()).all()
    if y.norm() > 0:
        assert off.norm() / y.norm() <= (half_step(BF16) + 3e-4 if dtype == BF16 else 2e-5)


SHAPES = [(1, 1, 1, 32, 16, F32), (2, 4, 4, 128, 16, BF16), (2, 8, 2, 64, 32, BF16), (1, 16, 1, 128, 64, BF16), (2, 6, 2, 64, 64, F32),
          (1, 4, 4, 128, 32, F32), (3, 3, 3, 32, 64, BF16), (1, 20, 1, 32, 16, BF16)]


@pytest.mark.parametrize("B,heads,H,d,block,dtype", SHAPES)
@pytest.mark.parametrize("n,q_len", [(1, 1), (2, 2), (15, 1), (16, 1), (17, 3), (64, 1), (65, 2), (130, 1), (255, 4), (400, 1), (300, 17)])
def test_attention(B, heads, H, d, block, dtype, n, q_len):
    kv, k, v, q = attention_case(B, heads, H, d, block, dtype, n, q_len, seed=n + d)
    y = ref.attention(q, k, v, n - q_len)
    check_attention(ops.attention_kv8(q.to(DEV), kv, n - q_len), y, q, k, v, dtype)


@pytest.mark.parametrize("B,heads,H,d,block,dtype", SHAPES[1:6])
def test_attention_of_every_row(B, heads, H, d, block, dtype):
    """As many queries as rows: the first sees one row, the last all."""
    n = 139
    kv, k, v, q = attention_case(B, heads, H, d, block, dtype, n, n, seed=d)
    check_attention(ops.attention_kv8(q.to(DEV), kv, 0), ref.attention(q, k, v, 0), q, k, v, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_with_a_device_position(dtype):
    """The position read on the device, behind the cache's end and before its start too."""
    kv, k, v, q = attention_case(2, 4, 2, 64, 16, dtype, 90, 3, seed=41)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    for p in (87, 40, 0, 63, 64):
        y = ref.attention(q, k[:, :, :p + 3], v[:, :, :p + 3], p)
        if p == 87:      # (rows behind p + 3 stand in codes: a smaller p would take some of them for the open block's)
            check_attention(ops.attention_kv8(q.to(DEV), kv, pos.fill_(p)), y, q, k, v, dtype)
        assert torch.equal(ops.attention_kv8(q.to(DEV), kv, pos.fill_(p), n_split=1).nan_to_num(7),
                           ops.attention_kv8(q.to(DEV), kv, p, n_split=1).nan_to_num(7))
    assert (ops.attention_kv8(q.to(DEV), kv, pos.fill_(-50)) == 0).all()
    assert ops.attention_kv8(q.to(DEV), kv, pos.fill_(1 << 30)).shape == (2, 3, 4, 64)


@pytest.mark.parametrize("B,heads,H,d,block,dtype", SHAPES[:6])
@pytest.mark.parametrize("n,q_len", [(40, 1), (200, 3), (520, 1)])
@pytest.mark.parametrize("as_bool", [False, True])
def test_attention_masks(B, heads, H, d, block, dtype, n, q_len, as_bool):
    """Padding on the left, holes, a sequence with nothing left; what is masked may be anything."""
    kv, k, v, q = attention_case(B, heads, H, d, block, dtype, n, q_len, seed=n)
    g = torch.Generator().manual_seed(n)
    mask = torch.rand(B, n + 5, generator=g) < 0.6
    mask[0, :n // 3] = False
    if B > 1:
        mask[1] = False
    if block < n:      # masked garbage: an infinite scale's codes cannot be masked out, NaN rows of the open block can
        hidden = (n // block * block) + 1
        if hidden < n:
            mask[:, hidden] = False
            kv[4][:, :, hidden % block] = float("nan")
            kv[5][:, :, :, hidden % block] = float("inf")
    y = ref.attention(q, k, v, n - q_len, mask)
    m = mask.to(DEV) if as_bool else mask.to(torch.uint8).to(DEV)
    out = ops.attention_kv8(q.to(DEV), kv, n - q_len, mask=m)
    check_attention(out, y, q, k, v, dtype)
    if B > 1:
        assert (out[1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_masked_infinities_of_a_full_block(dtype):
    """Padding rows that held infinities and NaN when their block was quantised, masked at the step."""
    B, H, d, block, n = 2, 2, 64, 16, 90
    x = rnd(B, n, 2, H, d, seed=31, dtype=dtype)
    x[:, 4:7] = float("inf")
    x[:, 20, :, :, ::3] = float("nan")
    kv, want = new_cache(B, H, n, d, dtype, block), ref.Cache(B, H, d, block, dtype)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    want.append(x[:, :, 0], x[:, :, 1])
    mask = torch.ones(B, n, dtype=torch.uint8)
    mask[:, 4:7], mask[:, 20] = 0, 0
    q = rnd(B, 1, H, d, seed=32, dtype=dtype)
    k, v = want.rows("k")[0], want.rows("v")[0]
    y = ref.attention(q, k, v, n - 1, mask)
    assert torch.isfinite(y).all()
    check_attention(ops.attention_kv8(q.to(DEV), kv, n - 1, mask=mask.to(DEV)), y, q, k, v, dtype)


@pytest.mark.parametrize("B,heads,H,d,block,dtype", SHAPES[1:6])
def test_attention_masked_blocks_that_were_never_written(B, heads, H, d, block, dtype):
    """Blocks that the mask hides as a whole may hold any codes and scales."""
    n = 5 * block + 70
    kv, k, v, q = attention_case(B, heads, H, d, block, dtype, n, 2, seed=43)
    mask = torch.ones(B, n, dtype=torch.uint8)
    for j, bad in ((0, "nan"), (2, "inf"), (3, "-inf"), (4, "nan")):
        mask[:, j * block:(j + 1) * block] = 0
        kv[2][:, :, j], kv[3][:, :, j] = float(bad), float(bad)
        kv[0][:, :, j * block:(j + 1) * block], kv[1][:, :, j] = -128, -128
    mask[0, :] = 0
    out = ops.attention_kv8(q.to(DEV), kv, n - 2, mask=mask.to(DEV))
    check_attention(out, ref.attention(q, k, v, n - 2, mask), q, k, v, dtype)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_queries_and_open_rows_that_are_not_finite(dtype):
    """NaN where a NaN or infinity takes part, and in those rows alone."""
    kv, k, v, q = attention_case(2, 2, 2, 64, 16, dtype, 40, 1, seed=33)
    q[1, 0, 1, 3] = float("nan")
    kv[4][0, 0, 5, 7] = float("nan")                          # row 37 of the open block
    out = ops.attention_kv8(q.to(DEV), kv, 39).cpu()
    assert out[1, 0, 1].isnan().all() and out[0, 0, 0].isnan().all()
    assert torch.isfinite(out[0, 0, 1]).all() and torch.isfinite(out[1, 0, 0]).all()
    q[1, 0, 1, 3] = float("inf")
    assert not torch.isfinite(ops.attention_kv8(q.to(DEV), kv, 39).cpu()[1, 0, 1]).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e-3, 40.0])
def test_attention_flat_and_peaked(dtype, q_scale):
    kv, k, v, q = attention_case(2, 4, 2, 64, 32, dtype, 330, 1, seed=34, q_scale=q_scale)
    y = ref.attention(q, k, v, 329)
    out = ops.attention_kv8(q.to(DEV), kv, 329)
    if q_scale <= 2:
        check_attention(out, y, q, k, v, dtype)
    else:      # scores near 1000: the worst case above says nothing, but the result is a mean of v's rows and no NaN
        assert torch.isfinite(out).all() and out.abs().max().cpu() <= v.abs().max() * 1.01


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_keeps_small_probabilities_beside_a_sink(dtype):
    """One row takes nearly everything but has v = 0: the result is what the many small probabilities say.  They are e^-12 = 6.1e-6 of the
    largest; the 63 that share its tile are held in steps of 1 / P = 1.2e-7, an error of 0.29 * 1.2e-7 / 6.1e-6 = 0.6 % each and so of
    0.006 sqrt(63 / 1000) = 1.4e-3 of the sum over 1000 rows in the 2-norm; 3e-3 is allowed."""
    B, H, d, block, n = 1, 1, 64, 16, 1000
    x = rnd(B, n, 2, H, d, seed=35, scale=0.2, dtype=dtype)
    q = torch.zeros(B, 1, H, d, dtype=dtype)
    q[..., 0] = 8.0
    x[0, :, 0, :, 0] = 0
    x[0, 0, 0, :, 0], x[0, 0, 1] = 12.0, 0                    # score 12, the others 0: e^-12 each
    x[0, 1:16, 0] = 0                                         # (they share the sink's scale)
    kv, want = new_cache(B, H, n, d, dtype, block), ref.Cache(B, H, d, block, dtype)
    ops.kv8_append(kv, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    want.append(x[:, :, 0], x[:, :, 1])
    y = ref.attention(q, want.rows("k")[0], want.rows("v")[0], n - 1)
    out = ops.attention_kv8(q.to(DEV), kv, n - 1).cpu().double()
    assert ((out - y).norm() / y.norm()) <= (half_step(BF16) + 3e-4 if dtype == BF16 else 3e-3)


@pytest.mark.parametrize("n_split", [1, 2, 3, 7, 40])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_splits(n_split, dtype):
    """Split over more workgroups than there are tiles too; empty parts and masked parts count for nothing."""
    B, heads, H, d, block, n = 2, 4, 2, 128, 16, 701
    kv, k, v, q = attention_case(B, heads, H, d, block, dtype, n, 2, seed=36)
    mask = torch.ones(B, n, dtype=torch.uint8)
    mask[0, :500] = 0
    mask[1, 100:] = 0
    y = ref.attention(q, k, v, n - 2, mask)
    first = ops.attention_kv8(q.to(DEV), kv, n - 2, mask=mask.to(DEV), n_split=n_split)
    check_attention(first, y, q, k, v, dtype)
    ws = torch.full((B * 2 * heads * n_split * (d + 2),), float("nan"), device=DEV)
    for _ in range(2):
        assert torch.equal(ops.attention_kv8(q.to(DEV), kv, n - 2, mask=mask.to(DEV), n_split=n_split, ws=ws), first)


def test_attention_strided_rows_and_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes: the last sequence's rows lie behind them."""
    B, H, d, block, n = 66, 4, 128, 16, 131072
    c = KV8Cache(1, B, H, n, d, BF16, DEV, block=block)
    assert c.k_codes.numel() > 1 << 32
    kv = c[0]
    for t in kv:
        t[B - 1].zero_()
    m = 1000
    x = rnd(1, m, 2, H, d, seed=37, dtype=BF16)
    far = rnd(1, 16, 2, H, d, seed=38, dtype=BF16)
    last = tuple(t[B - 1:] for t in kv)
    ops.kv8_append(last, None, x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], 0)
    ops.kv8_append(last, None, far.to(DEV)[:, :, 0], far.to(DEV)[:, :, 1], n - 16)
    want = ref.Cache(1, H, d, block, BF16)
    want.append(torch.cat([x[:, :992], far], 1)[:, :, 0], torch.cat([x[:, :992], far], 1)[:, :, 1])
    mask = torch.zeros(B, n, dtype=torch.uint8, device=DEV)
    mask[B - 1, :992] = 1
    mask[B - 1, n - 16:] = 1
    big = rnd(B, 1, 3, H, d, seed=39, dtype=BF16)
    q = big.to(DEV)[:, :, 1]
    out = ops.attention_kv8(q, kv, n - 1, mask=mask)
    k, v = want.rows("k")[0], want.rows("v")[0]
    y = ref.attention(big[B - 1:, :, 1], k, v, 1007)
    check_attention(out[B - 1:], y, big[B - 1:, :, 1], k, v, BF16)
    assert (out[:B - 1] == 0).all()
    got = ops.kv8_read(last, n, n - 16)[0].cpu().double()
    assert ((got - k[:, :, 992:]).abs() <= half_step(BF16) * k[:, :, 992:].abs()).all()


# ---- together ---------------------------------------------------------------------------------------------------------------
def layer(w, kv, x, pos, t, heads, d, mask=None):
    """The attention half of a GPT-NeoX layer in 8 bits: LayerNorm and QKV, append, attention, dense onto the residual stream."""
    B, T, H = x.shape
    qkv = ops.linear_q8(ops.quantize_rows(x, w["ln_w"], w["ln_b"]), w["qkv"], w["qkv_b"])
    q, k, v = qkv.view(B, T, heads, 3, d).unbind(3)
    q = ops.kv8_append(kv, q, k, v, pos, rope=t)
    a = ops.attention_kv8(q, kv, pos, mask=mask)
    return ops.linear_q8(a.view(B, T, H), w["dense"], w["dense_b"], residual=x)


def layer_weights(H, dtype, seed=50):
    w = {"ln_w": (rnd(H, seed=seed, scale=0.1) + 1).to(dtype), "ln_b": rnd(H, seed=seed + 1, scale=0.1, dtype=dtype),
         "qkv_b": rnd(3 * H, seed=seed + 2, scale=0.1, dtype=dtype), "dense_b": rnd(H, seed=seed + 3, scale=0.1, dtype=dtype)}
    raw = {"qkv": rnd(3 * H, H, seed=seed + 4, scale=H ** -0.5, dtype=dtype), "dense": rnd(H, H, seed=seed + 5, scale=H ** -0.5, dtype=dtype)}
    gpu = {k: v.to(DEV) for k, v in w.items()} | {k: ops.quantize_rows(v.to(DEV)) for k, v in raw.items()}
    return w, raw, gpu


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_layer_prefilled_and_stepped(dtype):
    """Prefill, then single tokens, against the same layer in float64 without any quantisation: 8-bit rounding has a relative error of
    about 1 / (127 sqrt(12)) * 3.5 = 0.8 % of each operand's spread; through QKV, K, V and dense that stays below 4 % of the layer's own
    contribution in the 2-norm (six such roundings, added in squares: 2 %; twice that is allowed)."""
    B, heads, d, n, steps, block = 3, 4, 64, 37, 14, 16
    H = heads * d
    w, raw, gpu = layer_weights(H, dtype)
    t = table(16)
    x = rnd(B, n + steps, H, seed=60, dtype=dtype)
    kv = new_cache(B, heads, n + steps, d, dtype, block)
    got = [layer(gpu, kv, x[:, :n].to(DEV), 0, t.to(DEV), heads, d)]
    for i in range(n, n + steps):
        got.append(layer(gpu, kv, x[:, i:i + 1].to(DEV), i, t.to(DEV), heads, d))
    got = torch.cat(got, 1).cpu().double()
    y = ref.layernorm(x, w["ln_w"], w["ln_b"], 1e-5) @ raw["qkv"].double().T + w["qkv_b"].double()
    q, k, v = y.view(B, n + steps, heads, 3, d).unbind(3)
    at = torch.arange(n + steps)
    a = ref.attention(ref.rope(q, at, t), ref.rope(k, at, t).transpose(1, 2), v.transpose(1, 2), 0)
    own = a.reshape(B, n + steps, H) @ raw["dense"].double().T + w["dense_b"].double()
    assert (got - x.double() - own).norm() <= (0.04 + 2 * half_step(dtype)) * own.norm()
    # the same rows all at once give the same codes, so nearly the same numbers
    again = layer(gpu, new_cache(B, heads, n + steps, d, dtype, block), x.to(DEV), 0, t.to(DEV), heads, d).cpu().double()
    assert (got - again).norm() <= 0.02 * own.norm()


def test_a_step_captured_and_replayed():
    """The layer's step as a graph that reads its position from the device: every replay, with eager work between, is the eager step."""
    B, heads, d, block, n = 2, 4, 64, 16, 70
    H = heads * d
    _, _, gpu = layer_weights(H, BF16)
    t = table(16).to(DEV)
    xs = rnd(n, B, 1, H, seed=61, dtype=BF16).to(DEV)
    eager_kv, kv = new_cache(B, heads, n, d, BF16, block), new_cache(B, heads, n, d, BF16, block)
    mask = torch.ones(B, kv[0].shape[2], dtype=torch.uint8, device=DEV)
    mask[1, :9] = 0
    pos, x = torch.zeros(1, dtype=torch.int32, device=DEV), xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(gpu, kv, x, pos, t, heads, d, mask)             # warm
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(gpu, kv, x, pos, t, heads, d, mask)
    for i in range(n):
        want = layer(gpu, eager_kv, xs[i], torch.full((1,), i, dtype=torch.int32, device=DEV), t, heads, d, mask)
        x.copy_(xs[i])
        pos.fill_(i)
        graph.replay()
        if i % 7 == 0:
            torch.cuda.synchronize()
        assert torch.equal(out, want), i
    assert all(same(a, b) for a, b in zip(kv, eager_kv))


def test_on_another_stream():
    """Every operator runs on torch's current stream: work queued there before it is seen, without a wait of the host."""
    B, heads, d, block, n = 2, 4, 64, 16, 50
    _, _, gpu = layer_weights(heads * d, BF16)
    t = table(16).to(DEV)
    x = rnd(B, n, heads * d, seed=62, dtype=BF16).to(DEV)
    want = layer(gpu, new_cache(B, heads, n, d, BF16, block), x, 0, t, heads, d)
    kv = new_cache(B, heads, n, d, BF16, block)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        junk = torch.randn(4096, 4096, device=DEV)
        for _ in range(20):
            junk = junk @ junk * 1e-3
        late.copy_(x)
        got = layer(gpu, kv, late, 0, t, heads, d)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
