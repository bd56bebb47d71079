"""CPU restatement, in float64, of the 8-bit serving operators (bt_quant_rows, bt_linear_q8, bt_kv8_*, bt_attention_kv8): test
infrastructure.  Loops over blocks and rows, no vectorised shortcuts: the definitions as they are written in include/bt_hip.h."""
import math

import torch


def scale_of(amax):
    """fl32(amax / 127) of a non-negative float64 tensor that holds fp32 values."""
    return (amax.float() / 127).double()


def codes_of(x, scale):
    """clamp(round_half_even(x / scale), -127, 127); float64.  The quotient of two fp32 numbers that is not a tie is further from it than
    float64 can round (2^-33 relative), so rounding the float64 quotient is exact."""
    q = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale)))
    return torch.where(scale > 0, q, torch.zeros_like(q)).clamp(-127, 127)


def layernorm(x, w, b, eps):
    x = x.double()
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * w.double() + b.double()


def quantize_rows(x):
    """(codes, scales) in float64 of finite rows [M, K]."""
    x = x.double()
    s = scale_of(x.abs().amax(-1))
    return codes_of(x, s[:, None]), s


def gelu(x):
    return x * 0.5 * torch.erfc(-x / math.sqrt(2.0))


def rope(x, pos, table):
    """x [B, t, h, d] (any float type) at positions pos[t]; table float32 [2, max_pos, rot / 2]; float64, not rounded."""
    y = x.double().clone()
    half = table.shape[2]
    c, s = (table[i].double()[pos][None, :, None] for i in (0, 1))
    a, b = y[..., :half].clone(), y[..., half:2 * half].clone()
    y[..., :half] = a * c - b * s
    y[..., half:2 * half] = b * c + a * s
    return y


def block_values(rows, dtype):
    """What a full block [block, d] of `dtype` rows stands for: (codes, scale)."""
    x = rows.to(dtype).double()
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), torch.zeros_like(x)).amax()
    s = scale_of(amax)
    codes = codes_of(torch.where(finite, x, torch.zeros_like(x)), s)
    codes = torch.where(torch.isinf(x) & (s > 0), torch.sign(x) * 127, codes)
    return codes, s


class Cache:
    """Rows as they came (already rotated, `dtype`), and what an 8-bit cache of them holds."""

    def __init__(self, batch, heads, d, block, dtype):
        self.block, self.dtype = block, dtype
        self.k = torch.zeros(batch, heads, 0, d, dtype=dtype)
        self.v = torch.zeros(batch, heads, 0, d, dtype=dtype)

    def append(self, k, v, pos=None, table=None):
        """k, v [B, t, h, d]."""
        if table is not None:
            k = rope(k, pos, table).to(self.dtype)
        self.k = torch.cat([self.k, k.transpose(1, 2)], 2)
        self.v = torch.cat([self.v, v.transpose(1, 2)], 2)

    def rows(self, which):
        """(values float64 [B, h, n, d], codes of the full blocks, scales)."""
        x = self.k if which == "k" else self.v
        n = x.shape[2]
        full = n // self.block
        out, codes, scales = x.double().clone(), [], []
        for j in range(full):
            at = slice(j * self.block, (j + 1) * self.block)
            for b in range(x.shape[0]):
                for h in range(x.shape[1]):
                    c, s = block_values(x[b, h, at], self.dtype)
                    out[b, h, at] = c * s
                    codes.append(c)
                    scales.append(s)
        return out, codes, scales


def attention(q, k, v, pos0, mask=None):
    """q [B, t, heads, d], k / v float64 [B, kv_heads, n, d]; mask [B, n] or None.  float64 [B, t, heads, d]."""
    B, t, heads, d = q.shape
    share = heads // k.shape[1]
    out = torch.zeros(B, t, heads, d, dtype=torch.float64)
    n = k.shape[2]
    for b in range(B):
        for r in range(t):
            see = torch.arange(n) <= pos0 + r
            if mask is not None:
                see &= mask[b, :n] != 0
            if not see.any():
                continue
            for h in range(heads):
                s = (k[b, h // share][see] * q[b, r, h].double()).sum(1) / math.sqrt(d)
                p = torch.exp(s - s.max())
                out[b, r, h] = (p[:, None] * v[b, h // share][see]).sum(0) / p.sum()
    return out
