"""The operators of 8-bit serving, as they are measured: a linear layer in 8-bit integers (quantised tokens, quantised weight
channels), the key/value cache held in 8 bits with one scale for each block of tokens and head, and the attention that reads it.

``run`` computes them in plain torch (``own = False``) or through ``block_transformer_amd.ops`` (``own = True``); ``exact`` gives the same
outputs from the definitions in 64 bits.

Definitions
  quantisation   s = fl32(max |x| / 127);  code = clamp(round_half_even(x / s), -127, 127), the quotient taken exactly
  linear         y[m, n] = act(sum_k cx[m, k] cw[n, k] * sx[m] * sw[n] + bias[n]) + residual[m, n];  cx, sx: the row x[m] (its LayerNorm if
                 one is given) quantised with one scale per token; cw, sw: the weight, one scale per output channel
  cache          rows [0, n): the rows of every full block of ``block`` tokens as codes with one scale per (sequence, head, block), the
                 rows of the open block as they came.  K codes [B, H, n_max, d], V codes [B, H, n_max / block, d, block], the open block's
                 rows K [B, H, block, d] and V [B, H, d, block]
  attention      softmax(q k^T / sqrt(d)) v over the rows j <= pos0 + t with mask[b, j] != 0; zeros where none is left
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def _linear(m, n, k, dtype="bf16", ln=False, act="none", residual=False):
    return {"op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "ln": ln, "act": act, "residual": residual}


def _append(b, q_len, pos0, heads, kv_heads, d, rot, block=16, dtype="bf16"):
    return {"op": "append", "b": b, "q_len": q_len, "pos0": pos0, "heads": heads, "kv_heads": kv_heads, "d": d, "rot": rot,
            "block": block, "dtype": dtype}


def _attention(b, q_len, n, heads, kv_heads, d, block=16, dtype="bf16", mask=False):
    return {"op": "attention", "b": b, "q_len": q_len, "n": n, "heads": heads, "kv_heads": kv_heads, "d": d, "block": block,
            "dtype": dtype, "mask": mask}


def listed():
    named = {
        # one sequence decodes a token: LayerNorm and the fused query/key/value projection of the 1.2B stacks
        "linear one token": _linear(1, 6144, 2048, ln=True),
        # a ragged batch of the fp32 parity path, odd in every size
        "linear odd fp32": _linear(77, 1001, 515, "f32", residual=True),
        # prefill, LayerNorm and h -> 4h with its GELU: the largest product of a layer
        "linear prefill h to 4h": _linear(8192, 8192, 2048, ln=True, act="gelu"),
        # a decode step of a large batch, 4h -> h onto the residual stream
        "linear step 4h to h": _linear(4096, 2048, 8192, residual=True),
        # a decode step in which every sequence fills its block
        "append step": _append(256, 1, 511, 16, 16, 128, 32),
        # prefill of a batch of prompts whose last block stays open
        "append prefill": _append(32, 509, 0, 16, 16, 128, 32),
        # a chunk that ends its block, shared heads, the fp32 path
        "append chunk fp32": _append(5, 45, 67, 8, 2, 64, 64, dtype="f32"),
        # the first steps of one sequence: latency
        "attention short": _attention(1, 1, 21, 16, 16, 128),
        # a decode step of a middling batch over a 2048-token prompt (512 blocks) and what follows it
        "attention step": _attention(256, 1, 543, 16, 16, 128),
        # few sequences with a long context and shared heads, padded on the left
        "attention long": _attention(4, 1, 32773, 32, 4, 128, block=32, mask=True),
        # the largest batch
        "attention large batch": _attention(1024, 1, 543, 16, 16, 128),
        # several query rows at once, fp32, padded, one sequence with nothing left to see
        "attention rows fp32": _attention(7, 5, 1037, 12, 12, 64, block=64, dtype="f32", mask=True),
    }
    return [dict(case, name=name) for name, case in named.items()]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, unit):
    """Spread over the logarithm; two in three are multiples of `unit`, as model sizes are, the others any number."""
    v = _log(rng, low, high)
    return max(unit, v // unit * unit) if rng.random() < 2 / 3 else v


def draw(rng):
    op = rng.choice(("linear", "append", "attention"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if op == "linear":
        while True:
            m, n, k = _log(rng, 1, 8192), _size(rng, 16, 8192, 64), _size(rng, 32, 8192, 64)
            if m * n * k <= 8192 * 8192 * 2048:
                break
        return _linear(m, n, k, dtype, dtype == "bf16" and rng.random() < 0.5, rng.choice(("none", "gelu")), rng.random() < 0.5)
    d = rng.choice((32, 64, 128))
    block = rng.choice((16, 32, 64))
    kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 8)) if kv_heads <= 4 else kv_heads
    if op == "append":
        rot = rng.choice((d // 4, d))
        while True:
            b, q_len = _log(rng, 1, 256), rng.choice((1, _log(rng, 2, 512)))
            if b * q_len <= 32 * 509 and b * q_len * (heads + 2 * kv_heads) * d <= 32 * 509 * 48 * 128:
                break
        # the pass can be run again on its own state: it starts a block, ends one, or stays inside one
        pos0 = rng.choice((0, block * rng.randrange(1, 20), block * 20 - q_len % block, block * 20))
        return _append(b, q_len, pos0, heads, kv_heads, d, rot, block, dtype)
    while True:
        b, n = _log(rng, 1, 1024), _log(rng, 1, 32768)
        q_len = min(n, rng.choice((1, 1, 1, rng.randrange(2, 9))))
        if b * n * kv_heads * d <= 1024 * 543 * 16 * 128 // (2 if dtype == "f32" else 1) and b * n * heads * q_len <= 1 << 28:
            break
    return _attention(b, q_len, n, heads, kv_heads, d, block, dtype, rng.random() < 0.4)


# --------------------------------------------------------------------------------------------------------------- inputs
def _positions(n, rot):
    """cos and sin of the rotary angles, [2, n, rot / 2], rounded once to fp32."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    angle = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()]).float().contiguous()


def _codes(shape, g):
    return (torch.randn(shape, generator=g, device=DEV) * 36).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def rnd(*shape, scale=1.0, to=t):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(to)

    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # rows of codes are kept in multiples of 16 bytes, zero behind the last
        kp = (k + 15) // 16 * 16
        w = torch.zeros(n, kp, dtype=torch.int8, device=DEV)
        w[:, :k] = _codes((n, k), g)
        s = (torch.rand(n, generator=g, device=DEV) * 0.5 + 0.75) * (3.5 / 127 * k ** -0.5)
        return {"case": case, "x": rnd(m, k), "w": w, "w_scale": s, "bias": rnd(n, scale=0.5),
                "residual": rnd(m, n) if case["residual"] else None,
                "ln": (rnd(k, scale=0.1) + 1, rnd(k, scale=0.1)) if case["ln"] else None}
    b, q_len, heads, hk, d, block = (case[x] for x in ("b", "q_len", "heads", "kv_heads", "d", "block"))
    pos0 = case["pos0"] if case["op"] == "append" else case["n"] - q_len
    n = pos0 + q_len
    blocks = n // block + 1
    scale = lambda: (torch.rand(b, hk, blocks, generator=g, device=DEV) * 0.4 + 0.8) * (3.0 / 127)  # noqa: E731
    state = {"case": case, "pos0": pos0,
             "cache": (_codes((b, hk, blocks * block, d), g), _codes((b, hk, blocks, d, block), g), scale(), scale(),
                       rnd(b, hk, block, d), rnd(b, hk, d, block))}
    if case["op"] == "append":
        # one fused projection row per token: the heads' queries, then the keys, then the values
        rows = rnd(b, q_len, heads + 2 * hk, d)
        state |= {"q": rows[:, :, :heads], "k": rows[:, :, heads:heads + hk], "v": rows[:, :, heads + hk:],
                  "rope": _positions(n, case["rot"])}
    else:
        state["q"] = rnd(b, q_len, heads, d, scale=2.0)
        state["mask"] = None
        if case["mask"]:
            first = torch.randint(0, max(1, n // 4), (b, 1), generator=g, device=DEV)
            if b > 1:
                first[b // 2] = n      # a sequence with nothing to see
            state["mask"] = (torch.arange(n, device=DEV) >= first).to(torch.uint8)
    return state


# ------------------------------------------------------------------------------------------------------- the plain form
def _quantise(x, dims):
    """Codes and scales of fp32 `x`, one scale over `dims`; the quotient in 64 bits, where a border is not missed."""
    s = x.abs().amax(dims, keepdim=True) / 127
    q = (x.double() / torch.where(s > 0, s, torch.ones_like(s)).double()).round().clamp(-127, 127).float()
    return q, s


def _plain_linear(s):
    x = s["x"].float()
    if s["ln"] is not None:
        x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-5) * s["ln"][0].float() + s["ln"][1].float()
    q, sx = _quantise(x, -1)
    y = (q @ s["w"][:, :x.shape[1]].float().T) * (sx * s["w_scale"]) + s["bias"].float()
    if s["case"]["act"] == "gelu":
        y = y * 0.5 * (1 + torch.erf(y * 0.5 ** 0.5))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _rotated(x, table, pos0):
    """Rotary positions of rows [b, t, h, d]; the products and their sum in 64 bits, rounded once, since codes follow from them."""
    half = table.shape[-1]
    cos, sin = table[:, pos0:pos0 + x.shape[1], None].double()
    a, b, rest = x[..., :half].double(), x[..., half:2 * half].double(), x[..., 2 * half:]
    return torch.cat([(a * cos - b * sin).to(x.dtype), (b * cos + a * sin).to(x.dtype), rest], -1)


def _plain_append(s):
    block, pos0 = s["case"]["block"], s["pos0"]
    kc, vc, ks, vs, kt, vt = s["cache"]
    n, dtype = pos0 + s["q"].shape[1], kt.dtype
    first = pos0 // block * block
    closed = n // block * block
    k = torch.cat([kt[:, :, :pos0 - first], _rotated(s["k"], s["rope"], pos0).transpose(1, 2)], 2)
    v = torch.cat([vt[..., :pos0 - first].transpose(2, 3), s["v"].transpose(1, 2)], 2)
    b, h, _, d = k.shape
    if closed > first:
        at = slice(first // block, closed // block)
        q, sc = _quantise(k[:, :, :closed - first].float().reshape(b, h, -1, block, d), (3, 4))
        kc[:, :, first:closed] = q.reshape(b, h, -1, d).to(torch.int8)
        ks[:, :, at] = sc[..., 0, 0]
        q, sc = _quantise(v[:, :, :closed - first].float().reshape(b, h, -1, block, d), (3, 4))
        vc[:, :, at] = q.transpose(3, 4).to(torch.int8)
        vs[:, :, at] = sc[..., 0, 0]
    if n > closed:
        kt[:, :, :n - max(first, closed)] = k[:, :, max(first, closed) - first:]
        vt[..., :n - max(first, closed)] = v[:, :, max(first, closed) - first:].transpose(2, 3)
    k, v = _plain_rows(s["cache"], n, first)
    return _rotated(s["q"], s["rope"], pos0), k.to(dtype), v.to(dtype)


def _plain_rows(cache, n, first=0):
    """The rows [first, n) that a cache stands for, in fp32; `first` starts a block."""
    kc, vc, ks, vs, kt, vt = cache
    block, d = kt.shape[2], kt.shape[3]
    b, h = kc.shape[:2]
    closed = n // block * block
    at = slice(first // block, closed // block)
    k = kc[:, :, first:closed].reshape(b, h, -1, block, d).float() * ks[:, :, at, None, None]
    v = (vc[:, :, at].float() * vs[:, :, at, None, None]).transpose(3, 4)
    return (torch.cat([k.reshape(b, h, -1, d), kt[:, :, :n - closed].float()], 2),
            torch.cat([v.reshape(b, h, -1, d), vt[..., :n - closed].transpose(2, 3).float()], 2))


def _plain_attention(s):
    q, pos0 = s["q"], s["pos0"]
    b, q_len, heads, d = q.shape
    n = pos0 + q_len
    k, v = _plain_rows(s["cache"], n)
    hk = k.shape[1]
    x = q.float().reshape(b, q_len, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = torch.matmul(x, k.transpose(2, 3).contiguous()).reshape(b, hk, heads // hk, q_len, n) * d ** -0.5
    seen = torch.arange(n, device=q.device) <= torch.arange(pos0, n, device=q.device)[:, None]
    if s["mask"] is not None:
        seen = seen & (s["mask"][:, None, None, None] != 0)
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    y = torch.matmul(p.reshape(b, hk, -1, n), v).reshape(b, hk, heads // hk, q_len, d)
    return y.permute(0, 3, 1, 2, 4).reshape(b, q_len, heads, d).to(q.dtype)


# --------------------------------------------------------------------------------------------------------------- a pass
def _own(s):
    from block_transformer_amd import ops

    op = s["case"]["op"]
    if op == "linear":
        codes = ops.quantize_rows(s["x"], *(s["ln"] or ()))
        return ops.linear_q8(codes, (s["w"], s["w_scale"]), s["bias"], s["residual"], act=s["case"]["act"], dtype=s["x"].dtype)
    if op == "append":
        q = ops.kv8_append(s["cache"], s["q"], s["k"], s["v"], s["pos0"], rope=s["rope"])
        block = s["case"]["block"]
        k, v = ops.kv8_read(s["cache"], s["pos0"] + s["q"].shape[1], first=s["pos0"] // block * block)
        return q, k, v
    return ops.attention_kv8(s["q"], s["cache"], s["pos0"], mask=s["mask"])


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "append": _plain_append, "attention": _plain_attention}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        floats = m * k + n + m * n * (2 if case["residual"] else 1) + (2 * k if case["ln"] else 0)
        return {"bytes": floats * size + n * k + 4 * n, "flops": 2 * m * n * k}
    b, q_len, heads, hk, d, block = (case[x] for x in ("b", "q_len", "heads", "kv_heads", "d", "block"))
    if case["op"] == "append":
        pos0 = case["pos0"]
        n, first = pos0 + q_len, pos0 // block * block
        closed = max(first, n // block * block)
        rows = b * (2 * q_len * heads + 2 * hk * q_len)                     # queries in and out, keys and values in
        rows += 2 * b * hk * ((pos0 - first if closed > first else 0) + n - max(closed, pos0))   # the open block: rows taken up, rows left
        rows += 2 * b * hk * (n - first)                                    # read back
        codes = 2 * b * hk * ((closed - first) * d + (closed - first) // block * 4)
        return {"bytes": rows * d * size + codes + q_len * case["rot"] * 4, "flops": 3 * b * q_len * (heads + hk) * case["rot"]}
    n = case["n"]
    closed = n // block * block
    cache = 2 * b * hk * (closed * d + closed // block * 4 + (n - closed) * d * size)
    return {"bytes": cache + 2 * b * q_len * heads * d * size + (b * n if case["mask"] else 0), "flops": 4 * b * heads * q_len * n * d}


# ---------------------------------------------------------------------------------------------------------- in 64 bits
def _exact_codes(x, axes):
    """What quantising stands for, from its definition: codes times scale, in 64 bits (the scale itself is an fp32 number)."""
    step = (x.abs().amax(axes, keepdim=True).float() / 127).double()
    whole = torch.round(x / step.clamp_min(1e-300))
    return torch.clamp(whole, -127.0, 127.0) * step


def _exact_turn(x, positions, rot):
    """Rotary positions by their angles' fp32 cosines and sines, in 64 bits."""
    angle = positions.double()[:, None] / 10000.0 ** (torch.arange(rot // 2, dtype=torch.float64, device=DEV) * 2 / rot)
    c, s = (f(angle).float().double()[None, :, None, :] for f in (torch.cos, torch.sin))
    x = x.double()
    y = x.clone()
    y[..., :rot // 2] = x[..., :rot // 2] * c - x[..., rot // 2:rot] * s
    y[..., rot // 2:rot] = x[..., rot // 2:rot] * c + x[..., :rot // 2] * s
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        if case["ln"]:
            gain, shift = (w.double() for w in s["ln"])
            x = (x - x.mean(1, keepdim=True)) / (x.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * gain + shift
        w = s["w"][:, :case["k"]].double() * s["w_scale"].double()[:, None]
        y = torch.mm(_exact_codes(x, 1), w.t().contiguous()) + s["bias"].double()
        if case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        return y if s["residual"] is None else y + s["residual"].double()
    kc, vc, ks, vs, kt, vt = s["cache"]
    block, d, hk, q_len = case["block"], case["d"], case["kv_heads"], case["q_len"]
    n = s["pos0"] + q_len
    whole = n // block          # blocks that are full
    if case["op"] == "append":
        place = torch.arange(s["pos0"], n, device=DEV)
        old = s["pos0"] % block
        out = []
        for new, tail in ((_exact_turn(s["k"], place, case["rot"]).to(kt.dtype), kt), (s["v"], vt.transpose(2, 3))):
            rows = torch.cat([tail[:, :, :old].double(), new.double().permute(0, 2, 1, 3)], 2)
            pieces = [_exact_codes(p, (2, 3)) if p.shape[2] == block else p for p in rows.split(block, 2)]
            out.append(torch.cat(pieces, 2))
        return _exact_turn(s["q"], place, case["rot"]), out[0], out[1]
    y = torch.zeros(case["b"], q_len, case["heads"], d, dtype=torch.float64, device=DEV)
    share = case["heads"] // hk
    step = max(1, (1 << 28) // (hk * n * (d + share * q_len)))
    for at in range(0, case["b"], step):
        part = slice(at, min(case["b"], at + step))
        k = kc[part, :, :whole * block].double() * ks[part, :, :whole].double().repeat_interleave(block, 2)[..., None]
        v = (vc[part, :, :whole].double() * vs[part, :, :whole, None, None].double()).permute(0, 1, 2, 4, 3).flatten(2, 3)
        k = torch.cat([k, kt[part, :, :n - whole * block].double()], 2)
        v = torch.cat([v, vt[part, :, :, :n - whole * block].double().transpose(2, 3)], 2)
        for h in range(hk):
            q = s["q"][part, :, h * share:(h + 1) * share].double().flatten(1, 2)
            logit = torch.bmm(q, k[:, h].transpose(1, 2).contiguous()) / math.sqrt(d)
            last = torch.arange(q_len, device=DEV).repeat_interleave(share) + s["pos0"]
            hidden = (torch.arange(n, device=DEV)[None, :] > last[:, None])[None]
            if s["mask"] is not None:
                hidden = hidden | (s["mask"][part] == 0)[:, None, :]
            p = torch.softmax(logit.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0)
            y[part, :, h * share:(h + 1) * share] = torch.bmm(p, v[:, h].contiguous()).unflatten(1, (q_len, share))
    return y
