"""The operators of 4-bit weights and 8-bit rows that janis_b200 is measured on.

Both forms are microscaling ones: 32 values that lie together along a row share a scale that is a power of two (8 bits of exponent,
bias 127; 255 stands for NaN).  A row of activations holds e4m3 values (8 bits), a row of weights e2m1 values (4 bits, the lower half of
a byte first).  Rows are padded to multiples of 128 values with zeros of scale 1.  The scales of 128 rows x 128 values are one block of
512 bytes, [row % 32][row / 32][group of 32], and the blocks of a matrix are [row / 128][value / 128]; rows past the end have scale 1.
A group's scale is the smallest power of two 2^s with max |v| <= 448 * 2^s (6 * 2^s for weights); a group of zeros has scale 1.

* norm:     h += norm(res; w_post) on the float32 stream (res itself without w_post), y = norm(h; w_next), y in 8 bits.
            Returns the stream, the codes as the e4m3 values they are and the scales as the powers of two they are.
* product:  out[t, n] = sum_k x[t, k] W[n, k] of 8-bit rows and 4-bit weights, in bfloat16 or float32.
* gated:    the same with act(gate) * up behind it, gate and up rows of W alternating in groups of 8, the result in 8 bits again
            (what the next product takes): codes and scales as for the norm.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
GROUP, BLOCK = 32, 128
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)        # between them; a tie goes to the even code
MOST_NORM, MOST_WEIGHT, MOST_PRODUCT = 8192 * 2304, 73728 * 4608, 2048 * 4608 * 36864


def _norm(name, rows, width, res="bfloat16", post=True):
    c = {"op": "norm", "rows": rows, "width": width, "res": res, "post": post}
    return dict(c, name=name) if name else c


def _product(name, rows, n, k, out="bfloat16"):
    c = {"op": "product", "rows": rows, "n": n, "k": k, "out": out}
    return dict(c, name=name) if name else c


def _gated(name, rows, n, k, act="gelu"):
    c = {"op": "gated", "rows": rows, "n": n, "k": k, "act": act}
    return dict(c, name=name) if name else c


def listed():
    return [
        _norm("norm-1x2304", 1, 2304),                          # one user's token between two sublayers of the 2B model
        _norm("norm-64x4608-plain", 64, 4608, post=False),      # a server's batch, blocks without a norm after the sublayer
        _norm("norm-8192x2304", 8192, 2304),                    # a long prompt
        _norm("norm-333x1000-float", 333, 1000, "float32"),     # an odd prompt at a width that is no multiple of a group
        _product("product-1-qkv-2b", 1, 4096, 2304),            # one token's queries, keys and values: latency counts
        _product("product-8-down-2b", 8, 2304, 9216),           # a small batch through the long down projection
        _gated("gated-1-27b", 1, 73728, 4608),                  # one token through the largest matrix: bandwidth counts
        _product("product-13-odd-float", 13, 1000, 777, "float32"),     # odd sizes all round, kept in 32 bits
        _product("product-64-qkv-2b", 64, 4096, 2304),          # a server's batch
        _gated("gated-2048-2b", 2048, 18432, 2304),             # a usual prompt through gate and up
        _product("product-683-o-2b", 683, 2304, 2048),          # an odd prompt through the output projection
        _product("product-2048-down-27b", 2048, 4608, 36864),   # the largest: a prompt through the large down projection
    ]


def _spread(rng, lo, hi):
    """A whole number from [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "product", "product", "gated"])
    if op == "norm":
        width = _spread(rng, 32, 4608)
        if rng.random() < 0.5:
            width = (width + 127) // 128 * 128
        return _norm(None, _spread(rng, 1, min(8192, MOST_NORM // width)), width, rng.choice(["bfloat16", "float32"]), rng.random() < 0.6)
    rows = _spread(rng, 1, 16) if rng.random() < 0.5 else _spread(rng, 17, 4096)
    k = _spread(rng, 32, 36864)
    if rng.random() < 0.6:
        k = (k + 127) // 128 * 128
    n = _spread(rng, 16, max(16, min(73728, MOST_WEIGHT // k, MOST_PRODUCT // (k * rows))))
    if op == "gated":
        return _gated(None, rows, (n + 15) // 16 * 16, k, rng.choice(["gelu", "silu"]))
    return _product(None, rows, n, k, rng.choice(["bfloat16", "bfloat16", "float32"]))


# ---------------------------------------------------------------------------
# the two forms, with torch operations
# ---------------------------------------------------------------------------

def _padded(k):
    return (k + BLOCK - 1) // BLOCK * BLOCK


def _to_blocks(s):
    """Scale bytes [rows, groups], groups a multiple of 4 -> blocks [rows / 128, groups / 4, 512]."""
    r, g = s.shape
    full = torch.full((_padded(r), g), 127, dtype=torch.uint8, device=s.device)
    full[:r] = s
    return full.view(-1, 4, 32, g // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, g // 4, 512).contiguous()


def _from_blocks(b, rows):
    r, kb = b.shape[:2]
    return b.view(r, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, kb * 4)[:rows]


def _scaled(v, most):
    """(v / scale as [rows, padded / 32, 32], scale bytes): the smallest power of two that brings a group under `most`."""
    r, k = v.shape
    v = torch.nn.functional.pad(v, (0, _padded(k) - k)).view(r, -1, GROUP)
    big = v.abs().amax(-1)
    m, e = torch.frexp(big / most)                     # big / most = m 2^e with m in [1/2, 1)
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(big > 0, e.clamp(min=-127), torch.zeros_like(e))
    return torch.ldexp(v, -e[..., None]), (e + 127).to(torch.uint8)


def _to_mx8(v):
    """float32 rows -> (codes uint8 [rows, padded], blocks of scales)."""
    q, s = _scaled(v, 448.0)
    return q.flatten(1).to(torch.float8_e4m3fn).view(torch.uint8), _to_blocks(s)


def _to_mx4(w):
    q, s = _scaled(w, 6.0)
    q = q.flatten(1)
    a = q.abs()
    code = torch.zeros(a.shape, dtype=torch.uint8, device=w.device)
    for i, m in enumerate(MIDDLES):
        code += (a >= m) if i % 2 else (a > m)
    code += (q < 0).to(torch.uint8) * 8
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), _to_blocks(s)


def _mx_values(codes, blocks, rows):
    """The float32 values [rows, padded] that a matrix in either form stands for."""
    kp = blocks.shape[1] * BLOCK
    if codes.shape[1] == kp:
        v = codes.view(torch.float8_e4m3fn).to(torch.float32)
    else:
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=codes.device)
        v = table[torch.stack([codes & 15, codes >> 4], -1).flatten(1).to(torch.int32)]
    s = _from_blocks(blocks, rows).view(torch.float8_e8m0fnu).to(torch.float32)
    return (v.view(rows, -1, GROUP) * s[..., None]).view(rows, kp)


# ---------------------------------------------------------------------------
# a state, a pass
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    draw_ = lambda *shape: torch.randn(*shape, generator=g, device="cuda")   # noqa: E731
    t = case["rows"]
    if case["op"] == "norm":
        h = case["width"]
        feature = torch.exp(0.6 * draw_(h))                   # features of unlike size, as a trained stream has
        s = {"h": draw_(t, h) * feature, "res": (draw_(t, h) * feature).to(getattr(torch, case["res"])),
             "w_post": 1 + 0.1 * draw_(h) if case["post"] else None, "w_next": 1 + 0.1 * draw_(h)}
        width = h
        if t > 3:
            s["h"][1], s["res"][1] = 0, 0                     # a padding row
    else:
        n, k = case["n"], case["k"]
        x = draw_(t, k) * torch.exp(0.6 * draw_(k))
        if t > 3:
            x[1] = 0
        s = {}
        s["x"], s["x_scales"] = _to_mx8(x)
        s["w"], s["w_scales"] = _to_mx4(draw_(n, k) / math.sqrt(k))
        width = n // 2
    if case["op"] == "product":
        s["out"] = torch.zeros(t, n, dtype=getattr(torch, case["out"]), device="cuda")
    else:                                                     # the room for 8-bit rows
        s["codes"] = torch.zeros(t, _padded(width), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.full(((t + 127) // 128, _padded(width) // 128, 512), 127, dtype=torch.uint8, device="cuda")
    s["case"] = dict(case)
    return s


def _as_values(codes, scales):
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from janis_b200.kernels import ops
    c = s["case"]
    if c["op"] == "norm":
        y = ops.MxRows(s["codes"], s["scales"], c["rows"], c["width"])
        ops.add_rmsnorm(s["h"], s["res"], s["w_post"], EPS, s["w_next"], EPS, y)
        return dict(_as_values(s["codes"], s["scales"]), h=s["h"])
    x = ops.MxRows(s["x"], s["x_scales"], c["rows"], c["k"])
    w = ops.MxWeight(s["w"], s["w_scales"], c["n"], c["k"])
    if c["op"] == "product":
        return ops.linear_mx(x, w, s["out"])
    ops.linear_mx(x, w, ops.MxRows(s["codes"], s["scales"], c["rows"], c["n"] // 2),
                  ops.EPI_GATED_GELU if c["act"] == "gelu" else ops.EPI_GATED_SILU)
    return _as_values(s["codes"], s["scales"])


def _normed(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _run_plain(s):
    c = s["case"]
    if c["op"] == "norm":
        r = s["res"].to(torch.float32)
        s["h"] += r if s["w_post"] is None else _normed(r, s["w_post"])
        codes, scales = _to_mx8(_normed(s["h"], s["w_next"]))
        return dict(_as_values(codes, scales), h=s["h"])
    v = _mx_values(s["x"], s["x_scales"], c["rows"]) @ _mx_values(s["w"], s["w_scales"], c["n"]).T
    if c["op"] == "product":
        return v.to(s["out"].dtype)
    v = v.view(c["rows"], -1, 2, 8)
    gate, up = v[:, :, 0].flatten(1), v[:, :, 1].flatten(1)
    if c["act"] == "gelu":
        act = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    else:
        act = gate / (1 + torch.exp(-gate))
    return _as_values(*_to_mx8(act * up))


def work(case):
    t = case["rows"]
    if case["op"] == "norm":
        h = case["width"]
        return {"bytes": t * h * (8 + (2 if case["res"] == "bfloat16" else 4) + 1 + 1 / GROUP) + 4 * h * (2 if case["post"] else 1), "flops": 10 * t * h}
    n, k = case["n"], case["k"]
    size = n * k * (1 / 2 + 1 / GROUP) + t * k * (1 + 1 / GROUP)
    size += t * n * (2 if case["out"] == "bfloat16" else 4) if case["op"] == "product" else t * n / 2 * (1 + 1 / GROUP)
    return {"bytes": size, "flops": 2 * t * n * k}


# ---------------------------------------------------------------------------
# the definition in 64 bits, from the bytes
# ---------------------------------------------------------------------------

def _exact_values(codes, scales, rows, k, bits):
    """Values [rows, k] by the formats' definitions: sign, exponent and mantissa taken apart."""
    i = torch.arange(k, device=codes.device)
    code = codes[:rows, i].long() if bits == 8 else codes[:rows, i // 2].long() >> 4 * (i % 2) & 15
    digits, bias = (3, 7) if bits == 8 else (1, 1)
    e, m = code >> digits & (15 if bits == 8 else 3), (code & (1 << digits) - 1).double() / (1 << digits)
    v = torch.where(e > 0, 1 + m, m) * 2.0 ** (e.clamp(min=1) - bias).double()
    v = torch.where(code >> bits - 1 > 0, -v, v)
    r = torch.arange(rows, device=codes.device)[:, None]
    at = (r // 128 * scales.shape[1] + i // 128) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + i % 128 // 32
    return v * 2.0 ** (scales.flatten()[at].double() - 127)


def _exact_mx8(y):
    t, k = y.shape
    kp = (k + 127) // 128 * 128
    full = torch.zeros(t, kp, dtype=torch.float64, device=y.device)
    full[:, :k] = y
    full = full.view(t, kp // 32, 32)
    big = full.abs().amax(-1, keepdim=True)
    s = torch.where(big > 0, torch.ceil(torch.log2(torch.where(big > 0, big, 1.0) / 448)), 0.0)
    s = torch.where(big > 448 * 2.0 ** s, s + 1, s)
    s = torch.where((big > 0) & (big <= 448 * 2.0 ** (s - 1)), s - 1, s)
    q = full / 2.0 ** s
    step = 2.0 ** (torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.round(q / step) * step                     # (ties go to the even one, as in the format's own rounding)
    scales = torch.ones((t + 127) // 128 * (kp // 128) * 512, dtype=torch.float64, device=y.device)
    r, g = torch.arange(t, device=y.device)[:, None], torch.arange(kp // 32, device=y.device)
    scales[(r // 128 * (kp // 128) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4] = 2.0 ** s[..., 0]
    return {"codes": q.view(t, kp), "scales": scales.view(-1, kp // 128, 512)}


def exact(case, seed):
    s, t = prepare(case, seed), case["rows"]
    if case["op"] == "norm":
        root = lambda v: torch.sqrt(torch.sum(v ** 2, -1, keepdim=True) / case["width"] + EPS)     # noqa: E731
        r = s["res"].double()
        h = s["h"].double() + (r if s["w_post"] is None else r / root(r) * s["w_post"].double())
        return dict(_exact_mx8(h / root(h) * s["w_next"].double()), h=h)
    n, k = case["n"], case["k"]
    x, w = _exact_values(s["x"], s["x_scales"], t, k, 8), _exact_values(s["w"], s["w_scales"], n, k, 4)
    v = torch.einsum("tk,nk->tn", x, w)
    if case["op"] == "product":
        return v
    j = torch.arange(n // 2, device=v.device)
    gate, up = v[:, j // 8 * 16 + j % 8], v[:, j // 8 * 16 + 8 + j % 8]
    if case["act"] == "gelu":
        return _exact_mx8(gate / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up)
    return _exact_mx8(gate * torch.sigmoid(gate) * up)
