"""8-bit rows and 4-bit weights: both forms, the operators that leave them, their products, and Gemma2 on them.

The oracle is `kernel_refs.quantised`, the formats' definition in 64 bits, and 64-bit sums of the values that the bytes stand for.

What is exact is compared bit for bit: a group's largest magnitude is one of its values, the scale follows from its bits, the division
by a power of two is exact, and one rounding to the code remains.  Products of two codes are exact in a float, and so are their scales;
what rounds is the addition of 32 products at a time (one addition a group, K / 32 of them, and at most 8 partial sums and the
conversion), each within 2^-23 of the sum of magnitudes so far even where it truncates: (K / 32 + 40) 2^-23 sum |x w|.
Norms: H additions in a block of 256 threads, ceil(H / 256) in a thread and 13 behind, then about 8 roundings of 2^-24 each; half of the
relative error of a mean of squares goes into a root: (ceil(H / 256) + 20) 2^-24 on each norm.
"""
from __future__ import annotations

import math

import pytest
import torch

from tests import kernel_refs as R
from tests.conftest import BF16_MODEL_TOL, TINY, plain_logits, random_tokens
from tests.helpers import run_in_pieces, run_requests

GPU = pytest.mark.gpu
E4M3, E2M1 = (448.0, 3, -6), (6.0, 1, 0)
INF, NAN = float("inf"), float("nan")


def ops():
    from janis_b200.kernels import ops as o
    return o


def rnd(*shape, seed=0, device="cuda"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(device)


def scale_rows(m, rows=None):
    """The scale bytes [rows, groups] out of their blocks."""
    r, kb = m.scales.shape[:2]
    return m.scales.view(r, kb, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(r * 128, kb * 4)[:m.rows if rows is None else rows]


def powers(m):
    """Its scales as the powers of two they are."""
    s = scale_rows(m)
    return torch.ldexp(torch.ones(s.shape, dtype=torch.float64, device=s.device), s.int() - 127)


def code_values(m):
    """The values of the codes without their scales, [rows, padded]."""
    if m.bits == 8:
        return m.codes.view(torch.float8_e4m3fn).double()
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=m.codes.device)
    c = torch.stack([m.codes & 15, m.codes >> 4], -1).flatten(1).long()
    return torch.where(c > 7, -table[c & 7], table[c & 7])


def stands_for(m):
    """The values of a matrix in 64 bits, [rows, width]."""
    s = scale_rows(m).double()
    s = torch.where(s == 255, torch.full_like(s, NAN), powers(m))
    return (code_values(m).view(m.rows, -1, 32) * s[..., None]).flatten(1)[:, :m.width]


def check_exact(m, v, form, what):
    """Codes and scales of `m` are those of the values v."""
    _, q, s = R.quantised(v.double().cpu(), *form)
    got_s = scale_rows(m).cpu().double()
    want_s = torch.where(torch.isnan(s), torch.full_like(s, 255.0), torch.log2(s) + 127)
    assert torch.equal(got_s, want_s), f"{what}: scales differ, first at {(got_s != want_s).nonzero()[0].tolist()}"
    got_q = code_values(m).cpu()
    assert torch.equal(got_q, q), f"{what}: codes differ, first at {(got_q != q).nonzero()[0].tolist()}"


def hard_rows(k, dtype):
    """Rows with what formats get wrong: zeros, ties, the largest value and a little over it, subnormals, infinities, NaN."""
    x = rnd(9, k, seed=3, device="cpu")
    x[0] = 0
    x[1] *= 2.0 ** torch.arange(k).remainder(40).sub(20)
    x[2, 0::2], x[2, 1::2] = 448.0, -449.0
    x[3, 0::2], x[3, 1::2] = 6.0, 6.03125
    x[4] = torch.arange(k) * 0.0625 - 2
    x[5] *= 1e-38
    x[6] = x[6].abs() * 3e38 / x[6].abs().max()
    x[7, k // 2], x[7, 0] = INF, -2.0
    x[8, k - 1] = NAN
    return x.to(dtype)


# ---------------------------------------------------------------------------
# the two forms
# ---------------------------------------------------------------------------

def test_the_oracle_rounds_to_the_nearest_value():
    for limit, digits, low in (E4M3, E2M1):
        top = int(math.floor(math.log2(limit)))
        codes = sorted({0.0} | {(1 + m / 2 ** digits) * 2.0 ** e for e in range(low, top + 1) for m in range(2 ** digits)}
                       | {m * 2.0 ** (low - digits) for m in range(2 ** digits)})
        codes = torch.tensor([c for c in codes if c <= limit], dtype=torch.float64)
        v = rnd(20, 64, device="cpu").double()
        val, q, s = R.quantised(v, limit, digits, low)
        big = v.view(20, 2, 32).abs().amax(-1)
        assert (big <= limit * s[:, :2]).all() and (big > limit * s[:, :2] / 2).all()
        x = (v.view(20, 2, 32) / s[:, :2, None]).flatten(1)
        assert torch.equal((x.abs()[..., None] - codes).abs().amin(-1), (x - q[:, :64]).abs())
        assert torch.equal(val, (q[:, :64].view(20, 2, 32) * s[:, :2, None]).flatten(1))


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 31, 32, 33, 128, 130, 777, 4608])
def test_rows_and_weights_are_the_formats_own(k, dtype):
    o = ops()
    x = hard_rows(k, dtype)
    for make, form in ((lambda v: o.mx_rows(v, o.MxRows.empty(*v.shape)), E4M3), (o.mx_weight, E2M1)):
        m = make(x.cuda())
        check_exact(m, x, form, f"{type(m).__name__} of {k} {dtype}")
        want = stands_for(m).float()
        assert torch.equal(torch.nan_to_num(m.values(), 7.0, 8.0, 9.0), torch.nan_to_num(want, 7.0, 8.0, 9.0))
        half = m.values(torch.empty(m.shape, dtype=torch.bfloat16, device="cuda"))
        assert torch.equal(torch.nan_to_num(half, 7.0, 8.0, 9.0), torch.nan_to_num(want.bfloat16(), 7.0, 8.0, 9.0))


@GPU
@pytest.mark.parametrize("rows", [1, 127, 128, 129, 300])
def test_scales_of_many_rows_and_padding_over_old_values(rows):
    o = ops()
    x = rnd(rows, 200, seed=rows) * torch.exp2(rnd(rows, 1, seed=rows + 1) * 5)
    m = o.MxRows.empty(rows, 200)
    m.codes.fill_(77)
    m.scales.fill_(200)
    o.mx_rows(x, m)
    check_exact(m, x, E4M3, f"{rows} rows")


@GPU
def test_the_first_rows_of_a_weight():
    o = ops()
    w = o.mx_weight(rnd(300, 96))
    for n in (1, 128, 130, 300):
        assert torch.equal(w[:n].values(), w.values()[:n])
    with pytest.raises(IndexError):
        w[1:]


# ---------------------------------------------------------------------------
# norms and gated activation
# ---------------------------------------------------------------------------

def check_near(m, y, err, what):
    """`m` holds the values y, each known to a relative error `err`: half a step of a code (2^-4 of the value, 2^-10 of the scale
    below the normal codes), and the scale is that of a largest magnitude within the error."""
    y = y.double().cpu()
    rows, k = y.shape
    pad = torch.zeros(rows, -(-k // 128) * 128, dtype=torch.float64)
    pad[:, :k] = y
    s = powers(m).cpu()
    big = pad.view(rows, -1, 32).abs().amax(-1)
    some = big > 0
    assert torch.equal(s[~some], torch.ones_like(s[~some])), f"{what}: the scale of a group of zeros is 1"
    assert (big * (1 - err) <= 448 * s)[some].all() and (big * (1 + err) >= 224 * s)[some].all(), f"{what}: scales"
    step = torch.maximum(pad.abs() * 2.0 ** -4, (2.0 ** -10 * s)[..., None].expand(-1, -1, 32).flatten(1))
    got = (code_values(m).cpu().view(rows, -1, 32) * s[..., None]).flatten(1)
    over = ((got - pad).abs() - step * (1 + err) - pad.abs() * err).max().item()
    assert over <= 0, f"{what}: a value is {over:.3e} off more than its rounding"


def norm_error(h):
    return (math.ceil(h / 256) + 20) * 2.0 ** -24


@GPU
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("res", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,h", [(1, 8), (1, 2304), (3, 33), (5, 4608), (130, 1000), (64, 36), (2, 9216), (2, 20000), (160, 4607),
                                    (800, 1001)])
def test_norm_with_the_residuals_addition(rows, h, res, post):
    o = ops()
    x, r = rnd(rows, h, seed=1) * torch.exp(rnd(h, seed=2)), (rnd(rows, h, seed=3) * 2).to(res)
    wp, wn = 1 + 0.1 * rnd(h, seed=4), 1 + 0.1 * rnd(h, seed=5)
    if rows > 1:
        x[1], r[1] = 0, 0
    got_h, out = x.clone(), o.MxRows.empty(rows, h)
    out.codes.fill_(1)
    o.add_rmsnorm(got_h, r, wp if post else None, 1e-6, wn, 1e-5, out)
    add = R._norm(r, wp, 1e-6) if post else r.double()
    want = x.double() + add
    err = norm_error(h)
    assert ((got_h.double() - want).abs() <= 2.0 ** -23 * want.abs() + 2 * err * add.abs() + 1e-30).all()
    # the second norm is held to the stream that was stored
    check_near(out, R._norm(got_h, wn, 1e-5), 2 * err, f"{rows} x {h}")
    kp = out.codes.shape[1]
    assert not out.codes[:, h:kp].any()


@GPU
def test_norm_of_partial_sums_and_of_gathered_rows():
    o = ops()
    rows, h = 6, 264
    x, parts, w = rnd(rows, h, seed=1), rnd(3, rows, h, seed=2).bfloat16(), 1 + 0.1 * rnd(h, seed=3)
    got, out = x.clone(), o.MxRows.empty(rows, h)
    o.add_rmsnorm(got, parts, w, 1e-6, w, 1e-6, out, n_part=3)
    want = x.double() + R._norm(parts.double().sum(0), w, 1e-6)
    assert ((got.double() - want).abs() <= 4 * norm_error(h) * (want.abs() + 4)).all()
    check_near(out, R._norm(got, w, 1e-6), 2 * norm_error(h), "partial sums")
    at = torch.tensor([5, 0, 3, 3], dtype=torch.int32, device="cuda")
    y = o.MxRows.empty(4, h)
    o.rmsnorm(x, w, 1e-6, y, at)
    check_near(y, R._norm(x[at.long()], w, 1e-6), 2 * norm_error(h), "gathered")
    whole = o.MxRows.empty(rows, h)
    o.rmsnorm(x, w, 1e-6, whole)
    assert torch.equal(whole.codes[5], y.codes[0]) and torch.equal(whole.codes[3], y.codes[2])


@GPU
def test_a_row_that_is_not_finite_spoils_itself_alone():
    o = ops()
    x = rnd(4, 256)
    x[1, 7], x[2, 9] = NAN, INF
    w, out = torch.ones(256, device="cuda"), o.MxRows.empty(4, 256)
    o.rmsnorm(x, w, 1e-6, out)
    v = out.values()
    # x / inf is 0 but where inf / inf is NaN, which takes its group along
    assert torch.isnan(v[1]).all() and torch.isnan(v[2, :32]).all() and not v[2, 32:].any()
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[3]).all()


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 40), (130, 264), (7, 9216)])
def test_gated_activation_into_rows(rows, cols, act, dtype):
    o = ops()
    gu = (rnd(rows, 2 * cols, seed=cols) * 3).to(dtype)
    out = o.MxRows.empty(rows, cols)
    out.codes.fill_(3)
    o.gated_act(gu, out, act, limit=2.5, alpha=1.702, up_add=1.0)
    g, u = gu.double().view(rows, cols // 8, 2, 8).unbind(2)
    g, u = g.reshape(rows, cols), u.reshape(rows, cols)
    want = R._clamped(g, u, 2.5, 1.702, 1.0) if act == 2 else R._act(g, act) * u
    # tanhf and expf are within 2 units in the last place; 1 + tanh loses up to its value near -1, where the result is a
    # small share of |g u|: that share is allowed for as an absolute error
    err = 2.0 ** -20
    s = powers(out).cpu()
    pad = torch.zeros(rows, out.codes.shape[1], dtype=torch.float64)
    pad[:, :cols] = want.cpu()
    slack = torch.zeros_like(pad)
    slack[:, :cols] = (g * u).abs().cpu() * 2.0 ** -22 + 2.0 ** -22
    step = torch.maximum(pad.abs() * 2.0 ** -4, (2.0 ** -10 * s)[..., None].expand(-1, -1, 32).flatten(1))
    got = (code_values(out).cpu().view(rows, -1, 32) * s[..., None]).flatten(1)
    assert ((got - pad).abs() <= step * (1 + err) + pad.abs() * err + slack).all()
    assert not out.codes[:, cols:].any()


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

def operands(t, n, k, seed=0):
    o = ops()
    x = rnd(t, k, seed=seed) * torch.exp(rnd(k, seed=seed + 1))
    if t > 3:
        x[2] = 0
    w = rnd(n, k, seed=seed + 2) * torch.exp(rnd(n, 1, seed=seed + 3)) / math.sqrt(k)
    return o.mx_rows(x, o.MxRows.empty(t, k)), o.mx_weight(w)


def product_error(x, w):
    """The allowance of the module's text for every sum."""
    return (x.width / 32 + 40) * 2.0 ** -23 * (stands_for(x).abs() @ stands_for(w).abs().T)


def check_product(t, n, k, dtype, seed=0):
    o = ops()
    x, w = operands(t, n, k, seed)
    out = torch.full((t, n), NAN, dtype=dtype, device="cuda")
    o.linear_mx(x, w, out)
    want = stands_for(x) @ stands_for(w).T
    tol = product_error(x, w) + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0)
    off = ((out.double() - want).abs() - tol).max().item()
    assert off <= 0, f"{t} x {n} x {k} {dtype}: {off:.3e} over the allowance"


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 64, 127, 128, 129, 255, 256, 257, 600])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 32), (130, 96), (200, 777), (1000, 2048)])
def test_product(t, n, k, dtype):
    check_product(t, n, k, dtype, seed=t)


@GPU
@pytest.mark.parametrize("t,n,k", [(1, 4096, 2304), (3, 2304, 9216), (8, 2304, 2048), (1, 73728, 512), (2, 128, 36864), (33, 4100, 1152),
                                   (683, 2304, 2048), (1500, 520, 384), (2048, 4096, 2304), (4097, 256, 256)])
def test_product_at_larger_sizes(t, n, k):
    check_product(t, n, k, torch.float32)
    check_product(t, n, k, torch.bfloat16, seed=9)


@GPU
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, "rows"])
@pytest.mark.parametrize("epi", [1, 3, 4])
@pytest.mark.parametrize("t,n,k", [(1, 16, 32), (1, 18432, 256), (5, 144, 200), (16, 4608, 2304), (70, 272, 130), (300, 512, 640), (1030, 1040, 512)])
def test_gated_product(t, n, k, epi, dtype):
    o = ops()
    x, w = operands(t, n, k, seed=n)
    three = dict(limit=1.5, alpha=1.702, up_add=1.0) if epi == 4 else {}
    v = stands_for(x) @ stands_for(w).T
    off = product_error(x, w).view(t, n // 16, 2, 8)
    g, u = v.view(t, n // 16, 2, 8).unbind(2)
    g, u, dg, du = (a.reshape(t, n // 2) for a in (g, u, off[:, :, 0], off[:, :, 1]))
    want = R._clamped(g, u, 1.5, 1.702, 1.0) if epi == 4 else R._act(g, 0 if epi == 1 else 1) * u
    # |act'| <= 1.2 and |act(g)| <= |g| + 0.3; the activation itself as in the test of the activation alone
    slack = 1.5 * dg * (u.abs() + 1 + du) + du * (g.abs() + 1) + want.abs() * 2.0 ** -20 + (g * u).abs() * 2.0 ** -22 + 2.0 ** -22
    if dtype == "rows":
        out = o.MxRows.empty(t, n // 2)
        out.codes.fill_(3)
        o.linear_mx(x, w, out, epi, **three)
        s = powers(out)[..., None].expand(-1, -1, 32).flatten(1)
        got = code_values(out) * s
        assert not out.codes[:, n // 2:].any()
        got, s = got[:, :n // 2], s[:, :n // 2]
        assert ((got - want).abs() <= torch.maximum((want.abs() + slack) * 2.0 ** -4, 2.0 ** -10 * s) + slack).all()
        big = torch.nn.functional.pad(want.abs(), (0, -(n // 2) % 32)).view(t, -1, 32).amax(-1)
        more = torch.nn.functional.pad(slack, (0, -(n // 2) % 32)).view(t, -1, 32).amax(-1)
        at = powers(out)[:, :big.shape[1]]
        assert (big - more <= 448 * at).all() and ((big + more >= 224 * at) | (at == 1)).all()
    else:
        out = torch.full((t, n // 2), NAN, dtype=dtype, device="cuda")
        o.linear_mx(x, w, out, epi, **three)
        tol = slack + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0)
        assert ((out.double() - want).abs() <= tol).all()


@GPU
@pytest.mark.parametrize("t,n,k", [(1, 256, 1024), (16, 300, 4608), (200, 128, 1300)])
def test_any_split_and_any_depth_of_the_ring(t, n, k):
    o = ops()
    x, w = operands(t, n, k)
    want, tol = stands_for(x) @ stands_for(w).T, product_error(x, w)
    try:
        for split in (1, 2, 4, 8):
            for stages in (0, 4):
                o.mx_set_few(split, stages)
                got = [o.linear_mx(x, w, torch.empty(t, n, device="cuda")) for _ in range(2)]
                assert torch.equal(*got), "the same call twice"
                assert ((got[0].double() - want).abs() <= tol).all(), (split, stages)
    finally:
        o.mx_set_few()


@GPU
@pytest.mark.parametrize("kernel,split", [(1, 0), (1, 4), (1, 8), (2, 0), (3, 0), (4, 2), (4, 4), (4, 8)])
@pytest.mark.parametrize("t,n,k", [(1, 144, 1024), (40, 1008, 1100), (129, 128, 2048), (260, 400, 1280), (33, 48016, 1030), (150, 333, 1100)])
def test_every_kernel_takes_every_size(t, n, k, kernel, split):
    o = ops()
    t = min(t, 64) if kernel == 1 else t
    x, w = operands(t, n, k, seed=k)
    want, tol = stands_for(x) @ stands_for(w).T, product_error(x, w)
    try:
        o.mx_set_kernel(kernel)
        o.mx_set_few(split)
        got = [o.linear_mx(x, w, torch.full((t, n), NAN, device="cuda")) for _ in range(2)]
        assert torch.equal(*got), "the same call twice"
        assert ((got[0].double() - want).abs() <= tol).all()
        half = o.linear_mx(x, w, torch.empty(t, n, dtype=torch.bfloat16, device="cuda"))
        assert torch.equal(half, got[0].bfloat16())
        if n % 16 == 0 and (split < 8 or kernel == 1):
            for epi in (1, 3):
                v = o.linear_mx(x, w, torch.full((t, n // 2), NAN, device="cuda"), epi)
                rows, again = o.MxRows.empty(t, n // 2), o.MxRows.empty(t, n // 2)
                rows.codes.fill_(5)
                o.linear_mx(x, w, rows, epi)
                o.mx_rows(v, again)
                assert torch.equal(rows.codes, again.codes) and torch.equal(scale_rows(rows), scale_rows(again))
                g, u = got[0].view(t, n // 16, 2, 8).unbind(2)
                act = R._act(g.double().reshape(t, n // 2), 0 if epi == 1 else 1) * u.double().reshape(t, n // 2)
                assert ((v.double() - act).abs() <= 2.0 ** -20 * act.abs() + 2.0 ** -22 * (g * u).abs().reshape(t, n // 2) + 1e-30).all()
    finally:
        o.mx_set_kernel()
        o.mx_set_few()


@GPU
@pytest.mark.parametrize("t", [3, 40, 300])
def test_groups_that_stand_for_nan_spoil_their_row_or_column(t):
    o = ops()
    x, w = operands(t, 140, 384)
    x.scales.view(-1)[0] = 255               # row 0, group 0
    w.scales.view(-1)[16 * 5 + 1] = 255      # row 5, group 1
    out = o.linear_mx(x, w, torch.empty(t, 140, device="cuda"))
    bad = torch.zeros(t, 140, dtype=torch.bool, device="cuda")
    bad[0], bad[:, 5] = True, True
    assert torch.equal(torch.isnan(out), bad)


@GPU
def test_scales_from_end_to_end_of_their_range():
    o = ops()
    x, w = operands(4, 32, 128)
    x.scales.fill_(127 + 60)
    w.scales.fill_(127 - 90)
    a = o.linear_mx(x, w, torch.empty(4, 32, device="cuda"))
    x.scales.fill_(127)
    w.scales.fill_(127)
    b = o.linear_mx(x, w, torch.empty(4, 32, device="cuda"))
    assert torch.equal(a, b * 2.0 ** -30)


@GPU
def test_another_stream_and_no_rows():
    o = ops()
    x, w = operands(9, 160, 256)
    want = o.linear_mx(x, w, torch.empty(9, 160, device="cuda"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = o.linear_mx(x, w, torch.empty(9, 160, device="cuda"))
    side.synchronize()
    assert torch.equal(got, want)
    none = o.MxRows.empty(0, 256)
    assert o.linear_mx(none, w, torch.empty(0, 160, device="cuda")).shape == (0, 160)
    o.mx_rows(torch.empty(0, 256, device="cuda"), none)


@GPU
def test_offsets_that_pass_32_bits():
    """Rows of x, of out and of the stream whose places pass 2^31 values; all but the last few are zeros."""
    o = ops()
    last, t = 5, 70016
    for n, k in ((256, 36864), (32768, 128)):                # x of 2.6e9 codes; out of 2.3e9 values
        x, w = o.MxRows.empty(t, k), o.mx_weight(rnd(n, k) / math.sqrt(k))
        tail, _ = operands(last, 1, k, seed=3)
        x.codes[-last:] = tail.codes
        r, g = torch.arange(t - last, t, device="cuda")[:, None], torch.arange(k // 32, device="cuda")
        x.scales.view(-1)[(r // 128 * (k // 128) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4] = scale_rows(tail)
        out = o.linear_mx(x, w, torch.empty(t, n, dtype=torch.bfloat16, device="cuda"))
        want = stands_for(tail) @ stands_for(w).T
        assert ((out[-last:].double() - want).abs() <= product_error(tail, w) + want.abs() * 2.0 ** -8).all()
        assert not out[:-last].any()
        del x, out
    rows, h = 240000, 9216
    stream, res = torch.zeros(rows, h, device="cuda"), torch.zeros(rows, h, dtype=torch.bfloat16, device="cuda")
    stream[-last:], res[-last:] = rnd(last, h), rnd(last, h, seed=1)
    y, w, before = o.MxRows.empty(rows, h), 1 + 0.1 * rnd(h, seed=2), stream[-last:].clone()
    o.add_rmsnorm(stream, res, None, 0.0, w, 1e-6, y)
    assert torch.equal(stream[-last:], before + res[-last:].float())
    part = o.MxRows.empty(last, h)
    o.rmsnorm(stream[-last:].contiguous(), w, 1e-6, part)
    assert torch.equal(y.codes[-last:], part.codes) and not y.codes[:-last].any()


@GPU
def test_a_recorded_product_follows_its_inputs():
    o = ops()
    x, w = operands(2, 512, 1024)
    out = torch.empty(2, 512, device="cuda")
    o.linear_mx(x, w, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.linear_mx(x, w, out)
    y, _ = operands(2, 512, 1024, seed=50)
    x.codes.copy_(y.codes)
    x.scales.copy_(y.scales)
    graph.replay()
    assert torch.equal(out, o.linear_mx(y, w, torch.empty(2, 512, device="cuda")))


@GPU
def test_refusals():
    o = ops()
    x, w = operands(4, 48, 64)
    out = torch.empty(4, 48, device="cuda")
    half = o.MxRows.empty(4, 24)
    for bad in (lambda: o.linear_mx(x, w, out[:, :40]), lambda: o.linear_mx(x, w, torch.empty(3, 48, device="cuda")),
                lambda: o.linear_mx(x, w, out.half()), lambda: o.linear_mx(x, w, out.cpu()), lambda: o.linear_mx(x, w, half),
                lambda: o.linear_mx(x, w, o.MxRows.empty(4, 25), 1), lambda: o.linear_mx(x, w, out, 1), lambda: o.linear_mx(x, w, out, 2),
                lambda: o.linear_mx(x, o.mx_weight(rnd(40, 64)), torch.empty(4, 20, device="cuda"), 1),
                lambda: o.linear_mx(x, o.mx_weight(rnd(48, 96)), out), lambda: o.linear_mx(rnd(4, 64), w, out), lambda: o.linear_mx(x, rnd(48, 64), out),
                lambda: o.linear_mx(w, w, out),
                lambda: o.MxRows(x.codes, x.scales, 5, 64), lambda: o.MxRows(x.codes, x.scales, 4, 200), lambda: o.MxRows(x.codes.int(), x.scales, 4, 64),
                lambda: o.MxRows(x.codes.cpu(), x.scales, 4, 64), lambda: o.MxRows(w.codes, w.scales, 48, 64), lambda: o.MxRows(x.codes, x.scales, 4, 0),
                lambda: o.MxRows(torch.zeros(4, 256, dtype=torch.uint8, device="cuda")[:, ::2], x.scales, 4, 64),
                lambda: o.MxRows(torch.zeros(1 + 4 * 128, dtype=torch.uint8, device="cuda")[1:].view(4, 128), x.scales, 4, 64),
                lambda: o.mx_rows(rnd(4, 65), x), lambda: o.mx_rows(rnd(4, 64).half(), x), lambda: o.mx_rows(rnd(64, 4).T, x),
                lambda: o.mx_weight(rnd(4, 64).half()), lambda: o.mx_weight(torch.randn(4, 64)), lambda: x.values(torch.empty(4, 65, device="cuda")),
                lambda: o.add_rmsnorm(rnd(4, 64), rnd(4, 64), None, 0.0, None, 0.0, x), lambda: o.add_rmsnorm(rnd(4, 64), rnd(5, 64), None, 0.0, rnd(64), 0.0, x),
                lambda: o.add_rmsnorm(rnd(4, 64).bfloat16(), rnd(4, 64), None, 0.0, rnd(64), 0.0, x), lambda: o.rmsnorm(rnd(3, 64), rnd(64), 0.0, x),
                lambda: o.rmsnorm(rnd(4, 64), rnd(65), 0.0, x), lambda: o.gated_act(rnd(4, 128), x, 5), lambda: o.gated_act(rnd(4, 128), x, 0, 4),
                lambda: o.gated_act(rnd(4, 120), x, 0)):
        with pytest.raises(o.KernelError):
            bad()
    torch.cuda.synchronize()
    assert torch.isfinite(o.linear_mx(x, w, out)).all()


@GPU
def test_no_wait_was_given_up():
    """In this library: other tests of the process make waits of theirs run out."""
    o = ops()
    count = torch.full((2,), -1, dtype=torch.int32).pin_memory()
    o.low_bits().janis_mx_timeouts_async(count.data_ptr(), o._stream())
    torch.cuda.synchronize()
    assert count.tolist() == [0, -1]


# ---------------------------------------------------------------------------
# Gemma2 on 4-bit weights
# ---------------------------------------------------------------------------

def plain_mx_logits(cfg, w, ids):
    """The plain model with its layers' matrices in 4 bits and every row that a product reads in 8."""
    from tests.plain import gemma2_plain as P
    w4 = lambda name: R.quantised(w[name].double(), *E2M1)[0]               # noqa: E731
    q8 = lambda v: R.quantised(v, *E4M3)[0]                                  # noqa: E731
    h = P.embed(list(ids), w["model.embed_tokens.weight"], cfg["hidden_size"], torch.float64)
    eps, heads, hd = cfg["rms_norm_eps"], cfg["num_attention_heads"], cfg["head_dim"]
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        a = p + "self_attn."
        ctx = P.attention(q8(P.rms_norm(h, w[p + "input_layernorm.weight"], eps)), w4(a + "q_proj.weight"), w4(a + "k_proj.weight"),
                          w4(a + "v_proj.weight"), torch.eye(heads * hd, dtype=torch.float64), heads, cfg["num_key_value_heads"], hd,
                          cfg["rope_theta"], cfg["query_pre_attn_scalar"], cfg["attn_logit_softcapping"],
                          cfg["sliding_window"] if P.layer_is_sliding(cfg, i) else None)
        h = h + P.rms_norm(q8(ctx) @ w4(a + "o_proj.weight").T, w[p + "post_attention_layernorm.weight"], eps)
        y = q8(P.rms_norm(h, w[p + "pre_feedforward_layernorm.weight"], eps))
        m = p + "mlp."
        act = q8(P.gelu_tanh(y @ w4(m + "gate_proj.weight").T) * (y @ w4(m + "up_proj.weight").T))
        h = h + P.rms_norm(act @ w4(m + "down_proj.weight").T, w[p + "post_feedforward_layernorm.weight"], eps)
    return P.final_logits(h, w, cfg)


def mx_engine(folder, dtype, on, **kw):
    import janis_b200
    if on == "cuda":
        return janis_b200.open(folder, dtype=dtype, weights="mx4", **kw)
    from janis_b200.config.base import read_config_json
    from janis_b200.engine.engine import Engine, _dtype, build_model, check_low_bits
    from janis_b200.parts.base import Runtime, WeightStore
    from janis_b200.weights.loader import load_tensors
    _, cfg, model = build_model(read_config_json(folder))
    check_low_bits(model)
    rt = Runtime(_dtype(dtype), "cpu", R, "mx4")
    model.load(WeightStore(load_tensors(folder, model.tensor_specs(), "cpu", model.ignorable_tensors)), rt)
    return Engine(model, rt, kw.pop("max_tokens"), use_graphs=False, **kw)


def far(got, want):
    """The 2-norm of the difference over that of the plain logits.  A last bit between two correct programs may turn a code (a step
    of 2^-3 of one value); such turns are rare and independent, so the whole is held to the model tolerance and not each logit."""
    return ((got.double().cpu() - want).norm() / want.norm()).item()


# What the kernels may add to the distance from the plain model that the roundings to bfloat16 alone make: those turn about one code
# in 32 of every row by a step of 2^-3 (2^-3 / sqrt(32) = 2.2%), 8 to 12 rows in turn, and which codes turn hangs on last bits.  Their
# share is that of the engine over `kernel_refs`, which rounds in the same places and sums in 64 bits.
MX_BF16_TOL = 4e-2
WHERE = [pytest.param("refs", "float32", BF16_MODEL_TOL), pytest.param("cuda", "float32", BF16_MODEL_TOL, marks=GPU),
         pytest.param("cuda", "bfloat16", MX_BF16_TOL, marks=GPU)]


@pytest.mark.parametrize("on,dtype,tol", WHERE)
@pytest.mark.parametrize("key", ["A", "B_hot", "C", "D"])
def test_model_whole_in_steps_and_in_pieces(key, on, dtype, tol, model_dirs, plain_models):
    cfg, w = plain_models[key]
    eng = mx_engine(model_dirs[key], dtype, on, max_tokens=1024)
    reqs = [random_tokens(TINY[key[0]]["vocab_size"], n, n) for n in ((37, 5, 70) if on == "cuda" else (19, 5))]
    want = [plain_mx_logits(cfg, w, r) for r in reqs]
    allowed = [tol] * len(reqs)
    if dtype == "bfloat16":
        refs = run_requests(mx_engine(model_dirs[key], dtype, "refs", max_tokens=1024), reqs, [len(r) for r in reqs])
        allowed = [tol + far(g, v) for g, v in zip(refs, want)]
    for got in (run_requests(eng, reqs, [len(r) for r in reqs]), run_requests(eng, reqs, [max(1, len(r) - 4) for r in reqs])):
        for g, v, most in zip(got, want, allowed):
            assert far(g, v) <= most, f"{key}: {far(g, v):.2e}"
    if on == "cuda":
        for g, v, most in zip(run_in_pieces(eng, reqs, 16), want, allowed):
            assert far(g, v) <= most, f"{key} in pieces: {far(g, v):.2e}"
    eng.close()


@GPU
def test_generation_is_the_step_functions(model_dirs):
    import janis_b200
    for graphs in (True, False):
        eng = janis_b200.open(model_dirs["B"], dtype="bfloat16", max_tokens=2048, weights="mx4", use_graphs=graphs)
        prompts = [random_tokens(384, n, n) for n in (9, 33, 4)]
        replies = eng.generate(prompts, max_tokens=12, stop=())
        for p, r in zip(prompts, replies):
            assert len(r) == 12
            ids = p + r
            logits = run_requests(eng, [ids], [len(ids)])[0]
            # each token is the largest logit behind what precedes it, to the distance at which two forms of a step differ
            for i, t in enumerate(r):
                row = logits[len(p) + i - 1]
                assert row[t] >= row.max() - 0.05 * row.abs().max()
        eng.close()


def test_models_whose_layers_cannot_are_refused():
    import janis_b200
    from janis_b200.engine.engine import check_low_bits
    from janis_b200.parts.base import Runtime
    from tests.conftest import TINY_A
    _, _, model = janis_b200.build_model(TINY_A)
    check_low_bits(model)
    model.blocks[1].mixer.low_bits = False
    with pytest.raises(ValueError, match="layer 1"):
        check_low_bits(model)
    with pytest.raises(ValueError, match="mx4"):
        Runtime(torch.float32, "cpu", R, "int3")
    rt = Runtime(torch.float32, "cpu", R, "mx4")
    with pytest.raises(ValueError, match="workspace"):
        rt.linear(torch.zeros(1, 8), rt.weight(torch.zeros(4, 8)), torch.zeros(1, 4))


def test_the_host_side_needs_a_device():
    from janis_b200.kernels.ops import KernelError, MxRows, MxWeight, linear_mx
    with pytest.raises(KernelError):
        MxRows(torch.zeros(1, 128, dtype=torch.uint8), torch.zeros(1, 1, 512, dtype=torch.uint8), 1, 128)
    with pytest.raises(KernelError):
        linear_mx(None, MxWeight, None)
