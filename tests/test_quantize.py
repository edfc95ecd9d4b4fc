"""Row passes with an 8-bit output (xf_rms_norm_quantize, xf_act_mul_quantize) against 64-bit formulas.

Tolerances, counted before the first run (u = 2^-24, the rounding of one fp32 operation):
 * norm codes: t = h * w is exact, L / a and its product with t round once each, so the value that is rounded
   to a code is within 2^-22 of the exact one; int8 codes near a tie are decided exactly, so they are equal.
 * norm scales: a sum of n non-negative terms per thread and ten levels of tree add at most (n + 10) u to the
   mean, half of it to rstd; division, root, product and division add 5 u.
 * gate: __expf(x) is within 2 + 1.173 |x| ulp (2 u each), which a sigmoid passes on at most once;
   the sum, the division (2 ulp) and the product with `up` add 8 u.  erf in gelu is within 1.5e-7 of 1 + erf.
"""
import math

import pytest
import torch

U = 2.0 ** -24
FLOOR = 2.0 ** -100
E4M3 = torch.float8_e4m3fn


def nearest_e4m3(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def nearest_s8(v):
    return torch.sign(v) * torch.floor(v.abs() + 0.5)


def block_max(t, s8):
    """Largest magnitude of each row (s8) or block of 128 columns, floored, and the same for every element."""
    M, N = t.shape
    if s8:
        a = t.abs().amax(1).clamp_min(FLOOR)
        return a, a[:, None].expand(M, N)
    p = torch.nn.functional.pad(t, (0, -N % 128)).view(M, -1, 128).abs().amax(2).clamp_min(FLOOR)
    return p, p.repeat_interleave(128, 1)[:, :N]


def padded(M, N, extra, dtype, gen=None, scale=1.0):
    """[M, N] with `extra` columns of something else behind each row."""
    t = torch.randn(M, N + extra, device="cuda", generator=gen).mul_(scale).to(dtype)
    return t, t[:, :N]


def out_tensors(M, N, s8, extra):
    whole = torch.full((M, N + extra), 77, device="cuda", dtype=torch.int8)
    q = (whole if s8 else whole.view(E4M3))[:, :N]
    scale = torch.full((M,), -1.0, device="cuda") if s8 else torch.full((-(-N // 128), M), -1.0, device="cuda").t()
    return whole, q, scale


def check_norm(h, w, q, scale, s8, eps, threads_terms):
    t = h.double() * (w.double() if w is not None else 1.0)
    L = 127.0 if s8 else 448.0
    a, wide = block_max(t, s8)
    v = t * L / wide
    if s8:
        assert torch.equal(q.double(), nearest_s8(v))
    else:
        lo, hi = nearest_e4m3(v * (1 - 2.0 ** -22)), nearest_e4m3(v * (1 + 2.0 ** -22))
        got = q.double()
        assert bool(((got == lo) | (got == hi)).all())
    rstd = 1.0 / torch.sqrt(h.double().square().mean(1) + eps)
    want = a * (rstd if s8 else rstd[:, None]) / L
    tol = ((threads_terms + 10) / 2 + 5) * U
    assert bool(((scale.double() - want).abs() <= tol * want).all())


NORM_SHAPES = [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (4, 4096), (33, 5003), (2, 8200), (3, 20000), (2, 40001)]


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
@pytest.mark.parametrize("residual", [None, "apart", "in place"])
@pytest.mark.parametrize("M,N", NORM_SHAPES)
@pytest.mark.parametrize("extra", [0, 24, 5])
def test_norm(capi, cuda, M, N, residual, s8, extra):
    gen = torch.Generator(device="cuda").manual_seed(M * 100003 + N)
    _, x = padded(M, N, extra, torch.bfloat16, gen)
    w = torch.randn(N, device=cuda, generator=gen).to(torch.bfloat16) if extra != 5 else None
    whole, q, scale = out_tensors(M, N, s8, extra)
    res = hout = None
    h = x
    if residual:
        rwhole, res = padded(M, N, extra, torch.bfloat16, gen, 3.0)
        before = rwhole.clone()
        h = (x.float() + res.float()).to(torch.bfloat16)
        hout = torch.zeros(M, N, device=cuda, dtype=torch.bfloat16) if residual == "apart" else None
    capi.rms_norm_quantize(q, scale, x, w, res, hout, 1e-5)
    torch.cuda.synchronize()
    terms = 16 * math.ceil(N / 16 / 512)      # 512 threads at most, 16 columns at a time
    check_norm(h, w, q, scale, s8, 1e-5, terms)
    assert bool((whole[:, N:] == 77).all())
    if residual:
        assert torch.equal(hout if residual == "apart" else res, h)
        want = before if residual == "apart" else torch.cat([h, before[:, N:]], 1)
        assert torch.equal(rwhole, want)


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
def test_norm_special_rows(capi, cuda, s8):
    N = 384
    x = torch.randn(6, N, device=cuda).to(torch.bfloat16)
    x[0] = 0                                   # nothing but zeros
    x[1, 128:256] = 0                          # one block of zeros
    x[2, 200] = float("nan")
    x[3, 5] = float("inf")
    x[4] = 1e-38                               # far below the floor once squared
    x[5] = 3e38                                # the sum of squares overflows: rstd is 0
    _, q, scale = out_tensors(6, N, s8, 0)
    capi.rms_norm_quantize(q, scale, x, None, eps=1e-6)
    torch.cuda.synchronize()
    v = q.double() * (scale.double()[:, None] if s8 else scale.double().repeat_interleave(128, 1))
    assert bool((q[0].float() == 0).all()) and bool(torch.isfinite(scale[0]).all()) and bool((scale[0] > 0).all())
    assert bool((q[1, 128:256].float() == 0).all())
    check_norm(x[1:2], None, q[1:2], scale[1:2], s8, 1e-6, 16)
    assert bool(torch.isnan(scale[2]).all())   # the row's mean is NaN
    assert bool(torch.isnan(scale[3]).any())   # inf * rstd, rstd = 0
    assert bool(torch.isfinite(v[4]).all()) and bool((v[4].abs() <= 1.001e-35).all())
    assert bool((scale[5] == 0).all()) and bool(torch.isfinite(q[5].float()).all())


def nearest_quotient_e4m3(t, wide):
    """Codes of t * 448 / wide: with 16 significant bits in t and `wide` a tie is exact in 64 bits, and no other quotient
    comes nearer to one than 2^-21 of it."""
    return nearest_e4m3(t * 448.0 / wide)


@pytest.mark.gpu
@pytest.mark.parametrize("scale_by", [2.0 ** -80, 1.0, 2.0 ** 100])
def test_norm_e4m3_ties_go_to_even(capi, cuda, scale_by):
    """Rows whose every quotient lies exactly between two codes: t = b w, largest value 448 b, quotient w."""
    b = torch.arange(1, 256, 2, device=cuda, dtype=torch.float64)
    m = torch.arange(17, 32, 2, device=cuda, dtype=torch.float64)
    w = (m[:, None] * 2.0 ** torch.arange(-10, 4, device=cuda)).flatten()          # normal codes
    w = torch.cat([w, (2 * torch.arange(8, device=cuda) + 1) * 2.0 ** -10])        # between subnormal codes
    w = torch.cat([w, -w, w])[:254].view(2, 127)
    w = torch.cat([torch.full((2, 1), 448.0, device=cuda, dtype=torch.float64), w], 1).flatten()
    h = (b[:, None] * scale_by).expand(-1, w.numel()).to(torch.bfloat16).contiguous()
    h[1::2] *= -1
    assert torch.equal(h.double().abs(), (b[:, None] * scale_by).expand_as(h)) and torch.equal(w.to(torch.bfloat16).double(), w)
    _, q, scale = out_tensors(len(b), w.numel(), False, 0)
    capi.rms_norm_quantize(q, scale, h, w.to(torch.bfloat16), eps=0.0)
    torch.cuda.synchronize()
    want = nearest_e4m3(w) * torch.sign(h[:, :1].double())
    assert torch.equal(q.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [False, True])
def test_norm_e4m3_codes_are_the_exact_quotients(capi, cuda, residual):
    """About 4 codes in 10000 of normal data are ties; N = 1000 ends in a short block."""
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(512, 1000, device=cuda, generator=gen).to(torch.bfloat16)
    x[0, 128:256] = float("inf")
    x[0, 130] = -0.0
    x[1, 5] = -0.0
    w = torch.randn(1000, device=cuda, generator=gen).mul_(0.1).add_(1.0).to(torch.bfloat16)
    res = torch.randn(512, 1000, device=cuda, generator=gen).to(torch.bfloat16) if residual else None
    h = (x.float() + res.float()).to(torch.bfloat16) if residual else x
    _, q, scale = out_tensors(512, 1000, False, 0)
    capi.rms_norm_quantize(q, scale, x, w, res)
    torch.cuda.synchronize()
    t = h.double() * w.double()
    _, wide = block_max(t, False)
    fine = torch.isfinite(t) & torch.isfinite(wide)
    assert torch.equal(q.double()[fine], nearest_quotient_e4m3(t, wide)[fine])
    # the only finite value of a block of infinities has the code of zero, and zeros keep their sign
    assert float(q[0, 130].float()) == 0.0
    if not residual:
        assert q.view(torch.int8)[0, 130] == -128 and q.view(torch.int8)[1, 5] == -128


def gate_tolerance(g, gelu):
    if gelu:      # 1.5e-7 of a factor 1 + erf(z) that is at least 1 on the positive side; on the other
        #           side P(t) exp(-z^2) with |error of P| <= 1.5e-7 / exp(-z^2) of P(0) = 1
        z2 = g.abs().clamp_max(13.0).square() / 2
        return torch.where(g >= 0, 3e-7 + 0 * g, 1.5e-7 * (1 + z2) * 8 + 1e-6)
    return (2 * (2 + 1.173 * g.abs()) + 8) * U


def check_act(x, d, q, scale, s8, gelu):
    g, u = x[:, :d].double(), x[:, d:].double()
    y = g * (torch.special.ndtr(g) if gelu else torch.sigmoid(g)) * u
    L = 127.0 if s8 else 448.0
    a, wide = block_max(y, s8)
    # absolute slack of one value: its relative error, and for gelu the absolute error of 1 + erf
    slack = (gate_tolerance(g, gelu) * y.abs()) + (1.5e-7 * (g * u).abs() if gelu else 0)
    most, _ = block_max(slack, s8)
    assert bool(((scale.double() * L - a).abs() <= most + 2 * U * a).all())
    wide_scale = scale.double()[:, None].expand_as(y) if s8 else scale.double().repeat_interleave(128, 1)[:, :d]
    got = q.double() * wide_scale
    v = (y / wide_scale).abs()
    half = 0.5 if s8 else torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 4)
    # half a step at the value itself, and its slack seen from either side of a border
    assert bool(((got - y).abs() <= half * wide_scale * (1 + 2.0 ** -20) + 2 * slack + 4 * U * y.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("M,d", [(1, 1), (1, 8), (3, 127), (2, 128), (5, 129), (4, 4096), (17, 1003), (2, 14336), (3, 20001)])
@pytest.mark.parametrize("extra", [0, 16, 3])
def test_act(capi, cuda, M, d, gelu, s8, extra):
    gen = torch.Generator(device="cuda").manual_seed(M * 100003 + d)
    _, x = padded(M, 2 * d, extra, torch.bfloat16, gen, 2.0)
    whole, q, scale = out_tensors(M, d, s8, extra)
    capi.act_mul_quantize(q, scale, x, gelu)
    torch.cuda.synchronize()
    check_act(x, d, q, scale, s8, gelu)
    assert bool((whole[:, d:] == 77).all())


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
@pytest.mark.parametrize("d", [1, 3, 130, 257])
def test_gelu_of_negative_gates_keeps_its_relative_precision(capi, cuda, d, s8):
    """A block of nothing but strongly negative gates has a scale of its own.  Errors in units of u: __expf(g^2 / 2)
    2 (2 + 1.173 g^2 / 2), the rest of the activation 8, the reciprocal 2 ulp, passed on 2.7 times at most: 8 more
    than the exact one counted before, products with `up` and 1 / L 2."""
    gen = torch.Generator(device="cuda").manual_seed(d)
    g = (torch.rand(64, d, device=cuda, generator=gen) * 8.5 + 2.5).neg().to(torch.bfloat16)
    g[:5, -1] = torch.tensor([-4.0, -5.0, -8.0, -10.0, -11.0], device=cuda).to(torch.bfloat16)
    u = (torch.rand(64, d, device=cuda, generator=gen) + 0.5).to(torch.bfloat16)
    _, q, scale = out_tensors(64, d, s8, 0)
    capi.act_mul_quantize(q, scale, torch.cat([g, u], 1), True)
    torch.cuda.synchronize()
    gd = g.double()
    y = gd * torch.exp(torch.special.log_ndtr(gd)) * u.double()
    slack = (2 * (2 + 1.173 * gd.square() / 2) + 18) * U * y.abs()
    L = 127.0 if s8 else 448.0
    a, _ = block_max(y, s8)
    most, _ = block_max(slack, s8)
    assert bool(((scale.double() * L - a).abs() <= most + 2 * U * a).all())
    wide = scale.double()[:, None].expand_as(y) if s8 else scale.double().repeat_interleave(128, 1)[:, :d]
    v = (y / wide).abs()
    half = 0.5 if s8 else torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 4)
    assert bool(((q.double() * wide - y).abs() <= half * wide * (1 + 2.0 ** -20) + 2 * slack + 4 * U * y.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
def test_act_special_values(capi, cuda, s8):
    d = 256
    x = torch.randn(4, 2 * d, device=cuda).to(torch.bfloat16)
    x[0, d:] = 0                                 # up half of zeros
    x[1, 3] = float("nan")
    x[2, 7] = -100.0                             # exp(100) is infinite: the gate is -0
    x[3, :d] = -200.0
    _, q, scale = out_tensors(4, d, s8, 0)
    capi.act_mul_quantize(q, scale, x)
    torch.cuda.synchronize()
    assert bool((q[0].float() == 0).all()) and bool(torch.isfinite(scale[0]).all())
    assert bool(torch.isnan(scale[1].reshape(-1)[0]))
    assert float(q[2, 7].float()) == 0.0 and bool(torch.isfinite(scale[2]).all())
    assert bool((q[3].float() == 0).all())


@pytest.mark.gpu
def test_no_rows_and_other_streams(capi, cuda):
    x = torch.randn(64, 512, device=cuda).to(torch.bfloat16)
    _, q, scale = out_tensors(64, 512, False, 0)
    capi.rms_norm_quantize(q[:0], scale[:0], x[:0])             # nothing to do, nothing written
    capi.act_mul_quantize(q[:0, :256], scale[:0, :2], x[:0])
    torch.cuda.synchronize()
    assert bool((scale == -1).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        capi.rms_norm_quantize(q, scale, x)
    side.synchronize()
    want_q, want_s = q.clone(), scale.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.rms_norm_quantize(q, scale, x)
    for k in (1.0, 2.0):
        q.view(torch.int8).zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(q.view(torch.int8), want_q.view(torch.int8)) and torch.equal(scale, want_s)


@pytest.mark.gpu
@pytest.mark.parametrize("s8", [False, True])
def test_offsets_past_32_bits(capi, cuda, s8):
    M, N, pitch = 40000, 256, 65536                  # the last rows start beyond 2^31 elements
    x = torch.empty(M, pitch, device=cuda, dtype=torch.bfloat16)[:, :N]
    x[:, :] = torch.randn(1, N, device=cuda)
    x[-3:] = torch.randn(3, N, device=cuda).to(torch.bfloat16)
    q = torch.empty(M, pitch * 2, device=cuda, dtype=torch.int8)[:, :N]
    q = q if s8 else q.view(E4M3)
    scale = torch.empty(M, device=cuda) if s8 else torch.empty(2, M, device=cuda).t()
    capi.rms_norm_quantize(q, scale, x, None, eps=1e-5)
    torch.cuda.synchronize()
    check_norm(x[-3:], None, q[-3:], scale[-3:], s8, 1e-5, 16)
    half = N // 2
    sc = torch.empty(M, device=cuda) if s8 else torch.empty(1, M, device=cuda).t()
    capi.act_mul_quantize(q[:, :half], sc, x)
    torch.cuda.synchronize()
    check_act(x[-3:], half, q[-3:, :half], sc[-3:], s8, False)


# ------------------------------------------------------------------ refusals: no GPU is touched
def desc(capi, **k):
    """A packed xf_quantize_desc of a valid norm, with some fields changed."""
    d = dict(out=0x1000, scale=0x2000, input=0x3000, residual=0, residual_out=0, weight=0, ld_out=512, scale_row=1, scale_blk=8,
             ld_in=512, ld_res=0, ld_res_out=0, out_dtype=4, M=8, N=512, eps=1e-6, gelu=0, pad=0)
    assert set(k) <= set(d)
    return capi._QUANTIZE_DESC.pack(*{**d, **k}.values())


def test_packed_descriptor_is_the_headers(capi):
    fields = "out scale input residual residual_out weight ld_out scale_row_stride scale_blk_stride ld_in ld_res " \
             "ld_res_out out_dtype M N eps gelu pad_".split()
    import os
    header = open(os.path.join(os.path.dirname(capi.HERE), "include", "xefuse_b200.h")).read()
    body = header[header.index("typedef struct xf_quantize_desc"):header.index("} xf_quantize_desc;")]
    import re
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n.strip(" *") for line in re.findall(r"\b(?:void\*|float\*|int64_t|int32_t|float)\s+([^;]+);", body) for n in line.split(",")]
    assert names == fields and capi._QUANTIZE_DESC.size == 120


BAD = [(dict(M=-1), 4), (dict(N=0), 4), (dict(out_dtype=0), 2), (dict(out=0), 4), (dict(scale=0), 4), (dict(input=0), 4),
       (dict(ld_in=511), 3), (dict(ld_out=511), 3), (dict(scale_row=0), 3), (dict(scale_blk=0), 3), (dict(N=(1 << 20) + 1), 5),
       (dict(input=0x3001), 1), (dict(scale=0x2002), 1)]


@pytest.mark.parametrize("change,status", BAD + [
    (dict(residual=0x4000, ld_res=512), 4), (dict(residual_out=0x4000, ld_res_out=512), 4),
    (dict(residual=0x4000, ld_res=511, residual_out=0x4000, ld_res_out=512), 3),
    (dict(residual=0x4001, ld_res=512, residual_out=0x4000, ld_res_out=512), 1), (dict(weight=0x5001), 1)])
def test_norm_refusals(capi, change, status):
    assert capi.lib().xf_rms_norm_quantize(desc(capi, **change), None) == status
    assert capi.lib().xf_last_error_string()


@pytest.mark.parametrize("change,status", BAD + [
    (dict(ld_in=1023), 3), (dict(weight=0x5000, ld_in=1024), 4),
    (dict(residual=0x4000, ld_res=512, residual_out=0x4000, ld_res_out=512, ld_in=1024), 4)])
def test_act_refusals(capi, change, status):
    assert capi.lib().xf_act_mul_quantize(desc(capi, **{"ld_in": 1024, **change}), None) == status


def test_empty_calls(capi):
    empty = desc(capi, M=0, out=0, input=0, scale=0)
    assert capi.lib().xf_rms_norm_quantize(empty, None) == 0
    assert capi.lib().xf_act_mul_quantize(empty, None) == 0
    assert capi.lib().xf_rms_norm_quantize(None, None) == 4
    assert capi.lib().xf_act_mul_quantize(None, None) == 4


def test_wrapper_refusals(capi, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)       # what a CPU tensor reports
    x, s = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(4, 2)
    q = torch.zeros(4, 256, dtype=E4M3)
    for bad in (
        lambda: capi.rms_norm_quantize(torch.zeros(4, 256), s, x),                  # output type
        lambda: capi.rms_norm_quantize(q, torch.zeros(4, 1), x),                    # scales of another width
        lambda: capi.rms_norm_quantize(q, s, x.float()),                            # input type
        lambda: capi.rms_norm_quantize(q[:, ::2], s, x),                            # another width
        lambda: capi.rms_norm_quantize(q.t().contiguous().t(), s, x),               # columns not contiguous
        lambda: capi.rms_norm_quantize(q, s, x, x[0, :128]),                        # weight of another width
        lambda: capi.rms_norm_quantize(q, s, x, residual=x[:2]),
        lambda: capi.act_mul_quantize(q, s, x),                                     # input is [M, 2 d]
    ):
        with pytest.raises(capi.XfError):
            bad()


def test_wrapper_refuses_other_dimensions_in_its_own_manner(capi, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    x, s, q = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(4, 2), torch.zeros(4, 256, dtype=E4M3)
    for bad in (
        lambda: capi.rms_norm_quantize(q[0], s[0], x[0]),
        lambda: capi.rms_norm_quantize(q[None], s[None], x[None]),
        lambda: capi.rms_norm_quantize(q, s, x[0]),
        lambda: capi.rms_norm_quantize(q, s, x, x[:1]),              # weight is a vector
        lambda: capi.act_mul_quantize(q[0], s[0], x[0]),
        lambda: capi.act_mul_quantize(q[:, :128], s[:, :1], x[None]),
        lambda: capi.act_mul_quantize(q[:, :128], s[0, :1], x),
    ):
        with pytest.raises(capi.XfError):
            bad()


def test_wrapper_refuses_rows_beyond_32_bits(capi, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    M = 2 ** 31
    x, s, q = torch.zeros(1, 32, dtype=torch.bfloat16), torch.zeros(1, 1), torch.zeros(1, 32, dtype=E4M3)
    with pytest.raises(capi.XfError, match="rows"):
        capi.rms_norm_quantize(q.expand(M, -1), s.expand(M, -1), x.expand(M, -1))
    with pytest.raises(capi.XfError, match="rows"):
        capi.act_mul_quantize(q[:, :16].expand(M, -1), s.expand(M, -1), x.expand(M, -1))


def test_a_residual_out_without_a_residual_is_refused(capi, monkeypatch):
    """It was left as it is without a word."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    x, s, q = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(4, 2), torch.zeros(4, 256, dtype=E4M3)
    with pytest.raises(capi.XfError, match="residual"):
        capi.rms_norm_quantize(q, s, x, residual_out=torch.zeros_like(x))
