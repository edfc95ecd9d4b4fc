"""The 8-bit path of a transformer layer and its expert form, as measured cases.

Four operators: `norm` (residual add + RMSNorm + 8-bit output with scales), `act` (SwiGLU / GeGLU of
the two halves of a row + 8-bit output with scales), `gemm` (e4m3 product with one fp32 scale for each
1 x 128 block of A and each 128 x 128 block of B) and `grouped` (products of ragged row groups, each with
its own weight, in bf16 or block-scaled e4m3).  With `own` false, run() is the plain form in elementary
torch operations; with `own` true it is the library's call.
"""
import math
import random

import torch

own = False

BLOCK = 128          # elements that share a scale
FLOOR = 2.0 ** -100  # least absolute maximum a scale is made from
E4M3 = torch.float8_e4m3fn
EPS = 1e-6


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step: launch latency
        dict(name="norm_token", op="norm", M=1, N=4096, out="e4m3", residual=True),
        # a prefill chunk, the residual stream updated on the way: HBM bandwidth
        dict(name="norm_prefill", op="norm", M=4096, N=8192, out="e4m3", residual=True),
        # an odd width into the int8 path, where no residual enters (first norm of a stack)
        dict(name="norm_s8_odd", op="norm", M=1000, N=5003, out="s8", residual=False),
        # gate and up halves of a small decode batch
        dict(name="act_batch", op="act", M=16, N=14336, out="e4m3", gelu=False),
        # the same of a prefill chunk
        dict(name="act_prefill", op="act", M=4096, N=14336, out="e4m3", gelu=False),
        # one token against a square projection: latency and weight streaming
        dict(name="gemm_token", op="gemm", M=1, N=4096, K=4096, nk=True, out="bf16", pair="none"),
        # a decode batch against the gate/up weights: every byte of the weights once
        dict(name="gemm_batch", op="gemm", M=64, N=28672, K=4096, nk=False, out="bf16", pair="swiglu"),
        # a prefill chunk against the gate/up weights: tensor cores
        dict(name="gemm_prefill", op="gemm", M=4096, N=28672, K=4096, nk=True, out="bf16", pair="none"),
        # ragged in every extent, fp32 results (a head whose logits are kept exact)
        dict(name="gemm_odd", op="gemm", M=777, N=5001, K=2000, nk=False, out="f32", pair="none"),
        # a decode batch routed to 64 experts, about half of them hit: weight streaming
        dict(name="grouped_batch", op="grouped", dtype="e4m3", G=64, M=48, N=4096, K=2048, nk=True, out="bf16", pair="none"),
        # a prefill chunk routed to 64 experts, skewed, some experts empty: tensor cores
        dict(name="grouped_prefill", op="grouped", dtype="e4m3", G=64, M=16384, N=4096, K=2048, nk=False, out="bf16", pair="swiglu"),
        # bf16 experts, few and large
        dict(name="grouped_bf16", op="grouped", dtype="bf16", G=8, M=4096, N=4096, K=4096, nk=False, out="bf16", pair="none"),
    ]


def draw(rng):
    def span(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "act", "gemm", "grouped"])
    while True:
        if op in ("norm", "act"):
            c = dict(op=op, M=span(1, 8192), N=span(32, 16384), out=rng.choice(["e4m3", "e4m3", "s8"]))
            c["residual" if op == "norm" else "gelu"] = rng.random() < 0.5
            if c["M"] * c["N"] <= 4096 * 8192:
                return c
            continue
        c = dict(op=op, M=span(1, 4096 if op == "gemm" else 16384), N=span(64, 28672 if op == "gemm" else 8192),
                 K=span(32, 16384 if op == "gemm" else 8192), nk=rng.random() < 0.5,
                 out=rng.choice(["bf16", "bf16", "f32"]), pair=rng.choice(["none", "none", "swiglu", "geglu"]))
        if c["pair"] != "none":
            c["N"] += c["N"] % 2
        if op == "grouped":
            c["G"] = span(1, 128)
            c["dtype"] = rng.choice(["e4m3", "bf16"])
        if 2.0 * c["M"] * c["N"] * c["K"] <= 2.0 * 16384 * 4096 * 2048 and c.get("G", 1) * c["N"] * c["K"] <= 64 * 4096 * 2048:
            return c


def _sizes(case):
    """Rows of each group, in descending order: a skewed routing that depends on the case alone."""
    r, G, M = random.Random(17), case["G"], case["M"]
    weight = [r.expovariate(1.0) if r.random() > 0.125 else 0.0 for _ in range(G)]
    total = sum(weight) or 1.0
    sizes = [int(M * w / total) for w in weight]
    for i in range(M - sum(sizes)):
        sizes[r.randrange(G)] += 1
    return sorted(sizes, reverse=True)


def _up(n, m):
    return -(-n // m) * m


# ---------------------------------------------------------------------------------------- prepare
def _codes(g, shape, pad):
    """Normal values as 8-bit codes of blocks whose largest value is near 448; rows padded to `pad` elements."""
    cols = _up(shape[-1], pad)
    t = torch.randn(*shape[:-1], cols, generator=g, device="cuda", dtype=torch.bfloat16)
    return t.mul_(130.0).clamp_(-448.0, 448.0).to(E4M3)[..., :shape[-1]]


def _scales(g, *shape):
    return torch.empty(shape, device="cuda").normal_(generator=g).mul_(0.3).exp_().mul_(1.0 / 512)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    op, M, N = case["op"], case["M"], case["N"]
    if op in ("norm", "act"):
        s["x"] = torch.randn(M, N if op == "norm" else 2 * N, generator=g, device="cuda").to(torch.bfloat16)
        if op == "norm":
            s["weight"] = torch.randn(N, generator=g, device="cuda").mul_(0.1).add_(1.0).to(torch.bfloat16)
            if case["residual"]:
                s["residual"] = torch.randn(M, N, generator=g, device="cuda").mul_(4.0).to(torch.bfloat16)
        if own:
            s["capi"] = _capi()
            # rows of the 8-bit output on 16-byte boundaries, scales with the rows side by side: what the products read
            s["q"] = torch.empty(M, _up(N, 16), device="cuda", dtype=E4M3 if case["out"] == "e4m3" else torch.int8)[:, :N]
            s["scale"] = torch.empty(-(-N // BLOCK), M, device="cuda").t() if case["out"] == "e4m3" else torch.empty(M, device="cuda")
            s["h"] = torch.empty_like(s["x"]) if case.get("residual") else None
        return s
    K, G, nk = case["K"], case.get("G"), case["nk"]
    kb, nb = -(-K // BLOCK), -(-N // BLOCK)
    shape = (N, K) if nk else (K, N)
    shape = shape if G is None else (G, *shape)
    if case.get("dtype", "e4m3") == "e4m3":
        s["A"], s["B"] = _codes(g, (M, K), 16), _codes(g, shape, 16)
        s["scale_a"] = _scales(g, kb, M).t()
        s["scale_b"] = _scales(g, *shape[:-2], nb, kb) if nk else _scales(g, *shape[:-2], kb, nb)
    else:
        s["A"] = torch.randn(M, _up(K, 8), generator=g, device="cuda").to(torch.bfloat16)[:, :K]
        s["B"] = torch.randn(*shape[:-1], _up(shape[-1], 8), generator=g, device="cuda", dtype=torch.bfloat16).mul_(K ** -0.5)[..., :shape[-1]]
    if G is not None:
        sizes = _sizes(case)
        random.Random(seed).shuffle(sizes)          # which expert is popular changes with the inputs
        s["most"] = max(sizes)
        s["offsets"] = torch.tensor([sum(sizes[:i]) for i in range(G + 1)], device="cuda", dtype=torch.int32)
    if own:
        s["D"] = torch.empty(M, N if case["pair"] == "none" else N // 2, device="cuda",
                             dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float32)
        s["plan"] = _capi().GroupedGemmPlan(s["A"], s["B"], s["D"], offsets=s.get("offsets"), scale_a=s.get("scale_a"),
                                            scale_b=s.get("scale_b"), b_nk=nk, pair=case["pair"])
    return s


def _capi():
    import xefuse_loader
    return xefuse_loader.load().capi


# -------------------------------------------------------------------------------------------- run
def _act(x, gelu):
    return x * 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) if gelu else x / (1.0 + torch.exp(-x))


def _blocks(t):
    """[M, N] -> [M, N / 128, 128], zeros behind the last column."""
    return torch.nn.functional.pad(t, (0, -t.shape[1] % BLOCK)).view(t.shape[0], -1, BLOCK)


def _quantize(t, rstd, out):
    """8-bit values of t * rstd and what one step of them stands for (int8: the values they stand for, in bf16);
    rstd is a row's common factor."""
    if out == "s8":
        a = t.abs().amax(1, keepdim=True).clamp_min(FLOOR)
        # in 64 bits: values next to the border between two steps
        v = t.double() * 127.0 / a.double()
        q = torch.sign(v) * torch.floor(v.abs() + 0.5)
        return ((q.float() * (a * rstd / 127.0)).to(torch.bfloat16),)
    b = _blocks(t)
    a = b.abs().amax(2, keepdim=True).clamp_min(FLOOR)
    q = (b * (448.0 / a)).clamp(-448.0, 448.0).view(t.shape[0], -1)[:, :t.shape[1]].to(E4M3)
    return q, a[:, :, 0] * rstd / 448.0


def _wide(scale, k_dim, n):
    """A scale for each block of 128 -> one for each of `n` elements along `k_dim`."""
    return scale.repeat_interleave(BLOCK, k_dim).narrow(k_dim, 0, n)


def _result(v, case):
    if case["pair"] != "none":
        v = _act(v[..., 0::2], case["pair"] == "geglu") * v[..., 1::2]
    return v.to(torch.bfloat16) if case["out"] == "bf16" else v


def _held(s):
    return (s["q"], s["scale"]) if s["case"]["out"] == "e4m3" else ((s["q"].float() * s["scale"][:, None]).to(torch.bfloat16),)


def run(s):
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        if own:
            s["capi"].rms_norm_quantize(s["q"], s["scale"], s["x"], s["weight"], s.get("residual"), s["h"], EPS)
            return _held(s) + ((s["h"],) if case["residual"] else ())
        h = s["x"].float()
        if case["residual"]:
            h = (h + s["residual"].float()).to(torch.bfloat16)
            kept, h = h, h.float()
        rstd = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        return _quantize(h * s["weight"].float(), rstd, case["out"]) + ((kept,) if case["residual"] else ())
    if op == "act":
        if own:
            s["capi"].act_mul_quantize(s["q"], s["scale"], s["x"], case["gelu"])
            return _held(s)
        gate, up = s["x"].float().chunk(2, 1)
        return _quantize(_act(gate, case["gelu"]) * up, 1.0, case["out"])
    if own:
        s["plan"].run()
        return s["D"]
    a, b, nk = s["A"].float(), s["B"].float(), case["nk"]
    if nk:
        b = b.transpose(-1, -2)
    if "scale_a" in s:
        sb = s["scale_b"].transpose(-1, -2) if nk else s["scale_b"]
        a = a * _wide(s["scale_a"], 1, case["K"])
        b = b * _wide(_wide(sb, sb.dim() - 2, case["K"]), sb.dim() - 1, case["N"])
    if op == "gemm":
        return _result(a @ b, case)
    # every group padded to the rows of the largest one
    off, row = s["offsets"].long(), torch.arange(case["M"], device="cuda")
    group = torch.searchsorted(off[1:].contiguous(), row, right=True)
    at = row - off[group]
    padded = torch.zeros(case["G"], s["most"], case["K"], device="cuda")
    padded[group, at] = a
    return _result(torch.bmm(padded, b)[group, at], case)


# ------------------------------------------------------------------------------------- work, exact
def work(case):
    op, M, N = case["op"], case["M"], case["N"]
    if op in ("norm", "act"):
        scales = 4 * M * (-(-N // BLOCK) if case["out"] == "e4m3" else 1)
        if op == "norm":
            return {"bytes": M * N * (7 if case["residual"] else 3) + 2 * N + scales, "flops": 8 * M * N}
        return {"bytes": 5 * M * N + scales, "flops": 12 * M * N}
    K, wide = case["K"], 1 if case.get("dtype", "e4m3") == "e4m3" else 2
    hit = 1 if op == "gemm" else sum(n > 0 for n in _sizes(case))
    cols = N if case["pair"] == "none" else N // 2
    moved = wide * (M * K + hit * N * K) + M * cols * (2 if case["out"] == "bf16" else 4)
    if wide == 1:
        moved += 4 * -(-K // BLOCK) * (M + hit * -(-N // BLOCK))
    return {"bytes": moved, "flops": 2 * M * N * K}


def _nearest_e4m3(v):
    """Nearest e4m3 value (3 mantissa bits, least step 2^-9, ties to even), in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448.0, 448.0)


def _exact_quantized(y, out):
    """8-bit values and scales of the finished values y."""
    M, N = y.shape
    if out == "s8":
        scale = y.abs().amax(1, keepdim=True).clamp_min(1e-300) / 127.0
        v = y / scale
        return (torch.trunc(v + 0.5 * torch.sign(v)) * scale,)
    q, scales = torch.empty_like(y), torch.empty(M, -(-N // BLOCK), device=y.device, dtype=y.dtype)
    for i in range(scales.shape[1]):
        part = y[:, i * BLOCK:(i + 1) * BLOCK]
        scales[:, i] = part.abs().amax(1).clamp_min(1e-300) / 448.0
        q[:, i * BLOCK:(i + 1) * BLOCK] = _nearest_e4m3(part / scales[:, i:i + 1])
    return q, scales


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    op = case["op"]
    if op == "norm":
        h, kept = s["x"].double(), ()
        if case["residual"]:
            # the stream is held in bf16; two bf16 values add up without loss in 64 bits
            h = (h + s["residual"].double()).to(torch.bfloat16).double()
            kept = (h,)
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["N"] + EPS) * s["weight"].double()
        return _exact_quantized(y, case["out"]) + kept
    if op == "act":
        x = s["x"].double()
        gate, up = x[:, :case["N"]], x[:, case["N"]:]
        y = gate * (torch.special.ndtr(gate) if case["gelu"] else torch.sigmoid(gate)) * up
        return _exact_quantized(y, case["out"])
    M, N, K = case["M"], case["N"], case["K"]
    ends = s["offsets"].tolist() if op == "grouped" else [0, M]
    v = torch.zeros(M, N, device="cuda", dtype=torch.float64)
    for i, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if lo == hi:
            continue
        b = s["B"][i] if op == "grouped" else s["B"]
        b = b.double().t() if case["nk"] else b.double()
        a = s["A"][lo:hi].double()
        if "scale_a" not in s:
            v[lo:hi] = a @ b
            continue
        sb = (s["scale_b"][i] if op == "grouped" else s["scale_b"]).double()
        sb = sb.t() if case["nk"] else sb
        col = torch.arange(N, device="cuda") // BLOCK
        for k in range(-(-K // BLOCK)):
            at = slice(k * BLOCK, min(K, (k + 1) * BLOCK))
            v[lo:hi].addcmul_(a[:, at] @ b[at], s["scale_a"][lo:hi, k, None].double() * sb[k, col][None])
    if case["pair"] != "none":
        gate, up = v[:, ::2], v[:, 1::2]
        v = gate * (torch.special.ndtr(gate) if case["pair"] == "geglu" else torch.sigmoid(gate)) * up
    return v
