"""Products of ragged row groups (xf_grouped_gemm_*), bf16 and block-scaled e4m3, against 64-bit sums.

Tolerances, counted before the first run.  Products of two bf16 or e4m3 values are exact in fp32.  The tensor
core's running sum is held to one rounding of 2^-23 (truncation) of the sum of magnitudes per addend: K of them
for bf16, 128 within a block and one per block outside it for e4m3, where the block's factor sa * sb and
its product with the block's sum add two more.  Joining a tile's shared K range adds one rounding per
sharer, at most 148.  A bf16 result adds half a step, 2^-8 of the value (its subnormals are far below).
SwiGLU and GeGLU pass an error of the gate on with a slope of at most 1.13 times `up`, and add their own
(exponential 2 + 1.173 |x| ulp; erf 1.5e-7 of 1 + erf)."""
import ctypes as C

import pytest
import torch

U = 2.0 ** -24
E4M3 = torch.float8_e4m3fn
NAN = float("nan")


def up(n, m):
    return -(-n // m) * m


def make(M, N, K, sizes=None, dtype=E4M3, nk=False, before=0, seed=0, shared=False, sa_rows_last=True):
    """Operands; what lies behind a row of A or B, and the weights of empty groups, is NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + M * 31 + N * 17 + K)
    G = len(sizes) if sizes is not None else None
    pad = 16 if dtype == E4M3 else 8

    def rows(*shape):
        t = torch.randn(*shape[:-1], up(shape[-1], pad) + pad, generator=g, device="cuda")
        t = (t * 90).clamp(-448, 448) if dtype == E4M3 else t
        t[..., shape[-1]:] = NAN
        return t.to(dtype)[..., :shape[-1]]

    A = rows(M, K)
    shape = (N, K) if nk else (K, N)
    B = rows(*shape) if G is None or shared else rows(G, *shape)
    op = dict(A=A, B=B, b_nk=nk)
    if dtype == E4M3:
        kb, nb = up(K, 128) // 128, up(N, 128) // 128
        lead = () if B.dim() == 2 else (G,)
        sa = torch.rand(kb, M, generator=g, device="cuda").add_(0.5).div_(128)
        op["scale_a"] = sa.t() if sa_rows_last else sa.t().contiguous()
        op["scale_b"] = torch.rand(*lead, *((nb, kb) if nk else (kb, nb)), generator=g, device="cuda").add_(0.5).div_(16)
    if G is not None:
        ends = [before]
        for n in sizes:
            ends.append(ends[-1] + n)
        assert ends[-1] <= M
        op["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        if not shared:
            for i, n in enumerate(sizes):
                if n == 0:
                    B[i] = torch.full((1,), NAN, device="cuda").to(dtype)
    return op


def wide(scale, dim, n):
    return scale.double().repeat_interleave(128, dim).narrow(dim, 0, n)


def want(op, pair, lo, hi, g):
    """64-bit result of rows [lo, hi) with group g's weight, and the bound of its fp32 error."""
    A, B, K = op["A"][lo:hi].double(), op["B"], op["A"].shape[1]
    B = (B[g] if B.dim() == 3 else B).double()
    terms = K + 4
    if "scale_a" in op:
        sb = op["scale_b"][g] if op["scale_b"].dim() == 3 else op["scale_b"]
        A = A * wide(op["scale_a"][lo:hi], 1, K)
        B = B * wide(wide(sb, 0, B.shape[0]), 1, B.shape[1])
        terms = min(K, 128) + up(K, 128) // 128 + 4
    B = B.t() if op["b_nk"] else B
    v, e = A @ B, (A.abs() @ B.abs()) * (terms + 148) * 2 * U
    if pair == "none":
        return v, e
    a, b, ea, eb = v[:, 0::2], v[:, 1::2], e[:, 0::2], e[:, 1::2]
    act = a * (torch.sigmoid(a) if pair == "swiglu" else torch.special.ndtr(a))
    own = (2 * (2 + 1.173 * a.abs()) + 8) * U * act.abs() if pair == "swiglu" else 3e-7 * a.abs() + 8 * U * act.abs()
    return act * b, (1.13 * ea + own) * (b.abs() + eb) + act.abs() * eb + 4 * U * (act * b).abs()


def check(op, D, pair, before_D):
    M = op["A"].shape[0]
    ends = op["offsets"].tolist() if "offsets" in op else [0, M]
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi > lo:
            v, e = want(op, pair, lo, hi, g)
            e = e + (v.abs() + e) * (2.0 ** -8 if D.dtype == torch.bfloat16 else U) + 1e-37
            bad = ~((D[lo:hi].double() - v).abs() <= e)
            assert not bool(bad.any()), (g, lo, hi, int(bad.sum()), bad.nonzero()[:4].tolist(), D[lo:hi][bad][:4], v[bad][:4])
    assert torch.equal(D[:ends[0]], before_D[:ends[0]]) and torch.equal(D[ends[-1]:], before_D[ends[-1]:])


def tiles(capi, dtype):
    """Flags for: the planner's choice, then every tile, then the same without sharing the last wave's tiles."""
    forced = [capi.FLAG_FORCE_1CTA | capi.FLAG_FORCE_BN128, capi.FLAG_FORCE_2CTA]
    forced += [capi.FLAG_FORCE_1CTA | capi.FLAG_FORCE_BN256] if dtype == E4M3 else []
    return [0] + forced + [f | capi.FLAG_NO_SPLIT for f in forced]


def run(capi, op, dtype_d=torch.bfloat16, pair="none", flags=0, extra=0):
    M = op["A"].shape[0]
    N = op["B"].shape[-2 if op["b_nk"] else -1]
    cols = N if pair == "none" else N // 2
    whole = torch.full((M, cols + extra), -7.0, device="cuda", dtype=dtype_d)
    D = whole[:, :cols]
    before = D.clone()
    plan = capi.GroupedGemmPlan(op["A"], op["B"], D, offsets=op.get("offsets"), scale_a=op.get("scale_a"),
                                scale_b=op.get("scale_b"), b_nk=op["b_nk"], pair=pair, flags=flags)
    for _ in range(2):           # what a launch leaves in the workspace suits the next one
        plan.run()
    torch.cuda.synchronize()
    assert plan.device_status() == 0
    check(op, D, pair, before)
    assert bool((whole[:, cols:] == -7.0).all())
    return plan, D


DENSE = [(1, 8, 16), (1, 1, 1), (3, 127, 127), (128, 128, 128), (129, 130, 129), (7, 256, 1000), (300, 520, 4096),
         (64, 1000, 2048), (257, 24, 640), (1, 4096, 4096), (513, 1030, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", DENSE)
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_one_group(capi, cuda, M, N, K, nk, dtype):
    op = make(M, N, K, dtype=dtype, nk=nk)
    for flags in tiles(capi, dtype):
        run(capi, op, flags=flags)
    run(capi, op, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype_d", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pair", ["none", "swiglu", "geglu"])
@pytest.mark.parametrize("extra", [0, 3, 8])
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_outputs(capi, cuda, dtype_d, pair, extra, dtype):
    op = make(150, 390, 512, dtype=dtype)
    if dtype == torch.bfloat16:
        op["B"].mul_(512 ** -0.5)
    for flags in tiles(capi, dtype)[1:4]:
        run(capi, op, dtype_d, pair, extra=extra, flags=flags)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_geglu_of_negative_gates_keeps_its_relative_precision(capi, cuda, dtype):
    """Gates and factors that the product gives exactly (one-hot rows); errors as for the row pass, in units of U:
    __expf(g^2 / 2) 2 (2 + 1.173 g^2 / 2), the square and its exponent one rounding each, seen g^2 / 2 times larger, the
    rest of the activation 8, the reciprocal 8, the product with the factor 1."""
    K, pairs = 128, 72
    gate = -(1.25 + torch.arange(pairs, device=cuda).double() / 8).view(1, -1).expand(K, -1)
    gate = gate.to(dtype if dtype == E4M3 else torch.bfloat16).float()
    factor = torch.tensor([0.5, -1.0, 1.75], device=cuda)[torch.arange(pairs, device=cuda) % 3].expand(K, -1)
    B = torch.stack([gate, factor], 2).view(K, 2 * pairs).to(dtype)
    A = torch.eye(K, device=cuda)[:40].to(dtype)
    D = torch.empty(40, pairs, device=cuda)
    one = dict(scale_a=torch.ones(40, 1, device=cuda), scale_b=torch.ones(1, 2, device=cuda)) if dtype == E4M3 else {}
    capi.GroupedGemmPlan(A, B, D, pair="geglu", **one).run()
    torch.cuda.synchronize()
    g = gate[:40].double()
    want = g * torch.exp(torch.special.log_ndtr(g)) * factor[:40].double()
    assert bool(((D.double() - want).abs() <= (2 * (2 + 1.173 * g.square() / 2) + g.square() + 17) * U * want.abs()).all())


GROUPS = [([5], 5, 0), ([0, 3, 0, 0, 9, 1, 0], 13, 0), ([130, 1, 127, 128, 129], 515, 0), ([0, 0, 0], 4, 0), ([2, 3], 20, 7),
          ([300, 0, 2, 700], 1100, 40), ([1] * 70, 70, 0), ([0] * 1023 + [33], 33, 0), ([1, 0] * 512, 512, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(GROUPS)))
@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_groups(capi, cuda, case, nk, dtype):
    sizes, M, before = GROUPS[case]
    N, K = (72, 80) if len(sizes) > 100 else (264, 700)
    op = make(M, N, K, sizes, dtype, nk, before)
    for flags in tiles(capi, dtype):
        run(capi, op, flags=flags)
    run(capi, op, torch.float32, pair="swiglu" if dtype == E4M3 else "none")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_long_sums_and_many_tiles(capi, cuda, dtype):
    """A few tiles with a long K range (every sharing of a tile between CTAs), and more tiles than one wave."""
    for M, N, K, sizes in ((20, 300, 9000, None), (400, 300, 9000, None), (30, 200, 7000, [10, 0, 20]), (2100, 5200, 320, None),
                           (2600, 2000, 500, [900, 0, 1000, 3, 697])):
        op = make(M, N, K, sizes, dtype)
        for flags in tiles(capi, dtype):
            _, first = run(capi, op, torch.float32, flags=flags)
            _, again = run(capi, op, torch.float32, flags=flags)
            assert torch.equal(first, again)     # fixed order of every sum


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(19, 300, 7572), (300, 520, 4236), (5, 136, 16000)])
def test_long_sums_keep_their_precision(capi, cuda, dtype, M, N, K):
    """At most 256 elements are summed inside the tensor core, in 16 steps (e4m3: 128 in 4) that each drop at most 2^-23 of
    the partial sum; the pieces' sums are added with rounding.  Their errors and their sums add up alike, so the
    result is off by at most 16 * 2^-23 in the norm, plus a rounding for each of up to 126 pieces that adds
    up like its square root."""
    op = make(M, N, K, dtype=dtype)
    for flags in tiles(capi, dtype):
        _, D = run(capi, op, torch.float32, flags=flags)
        v, _ = want(op, "none", 0, M, 0)
        assert float((D.double() - v).norm() / v.norm()) < 16 * 2.0 ** -23 + 126 ** 0.5 * U


@pytest.mark.gpu
def test_scale_strides_and_shared_weight(capi, cuda):
    run(capi, make(70, 300, 520, sa_rows_last=False))
    run(capi, make(70, 300, 520, [30, 0, 40], shared=True))
    op = make(70, 300, 520, nk=True)
    op["scale_b"] = op["scale_b"].t().contiguous().t()
    run(capi, op)
    op["scale_a"] = op["scale_a"][:1].expand(70, -1)             # one factor for all rows: stride 0
    run(capi, op)


@pytest.mark.gpu
def test_rows_do_not_mix(capi, cuda):
    """A row of NaN or infinity stays in its own output row; a NaN scale in its rows and columns."""
    op = make(140, 260, 300, [60, 80])
    op["A"].view(torch.int8)[61, 7] = 0x7F                         # NaN
    op["scale_a"][3, 1] = float("inf")
    D = torch.empty(140, 260, device=cuda)
    capi.GroupedGemmPlan(op["A"], op["B"], D, offsets=op["offsets"], scale_a=op["scale_a"], scale_b=op["scale_b"]).run()
    torch.cuda.synchronize()
    bad = ~torch.isfinite(D).all(1)
    assert bad.nonzero().flatten().tolist() == [3, 61]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_routing_changes_under_a_graph(capi, cuda, dtype):
    op = make(300, 264, 520, [100, 0, 150, 50], dtype)
    op["B"] = make(4, 264, 520, [1, 1, 1, 1], dtype)["B"]      # every group may get rows
    D = torch.zeros(300, 264, device=cuda)
    plan = capi.GroupedGemmPlan(op["A"], op["B"], D, offsets=op["offsets"], scale_a=op.get("scale_a"), scale_b=op.get("scale_b"))
    plan.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run()
    for ends in ([0, 100, 100, 250, 300], [0, 0, 0, 0, 300], [0, 1, 2, 3, 4], [10, 10, 200, 201, 290], [5, 5, 5, 5, 5]):
        op["offsets"].copy_(torch.tensor(ends, dtype=torch.int32))
        D.fill_(-7.0)
        before = D.clone()
        graph.replay()
        torch.cuda.synchronize()
        check(op, D, "none", before)
    assert plan.device_status() == 0


@pytest.mark.gpu
def test_offsets_out_of_range_are_clamped(capi, cuda):
    """Offsets below zero and above M reach no row outside A and D."""
    op = make(200, 136, 256, [100, 100])
    whole = torch.full((400, 136), -7.0, device=cuda)
    D = whole[100:300]
    op["offsets"].copy_(torch.tensor([-50, 90, 100000], dtype=torch.int32))
    capi.GroupedGemmPlan(op["A"], op["B"], D, offsets=op["offsets"], scale_a=op["scale_a"], scale_b=op["scale_b"]).run()
    torch.cuda.synchronize()
    assert bool((whole[:100] == -7).all()) and bool((whole[300:] == -7).all())
    op["offsets"].copy_(torch.tensor([0, 90, 200], dtype=torch.int32))
    check(op, D, "none", D.clone())


@pytest.mark.gpu
def test_no_rows(capi, cuda):
    op = make(4, 64, 64, [2, 2])
    plan = capi.GroupedGemmPlan(op["A"][:0], op["B"], torch.empty(0, 64, device=cuda), offsets=op["offsets"],
                                scale_a=op["scale_a"][:0], scale_b=op["scale_b"])
    plan.run()
    torch.cuda.synchronize()
    assert plan.device_status() == 0


@pytest.mark.gpu
def test_status_is_reported_once(capi, cuda):
    """A code in the status word, as a wait that gave up leaves one, is an error at the next query and then gone."""
    op = make(20, 300, 9000)
    plan, D = run(capi, op)
    plan.workspace[:4].view(torch.int32).fill_(3)
    torch.cuda.synchronize()
    with pytest.raises(capi.XfError, match="device code 3"):
        plan.device_status()
    assert plan.device_status() == 0
    plan.run()
    torch.cuda.synchronize()
    check(op, D, "none", D)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["all", "one CTA", "one warp"])
@pytest.mark.parametrize("shape", [(20, 300, 9000), (2100, 5200, 4096)])
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_a_wait_that_gives_up(capi, cuda, dtype, shape, which):
    """The flags that say "partial sums are there" start so far below zero that they never rise above it: with short waits
    the collecting warps give up after about a millisecond.  The launch ends (2100 x 5200: every unit has whole tiles
    behind the shared one, so the other roles' waits run out as well, at different blocks), the status is reported
    once, and the plan then runs as before."""
    op = make(*shape, dtype=dtype)
    D = torch.empty(shape[0], shape[1], device=cuda)
    for flags in [0] + [f for f in tiles(capi, dtype)[1:] if not f & capi.FLAG_NO_SPLIT]:
        plan = capi.GroupedGemmPlan(op["A"], op["B"], D, scale_a=op.get("scale_a"), scale_b=op.get("scale_b"),
                                    flags=flags | capi.FLAG_SHORT_WAITS)
        plan.run()
        torch.cuda.synchronize()
        assert plan.device_status() == 0
        good = D.clone()
        words = plan.workspace[256:].view(torch.int32)
        words[:{"all": 148 * 8, "one CTA": 8, "one warp": 1}[which]] = -1000000
        torch.cuda.synchronize()
        plan.run()
        torch.cuda.synchronize()                                 # returns: every wait is bounded
        with pytest.raises(capi.XfError, match="device code [1-5]"):
            plan.device_status()
        assert plan.device_status() == 0
        for _ in range(2):
            D.fill_(-7.0)
            plan.run()
            torch.cuda.synchronize()
            assert plan.device_status() == 0
            assert torch.equal(D, good)
    check(op, good, "none", good)


@pytest.mark.gpu
def test_plans_on_two_streams(capi, cuda):
    """Two plans with workspaces of their own, whose tiles are shared between CTAs, run at once."""
    ops = [make(40, 700, 8000, seed=s) for s in (1, 2)]
    outs = [torch.empty(40, 700, device=cuda) for _ in ops]
    plans = [capi.GroupedGemmPlan(o["A"], o["B"], D, scale_a=o["scale_a"], scale_b=o["scale_b"]) for o, D in zip(ops, outs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(20):
        for plan, s in zip(plans, streams):
            with torch.cuda.stream(s):
                plan.run()
    torch.cuda.synchronize()
    for o, D, plan in zip(ops, outs, plans):
        assert plan.device_status() == 0
        check(o, D, "none", D)


def renew(op, other):
    """Puts another operand set's values in place of this one's."""
    for k in ("A", "B"):
        if op[k].dtype == E4M3:
            op[k].view(torch.int8).copy_(other[k].view(torch.int8))
        else:
            op[k].copy_(other[k])
    for k in ("scale_a", "scale_b"):
        if k in op:
            op[k].copy_(other[k])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(20, 300, 9000), (400, 300, 9000), (2100, 1300, 4096)])
def test_shared_tiles_meet_new_data(capi, cuda, dtype, M, N, K):
    """Tiles whose K range several CTAs share, launch after launch with new operands and the old result overwritten: sums
    that an earlier launch published, or a flag that it left raised, would show in the result."""
    sets = [make(M, N, K, dtype=dtype, seed=s) for s in (1, 2, 3)]
    op = make(M, N, K, dtype=dtype, seed=4)
    D = torch.empty(M, N, device=cuda)
    plans = [capi.GroupedGemmPlan(op["A"], op["B"], D, scale_a=op.get("scale_a"), scale_b=op.get("scale_b"), flags=f)
             for f in tiles(capi, dtype) if not f & capi.FLAG_NO_SPLIT]
    assert all(plan.workspace.numel() > 256 for plan in plans)       # they may share tiles
    for plan in plans:
        got = []
        for i in (0, 1, 2, 1, 0):                                    # no pause: one launch's end meets the next one's start
            renew(op, sets[i])
            D.fill_(-7.0)
            plan.run()
            got.append((i, D.clone()))
        assert plan.device_status() == 0
        for i, D_i in got:
            check(sets[i], D_i, "none", D_i)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_routing_of_shared_tiles_changes_under_a_graph(capi, cuda, dtype):
    """K = 8000 and few row tiles: every launch shares its tiles, other ones each time, among other CTAs."""
    M, N, K = 300, 264, 8000
    sets = [make(M, N, K, [75] * 4, dtype, seed=s) for s in (1, 2)]
    for flags in tiles(capi, dtype):
        if flags & capi.FLAG_NO_SPLIT:
            continue
        op = make(M, N, K, [75] * 4, dtype, seed=3)
        D = torch.zeros(M, N, device=cuda)
        plan = capi.GroupedGemmPlan(op["A"], op["B"], D, offsets=op["offsets"], scale_a=op.get("scale_a"),
                                    scale_b=op.get("scale_b"), flags=flags)
        plan.run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run()
        for i, ends in enumerate(([0, 100, 100, 250, 300], [0, 0, 0, 0, 300], [0, 1, 2, 3, 4], [10, 10, 200, 201, 290],
                                  [5, 5, 5, 5, 5], [0, 299, 299, 299, 300], [0, 100, 100, 250, 300])):
            renew(op, sets[i % 2])
            op["offsets"].copy_(torch.tensor(ends, dtype=torch.int32))
            D.fill_(-7.0)
            before = D.clone()
            graph.replay()
            check(op, D, "none", before)
        assert plan.device_status() == 0


@pytest.mark.gpu
def test_plans_on_two_streams_meet_new_data(capi, cuda):
    """Two plans with workspaces of their own and shared tiles at once, each launch on other operands."""
    sets = [[make(40, 700, 8000, seed=10 * p + s) for s in range(3)] for p in (1, 2)]
    ops = [make(40, 700, 8000, seed=p) for p in (5, 6)]
    outs = [torch.empty(40, 700, device=cuda) for _ in ops]
    plans = [capi.GroupedGemmPlan(o["A"], o["B"], D, scale_a=o["scale_a"], scale_b=o["scale_b"]) for o, D in zip(ops, outs)]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    got = [[], []]
    for step in range(9):
        for p, s in enumerate(streams):
            with torch.cuda.stream(s):
                renew(ops[p], sets[p][step % 3])
                outs[p].fill_(-7.0)
                plans[p].run()
                got[p].append(outs[p].clone())
    torch.cuda.synchronize()
    for p in (0, 1):
        assert plans[p].device_status() == 0
        for step, D in enumerate(got[p]):
            check(sets[p][step % 3], D, "none", D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, torch.bfloat16])
def test_shared_tiles_beside_other_work(capi, cuda, dtype):
    """While large products of another stream hold SMs, a launch's CTAs start one after another: those that collect
    partial sums only wait for CTAs of lower index, which have started before them."""
    sets = [make(300, 700, 8000, dtype=dtype, seed=s) for s in (1, 2, 3)]
    a = torch.randn(8192, 8192, device=cuda).to(torch.bfloat16)
    op = make(300, 700, 8000, dtype=dtype, seed=4)
    D = torch.empty(300, 700, device=cuda)
    side = torch.cuda.Stream()
    for flags in [f for f in tiles(capi, dtype) if not f & capi.FLAG_NO_SPLIT]:
        plan = capi.GroupedGemmPlan(op["A"], op["B"], D, scale_a=op.get("scale_a"), scale_b=op.get("scale_b"), flags=flags)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(4):
                b = a @ a
        got = []
        for i in range(12):
            renew(op, sets[i % 3])
            D.fill_(-7.0)
            plan.run()
            got.append(D.clone())
        torch.cuda.synchronize()
        assert plan.device_status() == 0
        for i, D_i in enumerate(got):
            check(sets[i % 3], D_i, "none", D_i)


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [False, True])
def test_feed_forward_in_8_bits(capi, cuda, experts):
    """norm + quantise -> gate/up product -> activation + quantise -> down product, captured in one graph."""
    M, H, F = 96, 512, 384
    sizes = [40, 0, 56] if experts else None
    gate_up, down = make(M, 2 * F, H, sizes, seed=1), make(M, H, F, sizes, nk=True, seed=2)
    off = gate_up.get("offsets")
    x = torch.randn(M, H, device=cuda).to(torch.bfloat16)
    first_x = x.clone()
    res = torch.randn(M, H, device=cuda).to(torch.bfloat16)
    w = torch.rand(H, device=cuda).to(torch.bfloat16)
    h = torch.empty_like(x)
    up_out = torch.empty(M, 2 * F, device=cuda, dtype=torch.bfloat16)
    y = torch.empty(M, H, device=cuda)
    p1 = capi.GroupedGemmPlan(gate_up["A"], gate_up["B"], up_out, offsets=off, scale_a=gate_up["scale_a"], scale_b=gate_up["scale_b"])
    p2 = capi.GroupedGemmPlan(down["A"], down["B"], y, offsets=off, scale_a=down["scale_a"], scale_b=down["scale_b"], b_nk=True)

    def layer():
        capi.rms_norm_quantize(gate_up["A"], gate_up["scale_a"], x, w, res, h)
        p1.run()
        capi.act_mul_quantize(down["A"], down["scale_a"], up_out)
        p2.run()

    layer()
    torch.cuda.synchronize()
    assert torch.equal(h, (x.float() + res.float()).to(torch.bfloat16))
    check(gate_up, up_out, "none", up_out)
    check(down, y, "none", y)
    first = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, y)
    # new inputs without a pause between the calls: no kernel reads what an earlier one left in a cache
    xs = [torch.randn(M, H, device=cuda).to(torch.bfloat16) for _ in range(12)]
    def all_of(wait):
        got = []
        for v in xs:
            x.copy_(v)
            layer()
            got.append(y.clone())
            if wait:
                torch.cuda.synchronize()
        return got
    for one, other in zip(all_of(True), all_of(False)):
        assert torch.equal(one, other)
    x.copy_(first_x)
    layer()
    # against the same layer in 64 bits without any quantisation: 8-bit steps of 2^-4 at three places
    ends = off.tolist() if experts else [0, M]
    n = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + 1e-6) * w.double()
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        b1 = gate_up["B"][g] if experts else gate_up["B"]
        s1 = gate_up["scale_b"][g] if experts else gate_up["scale_b"]
        b2 = down["B"][g] if experts else down["B"]
        s2 = down["scale_b"][g] if experts else down["scale_b"]
        if hi > lo:
            v = n[lo:hi] @ (b1.double() * wide(wide(s1, 0, H), 1, 2 * F))
            a = v[:, :F] * torch.sigmoid(v[:, :F]) * v[:, F:]
            full = a @ (b2.double() * wide(wide(s2, 0, H), 1, F)).t()
            # each 8-bit code is off by at most 2^-4 of its value, roughly uniformly: about 2^-4 / sqrt(3) in the
            # mean square for the input and again for the activation, which also doubles the first one's error
            assert float((y[lo:hi].double() - full).norm() / full.norm()) < 3 * 2.0 ** -4


@pytest.mark.gpu
def test_offsets_past_32_bits(capi, cuda):
    """Rows of A and D that start beyond 4 GB, and weights of a group beyond it."""
    M, N, K, pitch = 70000, 64, 96, 65536
    op = make(40, N, K, [40])
    A = torch.empty(M, pitch, device=cuda, dtype=torch.int8).view(E4M3)[:, :K]
    A[-40:].view(torch.int8).copy_(op["A"].view(torch.int8))
    B = torch.empty(1 << 33, device=cuda, dtype=torch.int8).view(E4M3).as_strided((3, K, N), ((1 << 32) - 4096 * 16, N, 1))
    B[2].view(torch.int8).copy_(op["B"][0].view(torch.int8))
    sa = torch.ones(M, 1, device=cuda)
    sa[-40:] = op["scale_a"]
    sb = op["scale_b"].expand(3, -1, -1)
    D = torch.empty(M, pitch // 2, device=cuda, dtype=torch.bfloat16)[:, :N]
    off = torch.tensor([M - 40, M - 40, M - 40, M], dtype=torch.int32, device=cuda)
    for flags in tiles(capi, E4M3):
        D[-40:] = 0
        capi.GroupedGemmPlan(A, B, D, offsets=off, scale_a=sa, scale_b=sb, flags=flags).run()
        torch.cuda.synchronize()
        check(op, D[-40:].contiguous(), "none", D[-40:])


# ------------------------------------------------------------------ refusals: no GPU is touched
def desc(capi, **k):
    d = capi.XfGroupedGemmDesc()
    v = dict(dtype_ab=4, dtype_d=0, M=64, N=256, K=256, num_groups=1, A=0x10000, lda=256, B=0x20000, ldb=256, batch_b=0,
             scale_a=0x30000, scale_a_row_stride=1, scale_a_blk_stride=64, scale_b=0x40000, scale_b_k_stride=2,
             scale_b_n_stride=1, D=0x50000, ldd=256, workspace_bytes=0)
    v.update(k)
    for name, x in v.items():
        setattr(d, name, x)
    return d


@pytest.mark.parametrize("change,status", [
    ({}, 0), (dict(M=0, A=None, D=None, scale_a=None), 0),
    (dict(dtype_ab=1), 2), (dict(dtype_d=3), 2), (dict(M=-1), 4), (dict(N=0), 4), (dict(K=0), 4), (dict(num_groups=0), 4),
    (dict(num_groups=1025, group_offsets=0x60000), 5), (dict(num_groups=2), 4), (dict(b_layout=2), 3), (dict(pair=3), 5),
    (dict(pair=1, N=255), 4), (dict(pair=1, ldd=128), 0), (dict(lda=240), 3), (dict(ldb=240), 3), (dict(ldd=255), 3),
    (dict(num_groups=2, group_offsets=0x60000, batch_b=1024), 3), (dict(A=None), 4), (dict(B=None), 4), (dict(D=None), 4),
    (dict(A=0x10008), 1), (dict(B=0x20001), 1), (dict(lda=264), 1), (dict(ldb=257), 1), (dict(D=0x50001), 1),
    (dict(num_groups=2, group_offsets=0x60000, batch_b=65544), 1), (dict(group_offsets=0x60002), 1), (dict(scale_a=None), 4),
    (dict(scale_b=None), 4), (dict(scale_a=0x30002), 1), (dict(scale_a_row_stride=-1), 3), (dict(dtype_ab=0), 4),
    (dict(dtype_ab=0, scale_a=None, scale_b=None), 0), (dict(flags=1), 5), (dict(M=1 << 30, N=1 << 20, ldb=1 << 20, ldd=1 << 20), 5),
])
def test_refusals(capi, change, status):
    assert capi.lib().xf_grouped_gemm_can_implement(C.byref(desc(capi, **change))) == status


@pytest.mark.parametrize("bf16,flags,status", [
    (0, ("1CTA", "BN256"), 0), (0, ("2CTA", "BN256"), 0), (0, ("1CTA", "BN128"), 0), (0, ("BN128",), 0), (0, ("2CTA",), 0),
    (0, ("2CTA", "BN128"), 5), (0, ("1CTA", "2CTA"), 5), (0, ("BN128", "BN256"), 5),
    (1, ("2CTA", "BN256"), 0), (1, ("1CTA", "BN128"), 0), (1, ("1CTA", "BN256"), 5), (1, ("2CTA", "BN128"), 5)])
def test_flags_that_leave_no_tile_are_refused_at_once(capi, bf16, flags, status):
    word = sum(getattr(capi, "FLAG_FORCE_" + f) for f in flags)
    more = dict(dtype_ab=0, scale_a=None, scale_b=None) if bf16 else {}
    assert capi.lib().xf_grouped_gemm_can_implement(C.byref(desc(capi, flags=word, **more))) == status


@pytest.mark.parametrize("big", [dict(M=2 ** 31 - 255), dict(N=2 ** 31 - 255, ldb=2 ** 31, ldd=2 ** 31),
                                 dict(K=2 ** 31 - 255, lda=2 ** 31)])
def test_extents_next_to_32_bits(capi, big):
    """An extent that leaves 32 bits when it is rounded up to a tile is refused, the largest one that does not is taken."""
    name = next(iter(big))
    assert capi.lib().xf_grouped_gemm_can_implement(C.byref(desc(capi, **big))) == 5
    assert capi.lib().xf_grouped_gemm_can_implement(C.byref(desc(capi, **{**big, name: 2 ** 31 - 256}))) == 0


def test_wrapper_refuses_extents_beyond_32_bits(capi, monkeypatch):
    """They would wrap around in the descriptor."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    A, B, D = torch.zeros(8, 256, dtype=torch.bfloat16), torch.zeros(256, 128, dtype=torch.bfloat16), torch.zeros(8, 128)
    M = 2 ** 32 + 8
    with pytest.raises(capi.XfError, match="32-bit"):
        capi.GroupedGemmPlan(A[:1].expand(M, -1), B, D[:1].expand(M, -1))


def test_null_arguments(capi):
    L = capi.lib()
    assert L.xf_grouped_gemm_can_implement(None) == 4
    assert L.xf_grouped_gemm_workspace_size(None, None) == 4
    assert L.xf_grouped_gemm_plan_create(C.byref(desc(capi)), None, None, None) == 4
    assert L.xf_grouped_gemm_run(None, None) == 4
    assert L.xf_grouped_gemm_plan_device_status(None, None) == 4
    assert L.xf_grouped_gemm_plan_kernel_name(None) == b""
    assert L.xf_grouped_plan_destroy(None) == 0


def test_wrapper_refusals(capi, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)       # what a CPU tensor reports
    A, B, D = torch.zeros(8, 256, dtype=E4M3), torch.zeros(256, 128, dtype=E4M3), torch.zeros(8, 128)
    sa, sb, off = torch.ones(8, 2), torch.ones(2, 1), torch.zeros(3, dtype=torch.int32)
    for a, k in (
        ((A, B.to(torch.bfloat16), D), dict(scale_a=sa, scale_b=sb)),
        ((A, B, D), dict()),                                                   # no scales
        ((A, B, D), dict(scale_a=sa[:, :1], scale_b=sb)),
        ((A, B, D), dict(scale_a=sa, scale_b=sb.t())),
        ((A, B, D[:4]), dict(scale_a=sa, scale_b=sb)),
        ((A, B, D), dict(scale_a=sa, scale_b=sb, pair="swiglu")),              # D is [M, N / 2] then
        ((A, B[:128], D), dict(scale_a=sa, scale_b=sb)),
        ((A, B[None].expand(3, -1, -1), D), dict(scale_a=sa, scale_b=sb, offsets=off)),
        ((A, B, D), dict(scale_a=sa, scale_b=sb, offsets=off.long())),
        ((A, B.t().contiguous().t(), D), dict(scale_a=sa, scale_b=sb)),
    ):
        with pytest.raises(capi.XfError):
            capi.GroupedGemmPlan(*a, **k)


def test_wrapper_refuses_types_and_shapes_in_its_own_manner(capi, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    A, B, D = torch.zeros(8, 256, dtype=E4M3), torch.zeros(256, 128, dtype=E4M3), torch.zeros(8, 128)
    k = dict(scale_a=torch.ones(8, 2), scale_b=torch.ones(2, 1))
    half = [t.to(torch.float16) for t in (A.float(), B.float())]
    for a, more in (
        ((A, B, D.half()), k),                                       # no such result
        ((half[0], half[1], D), {}),                                 # nor such operands
        ((A[0], B, D), k), ((A[None], B, D), k), ((A, B[0], D), k), ((A, B[None, None], D), k),
        ((A, B, D[0]), k), ((A, B, D[None]), k),
        ((A, B, D), dict(k, offsets=torch.zeros((), dtype=torch.int32))),
        ((A, B, D), dict(k, offsets=torch.zeros(0, dtype=torch.int32))),
        ((A, B, D), dict(k, offsets=torch.zeros(1, 2, dtype=torch.int32))),
        ((A, B, D), dict(k, pair="relu")),
        ((A, B, D), dict(k, scale_a=torch.ones(8))),
    ):
        with pytest.raises(capi.XfError):
            capi.GroupedGemmPlan(*a, **more)
