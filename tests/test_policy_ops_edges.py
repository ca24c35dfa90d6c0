"""rlgymppo_cpp_amd.ops at the edges of what its calls accept: mask constants and temperatures of any size, logits next to the type's lowest value, infinities among
a row's inputs, gradients of 40 decades, what autograd is told.  The definitions in 64 bits and the tolerances are those of test_policy_ops."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from rlgymppo_cpp_amd import _lib, ops
from test_policy_ops import (DTYPES, FLOOR, U, check, check_clip, half_step, loss_inputs, make, ref_gradient, ref_loss, ref_rows, tol_entropy, tol_gradient,
                             tol_logp)

gpu = pytest.mark.gpu


def check_row_calls(x, act, mask, temperature, g, some=None, size=1.0):
    """All three calls on rows `some` of x against 64 bits; gradients of `size`; forbidden actions have exactly no gradient.  x, act, mask are on the CPU."""
    rows, A = x.shape
    dtype = x.dtype
    some = torch.arange(rows) if some is None else some
    xg, ag, mg = x.cuda(), act.cuda(), None if mask is None else mask.cuda()
    sub = (x[some], act[some], None if mask is None else mask[some])
    # logits that are masks by themselves
    ok = ~(sub[0] <= (-65504.0 if dtype is torch.float16 else -1.875 * 2.0 ** 122))
    ok = ok if mask is None else ok & sub[2]
    clean = torch.where(ok, sub[0], torch.zeros_like(sub[0]))
    r = ref_rows(clean, sub[1], ok, temperature)
    zero = torch.zeros(len(some), dtype=torch.float64)
    forbidden = ~ok
    logp, H = ops.action_logp(xg, ag, mg, temperature=temperature)
    check(logp[some], r["logp"], tol_logp(r, A), "logp")
    check(H[some], r["H"], tol_entropy(r, A), "entropy")
    dl, dh = size * torch.randn(rows, generator=g), size * torch.randn(rows, generator=g)
    c, h = torch.where(r["floored"] | ~r["on"], 0.0, dl[some].double()), torch.where(r["on"], dh[some].double(), 0.0)
    want = ref_gradient(r, c, h, temperature)
    for out in (None, xg.clone()):
        got = ops.action_logp_backward(xg if out is None else out, ag, dl.cuda(), dh.cuda(), mg, temperature=temperature, out=out)[some]
        check(got, want, tol_gradient(r, c, h, zero, want, dtype, temperature), f"dlogits (in place: {out is not None})")
        assert (got[forbidden.cuda()] == 0).all()
    old, adv, ref = loss_inputs(rows, g, torch.zeros(rows, dtype=torch.float64))
    old[some] += r["logp"].float()
    ref[some] += r["logp"].float()
    rr, rho, d, ww, c, h, per_row = ref_loss(clean, sub[1], old[some], adv[some], ref[some], ok, None, ent=0.01, kl=0.1, temperature=temperature, scale=size)
    want = ref_gradient(rr, c, h, temperature)
    step = tol_logp(r, A) + 8 * U + U * (old[some].double().abs() + ref[some].double().abs() + r["logp"].abs())
    dc = rr["on"].double() * size * (rho * adv[some].double().abs() + 0.1 * (torch.exp(d) + 1)) * step
    for out in (None, xg.clone()):
        res = ops.policy_loss(xg if out is None else out, ag, old.cuda(), adv.cuda(), ref.cuda(), mg, ent_coef=0.01, kl_coef=0.1, temperature=temperature, scale=size, out=out)
        check(res.logp[some], r["logp"], tol_logp(r, A), "loss: logp")
        check(res.dlogits[some], want, tol_gradient(rr, c, h, dc, want, dtype, temperature), f"loss: dlogits (in place: {out is not None})")
        assert (res.dlogits[some][forbidden.cuda()] == 0).all()
    if len(some) == rows:
        th, on = tol_entropy(r, A), rr["on"].double()
        check(res.stats[ops.STAT_ENTROPY], per_row[0].sum(), (on * th).sum() + U * per_row[0].abs().sum(), "loss: entropy")
        check(res.stats[ops.STAT_LOSS], per_row[6].sum(), (dc + on * size * 0.01 * th).sum() + U * per_row[6].abs().sum(), "loss")
        assert res.stats[ops.STAT_ROWS] == per_row[5].sum()


# ---- masks by large negative logits ----------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("low,temperature", [(-1e9, 0.6), (-2e9, 1.2), (-4e9, 2.4), (-3e9, 1.0)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("A,rows,front", [(30, 9, 7), (90, 9, 22), (700, 9, 175), (700, 9, 20), (9000, 9, 2250), (9000, 9, 20), (40000, 9, 10000), (40000, 9, 20), (40000, 131, 20)])
def test_masked_by_a_large_negative_logit(A, rows, front, dt, low, temperature):
    """A lane that has nothing but the caller's -1e9: its exponents are past 2^30, where the rounding of one is itself an exponent of up to 2^7."""
    _, x, act, _, g = make(rows, A, DTYPES[dt], seed=12, temperature=temperature)
    x = x.clone()
    x[:, front:] = low
    act = (act % front).to(torch.int32)
    check_row_calls(x, act, None, temperature, g, some=torch.arange(min(rows, 9)))


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_masked_by_a_large_negative_logit_of_any_size(dt):
    """Mask constants over six decades and temperatures about 1: 20 logits in front of 70 of the constant."""
    g = torch.Generator().manual_seed(3)
    front = torch.randn((3, 20), generator=g)
    for low in [-(10.0 ** (e / 7)) for e in range(49, 92)]:
        for temperature in (0.45, 0.5, 0.6, 0.7, 0.77, 0.9, 1.0, 1.1, 1.2, 1.3, 1.7, 2.3):
            x = torch.full((3, 90), low)
            x[:, :20] = front
            x = x.to(DTYPES[dt])
            act = torch.tensor([0, 5, 19], dtype=torch.int32)
            r = ref_rows(x, act, None, temperature)
            logp, H = ops.action_logp(x.cuda(), act.cuda(), temperature=temperature)
            check(logp, r["logp"], tol_logp(r, 90), f"logp, {low} at {temperature}")
            check(H, r["H"], tol_entropy(r, 90), f"entropy, {low} at {temperature}")


@gpu
@pytest.mark.parametrize("temperature", [1.0, 1e-3])
@pytest.mark.parametrize("base", [1.5e9, 1.9e9, 3.9e9, -1.9e9, 7e9, 1.7e10, 1.3e20])
@pytest.mark.parametrize("A,rows", [(90, 200), (700, 200), (9000, 150), (20000, 100), (20000, 130)])
def test_largest_values_of_one_rounded_exponent(A, rows, base, temperature):
    """Far rows whose largest logits are one or two of float32's steps apart, so that their rounded exponents may be one: the largest has all of the probability."""
    g = torch.Generator().manual_seed(A + rows)
    base = base * temperature
    a = (base * (1 + 0.1 * torch.rand(rows, generator=g).double())).float()
    x = a[:, None].expand(rows, A).clone()
    x[:, ::7] -= abs(base) / 1000
    inf = torch.full_like(a, math.inf)
    act = torch.randint(0, A, (rows,), generator=g)
    x[torch.arange(rows), act] = torch.nextafter(a, inf)
    two = torch.arange(rows) % 2 == 0
    x[torch.arange(rows)[two], act[two]] = torch.nextafter(torch.nextafter(a, inf), inf)[two]
    check_row_calls(x, act.to(torch.int32), None, temperature, g, some=torch.randperm(rows, generator=g)[:64].sort().values if A > 5000 else None)


@gpu
@pytest.mark.parametrize("temperature", [1.0, 1.25, 0.6, 1e-3])
@pytest.mark.parametrize("border", [1e8, -1e8, 5e7, -5e7])
@pytest.mark.parametrize("A,rows", [(60, 300), (700, 60), (9000, 9), (40000, 9), (40000, 130)])
def test_rows_across_the_border_of_far(A, rows, border, temperature):
    """Exponents within a few steps of where they count as far, on both sides of it in one row, in one lane, in one part."""
    g = torch.Generator().manual_seed(A)
    x = torch.full((rows, A), border / math.log2(math.e) * temperature, dtype=torch.float64)
    ulp = abs(float(torch.nextafter(x[0, 0].float(), torch.tensor(math.inf))) - float(x[0, 0].float()))
    x = (x + ulp * torch.randint(-3, 4, (rows, 1), generator=g) - ulp * torch.randint(0, 3, (rows, A), generator=g)).float()
    act = torch.randint(0, A, (rows,), generator=g).to(torch.int32)
    check_row_calls(x, act, None, temperature, g, some=torch.randperm(rows, generator=g)[:64].sort().values if A > 5000 else None)


# ---- temperatures at which a type's lowest value is an ordinary exponent ------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("temperature", [500.0, 1e3, 2600.0, 1e4, 1e5])
@pytest.mark.parametrize("A,rows", [(5, 9), (30, 9), (90, 67), (90, 1), (129, 9), (700, 9), (3001, 9), (9001, 9), (21001, 131), (50021, 1), (50021, 9), (50021, 131), (140001, 131)])
def test_float16_at_high_temperatures(A, rows, temperature, masked):
    """Forbidden actions and empty places have no probability, whatever 65504 / T is."""
    _, x, act, mask, g = make(rows, A, torch.float16, seed=13, masked=masked, temperature=min(temperature, 3000.0))
    if masked and rows > 4:
        mask[4] = False
    some = None if rows * A < 2_000_000 else torch.tensor([0, 1, 2, 4, rows - 1])
    check_row_calls(x, act, mask, temperature, g, some=some, size=temperature)


@gpu
def test_a_forbidden_action_stays_at_the_floor():
    """... also under a floor that is float32's smallest number."""
    for dtype, temperature in [(torch.float16, t) for t in (1.0, 400.0, 700.0, 2600.0, 1e4, 1e6)] + [(torch.float32, 1e36), (torch.bfloat16, 1e36)]:
        for A in (6, 90, 700, 40000):
            x = torch.zeros((5, A), dtype=dtype, device="cuda")
            mask = torch.ones((5, A), dtype=torch.bool, device="cuda")
            mask[:, 1] = False
            act = torch.ones(5, dtype=torch.int32, device="cuda")
            for floor in (1e-11, 1e-45):
                logp, H = ops.action_logp(x, act, mask, temperature=temperature, min_prob=floor)
                assert (logp == np.float32(math.log(np.float32(floor)))).all(), (dtype, temperature, A)
                assert (H.double() - math.log(A - 1)).abs().max() <= U * 2000 * math.log(A)


@gpu
@pytest.mark.parametrize("temperature", [1.0, 10.0, 100.0])
@pytest.mark.parametrize("A,rows", [(30, 9), (90, 9), (1003, 9), (50021, 9), (50021, 131)])
def test_float16_logits_next_to_the_lowest(A, rows, temperature):
    """Rows whose largest logits are a few steps above -65504, some logits at it, in masked places too."""
    g = torch.Generator().manual_seed(A)
    x = (-65504.0 + 32.0 * torch.randint(0, 12, (rows, A), generator=g)).half()
    act = torch.randint(0, A, (rows,), generator=g).to(torch.int32)
    mask = torch.rand((rows, A), generator=g) < 0.7
    mask[torch.arange(rows), act.long()] = True
    x[2] = -65504.0                                         # left out
    some = None if rows * A < 2_000_000 else torch.tensor([0, 1, 2, 4, rows - 1])
    check_row_calls(x, act, mask, temperature, g, some=some)
    check_row_calls(x, act, None, temperature, g, some=some)


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("A,rows", [(30, 9), (90, 9), (1003, 9), (20011, 9), (50021, 9), (50021, 131)])
def test_temperatures_near_the_largest_number(A, rows, dt, masked):
    """Forbidden actions where float32's and bfloat16's numbers end as well."""
    for temperature in (1e34, 1e35, 1e36):
        _, x, act, mask, g = make(rows, A, DTYPES[dt], seed=14, masked=masked)
        x = (x.float() * (temperature / 4)).to(DTYPES[dt])
        some = None if rows * A < 2_000_000 else torch.tensor([0, 1, 2, 4, rows - 1])
        check_row_calls(x, act, mask, temperature, g, some=some, size=1e30)


@gpu
@pytest.mark.parametrize("how", ["mask", "-inf", "-1e20", "none"])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("A,rows", [(6, 9), (90, 9), (1003, 9), (20011, 9), (50021, 9)])
def test_temperatures_near_the_smallest_number(A, rows, dt, how):
    """Gradients of 1 / T = 10^35 beside actions that have no probability at all: those get 0."""
    for temperature in (1e-30, 1e-35, 2.3e-36):
        _, x, act, mask, g = make(rows, A, DTYPES[dt], seed=15, masked=True)
        x = (x.float() * temperature).to(DTYPES[dt])
        x[:, 0] -= 1e-20                                    # (far below, whatever the mask)
        if how in ("-inf", "-1e20"):
            x = torch.where(mask, x, torch.full_like(x, float(how)))
        act[act == 0] = A - 1
        check_row_calls(x, act, mask if how == "mask" else None, temperature, g, size=0.5)


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("A", [90, 700, 40000])
def test_where_a_row_begins_to_count(A, dt):
    """A logit of -9.5e36 is one as any other; -1e37 is a mask (the limit is between them, -9.97e36)."""
    x = torch.full((4, A), -1e37, dtype=DTYPES[dt], device="cuda")
    x[0, 3] = -9.5e36
    x[1] = -9.5e36
    x[2, 3] = -math.inf
    act = torch.full((4,), 3, dtype=torch.int32, device="cuda")
    logp, H = ops.action_logp(x, act)
    assert logp[0] == 0 and H[0] == 0
    assert abs(float(logp[1]) + math.log(A)) < 1e-5 and abs(float(H[1]) - math.log(A)) < 1e-5
    assert (logp[2:] == 0).all() and (H[2:] == 0).all()
    d = ops.action_logp_backward(x, act, torch.ones(4, device="cuda"))
    assert (d[2:] == 0).all() and float(d[1, 3]) > 0.9 and (d[0] == 0).all()


# ---- what is not finite ------------------------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("A", [6, 90, 700, 9001, 40001])
def test_forbidden_actions_have_no_gradient_whatever_the_row_has(A, dt):
    """Infinite and NaN gradients from above, and NaN and infinite logits among the allowed ones, do not reach the places that the mask forbids."""
    dtype = DTYPES[dt]
    g = torch.Generator().manual_seed(A)
    R = 10
    x = torch.randn((R, A), generator=g).to(dtype)
    mask = torch.rand((R, A), generator=g) < 0.5
    act = torch.full((R,), 1, dtype=torch.int32)
    mask[:, 1] = True
    mask[:, 2] = True
    mask[:, 3] = False
    act[7] = act[8] = 3                                     # forbidden actions
    x[~mask] = math.nan
    x[4, 2], x[5, 2], x[8, 2] = math.nan, math.inf, math.nan
    dl = torch.tensor([math.inf, math.nan, 1.0, 1.0, 1.0, 1.0, -math.inf, 1.0, 3e38, 1.0])
    dh = torch.tensor([1.0, 0.0, math.inf, math.nan, 1.0, 1.0, 1.0, math.inf, 1.0, 3e38])
    xg, ag, mg = x.cuda(), act.cuda(), mask.cuda()
    for temperature in (1.0, 0.01, 3e3):
        d = ops.action_logp_backward(xg, ag, dl.cuda(), dh.cuda(), mg, temperature=temperature)
        assert (d[~mg] == 0).all()
        assert d[4][mg[4]].isnan().all() and d[5][mg[5]].isnan().all()
        if temperature >= 1.0:                              # (at 0.01 logits 0.25 apart are 25 apart in log-probability: the action may be at the floor, which passes none)
            assert not d[0, 1].isfinite() and d[1, 1].isnan()
        adv = torch.tensor([math.inf, math.nan, 1.0, 1.0, 1.0, 1.0, -math.inf, 1.0, 3e38, 1.0]).cuda()
        r = ops.policy_loss(xg, ag, torch.full((R,), -1.0).cuda(), adv, None, mg, ent_coef=0.5, scale=1e3, temperature=temperature)
        assert (r.dlogits[~mg] == 0).all() and r.dlogits[4][mg[4]].isnan().all()


@gpu
def test_a_reference_that_rules_the_action_out():
    """ref_logp far below logp, down to -inf (an action that the reference's own mask forbids): the KL term's derivative is 1 - exp(d), to float32's last bits."""
    refs = [-math.inf, -1e30, -1e8, -1e6, -1e4, -1000.0, -300.0, -90.0, -50.0, -20.0, -5.0, -2.5, -1.7, -1.2]
    R, A = len(refs), 6
    g = torch.Generator().manual_seed(4)
    x = torch.randn((R, A), generator=g)
    act = torch.arange(R).remainder(A).to(torch.int32)
    r = ref_rows(x, act)
    old = r["logp"].float()
    ref, adv = torch.tensor(refs), torch.zeros(R)
    got = ops.policy_loss(x.cuda(), act.cuda(), old.cuda(), adv.cuda(), ref.cuda(), kl_coef=0.5)
    d = ref.double() - r["logp"]
    c = -0.5 * torch.expm1(d)
    want = ref_gradient(r, c, 0 * c, 1.0)
    # d is off by what logp is off and its own rounding, exp(d) by that and by its own 4 u; nothing of it grows with |d| beyond exp(d) |d|
    step = tol_logp(r, A) + U * d.abs().clamp(max=200)
    dc = 0.5 * (torch.exp(d) * (step + 4 * U) + 2 * U)
    check(got.dlogits, want, tol_gradient(r, c, 0 * c, dc, want, torch.float32, 1.0), "dlogits")
    assert got.stats[ops.STAT_LOSS] == math.inf and got.stats[ops.STAT_REF_KL] == math.inf
    less = ops.policy_loss(x[5:].cuda(), act[5:].cuda(), old[5:].cuda(), adv[5:].cuda(), ref[5:].cuda(), kl_coef=0.5)
    want = 0.5 * (torch.expm1(d) - d)[5:].sum()
    tol = 0.5 * (torch.expm1(d).abs() * step + 16 * U * (torch.exp(d) + 1 + d.abs()))
    assert abs(float(less.stats[ops.STAT_LOSS]) - want) <= float(tol[5:].sum())


@gpu
def test_an_advantage_of_zero_has_no_loss():
    """... also where the ratio is past float32's range."""
    x = torch.zeros((3, 5), device="cuda")
    act = torch.zeros(3, dtype=torch.int32, device="cuda")
    old = torch.tensor([-95.0, -200.0, -1.0], device="cuda")
    r = ops.policy_loss(x, act, old, torch.zeros(3, device="cuda"))
    assert r.stats[ops.STAT_LOSS] == 0 and (r.dlogits == 0).all()
    assert r.stats[ops.STAT_CLIPPED] == 3 and r.stats[ops.STAT_RATIO] == math.inf
    r = ops.policy_loss(x, act, old, torch.tensor([2.0, 0.0, 0.0], device="cuda"))
    assert abs(float(r.stats[ops.STAT_LOSS]) + 2.4) < 1e-6 and (r.dlogits == 0).all()


# ---- sums ----------------------------------------------------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("R,A", [((1 << 26) + 77, 2), (3_000_001, 90)])
def test_statistics_of_millions_of_rows(R, A):
    """Rows that are all the same: what is added up has the rounding of a workgroup's sum and of the total, not one for every row."""
    x = torch.zeros((R, A), device="cuda")
    x[:, 0] = 0.7
    act = torch.zeros(R, dtype=torch.int32, device="cuda")
    old, adv = torch.full((R,), -0.31, device="cuda"), torch.full((R,), 0.37, device="cuda")
    ref, w = torch.full((R,), -0.9, device="cuda"), torch.full((R,), 1.1, device="cuda")
    kw = dict(ent_coef=0.01, kl_coef=0.1, scale=0.3, grad=False)
    one = ops.policy_loss(x[:1], act[:1], old[:1], adv[:1], ref[:1], None, w[:1], **kw).stats.double()
    got = ops.policy_loss(x, act, old, adv, ref, None, w, **kw).stats.double()
    assert ((got - R * one).abs() <= 2 * U * R * one.abs()).all(), got / (R * one) - 1


@gpu
def test_clip_by_a_factor_under_float32_s_smallest():
    """Gradients near float32's largest value, clipped to norms of 10^-18 and less: the factor is under 2^-190, the result an ordinary number."""
    for norm in (1e-18, 1e-20, 1e-25, 1e-30, 1e-36):
        g = torch.Generator().manual_seed(1)
        a = (torch.randn(300, generator=g) * 1e37).cuda()
        b = (torch.randn(77, generator=g) * 1e37).bfloat16().cuda()
        before = [a.clone(), b.clone()]
        got = ops.clip_grad_norm([a, b], norm)
        exact = math.sqrt(sum(float((t.double() ** 2).sum()) for t in before))
        assert abs(float(got) - exact) <= 2 * U * exact
        for t, was in zip((a, b), before):
            want = was.double().cpu() * (norm / (exact + 1e-6))
            check(t, want, (half_step(t.dtype) + 4 * U) * want.abs() + 2.0 ** (-133 if t.dtype is torch.bfloat16 else -148), f"clipped to {norm}")
    for scale in (2.0 ** -126, 2.0 ** -140):
        check_clip([(torch.randn(300) * 1e30).cuda()], math.inf, scale)


# ---- autograd ------------------------------------------------------------------------------------------------------------------------------------------------

@gpu
def test_autograd_hears_of_what_is_written():
    """A layer that keeps its output for its own gradient (a soft cap) raises when the gradient was written over it, as after torch's own in-place operations."""
    x = torch.randn((9, 90), device="cuda", requires_grad=True)
    act = torch.zeros(9, dtype=torch.int32, device="cuda")
    v = torch.ones(9, device="cuda")
    for call in (lambda y: ops.action_logp_backward(y, act, v, out=y), lambda y: ops.policy_loss(y, act, -v, v, out=y).dlogits,
                 lambda y: ops.action_logp_backward(y.detach().clone(), act, v, out=y.detach())):
        y = torch.tanh(x)
        d = call(y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(d.detach())
        y = 5.0 * torch.tanh(x / 5.0)                       # (a product keeps its inputs, not its output)
        y.backward(call(y).detach())
    # a gradient that another graph keeps
    p = torch.ones(5, device="cuda", requires_grad=True)
    grad = torch.full((5,), 2.0, device="cuda")
    z = (p * grad).sum()
    before = grad._version
    ops.clip_grad_norm([grad])                              # the norm alone writes nothing
    assert grad._version == before
    ops.clip_grad_norm([grad, torch.ones(3, device="cuda")], 0.5)
    assert grad._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        q = torch.ones((2, 4), device="cuda")
        ops.action_logp_backward(q, act[:2], v[:2], out=q)
        ops.clip_grad_norm([q], 0.5)


def test_what_may_not_be_written():
    """Parameters in the place of gradients, and leaves that require a gradient, are refused before anything runs."""
    net = torch.nn.Linear(3, 2)
    with pytest.raises(ValueError, match="parameter"):
        ops.clip_grad_norm(net.parameters(), 0.5)
    with pytest.raises(ValueError, match="parameter"):
        ops.clip_grad_norm([torch.zeros(3), net.bias], 0.5)
    with pytest.raises(ValueError, match="parameter"):
        ops.clip_grad_norm(net.weight, math.inf, 0.5)
    with pytest.raises(ValueError, match="GPU"):            # their norm may be taken
        ops.clip_grad_norm(net.parameters())


@gpu
def test_a_leaf_may_not_be_written():
    x = torch.zeros((2, 6), device="cuda", requires_grad=True)
    a, v = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda")
    with pytest.raises(ValueError, match="leaf"):
        ops.action_logp_backward(x, a, v, out=x)
    with pytest.raises(ValueError, match="leaf"):
        ops.policy_loss(x, a, v, v, out=x)
    with torch.no_grad():
        ops.action_logp_backward(x, a, v, out=x)
    assert float(x.detach()[0, 0]) > 0.8


@gpu
def test_outputs_are_tensors_of_their_own():
    """What happens to one output does not count as a change of another."""
    x = torch.randn((9, 90), device="cuda")
    act = torch.zeros(9, dtype=torch.int32, device="cuda")
    v = torch.ones(9, device="cuda")
    p = torch.ones(9, device="cuda", requires_grad=True)
    logp, H = ops.action_logp(x, act)
    y = (p * H).sum()
    logp += 1.0
    y.backward()
    assert torch.equal(p.grad, H)
    r = ops.policy_loss(x, act, logp, v)
    p.grad = None
    y = (p * r.logp).sum()
    r.stats.zero_()
    y.backward()
    assert torch.equal(p.grad, r.logp)


# ---- refusals ------------------------------------------------------------------------------------------------------------------------------------------------

def test_a_temperature_whose_reciprocal_is_no_float():
    """log2(e) / T has to be a float32 as well as 1 / T."""
    lib = _lib.load()
    P = 1 << 20
    for temperature in (2.95e-39, 3.5e-39, 4.2e-39, 1e-39):
        p = _lib.PolicyRows(logits=P, ld=6, mask=None, ld_mask=0, actions=P, dtype=0, rows=4, n_actions=6, temperature=temperature, min_prob=1e-11)
        # (logp is null: refused all the same, if later)
        assert lib.rlgpu_action_logp(0, C.byref(p), None, None, P, 1 << 20, None) == -1
        assert b"temperature" in lib.rlgpu_ops_last_error(), temperature


def test_more_tensors_than_can_be_counted():
    lib = _lib.load()
    P = 1 << 20
    for n in ((1 << 24) + 1, (1 << 31) - 1, (1 << 31) - 100):
        assert lib.rlgpu_clip_grad_workspace(n) < 0
        # (no array is looked at)
        assert lib.rlgpu_clip_grad_norm(0, n, P, P, P, 1.0, 1.0, P, P, 1 << 40, None) == -1 and b"tensors" in lib.rlgpu_ops_last_error()
    assert lib.rlgpu_clip_grad_workspace(1 << 24) > 0


def test_sparse_tensors_are_refused():
    s = torch.eye(4).to_sparse()
    x, a = torch.zeros((4, 4)), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="strided"):
        ops.clip_grad_norm([torch.zeros(3), s], 1.0)
    with pytest.raises(ValueError, match="logits"):
        ops.action_logp(s, a)
    with pytest.raises(ValueError, match="mask"):
        ops.action_logp(x, a, s.bool())
    with pytest.raises(ValueError, match="actions"):
        ops.action_logp(x, a.to_sparse())


@gpu
def test_sparse_row_vectors_and_outputs_are_refused():
    x, a, v = torch.zeros((4, 4), device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="adv"):
        ops.policy_loss(x, a, v, v.to_sparse())
    with pytest.raises(ValueError, match="weights"):
        ops.policy_loss(x, a, v, v, weights=v.to_sparse())
    with pytest.raises(ValueError, match="out"):
        ops.action_logp_backward(x, a, v, out=x.to_sparse())
