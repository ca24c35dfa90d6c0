"""rlgymppo_cpp_amd.ops: log-probabilities and entropy of given actions, the clipped policy loss with a KL term (both with their gradients) and the gradient
norm with the clip, against plain implementations in 64 bits.

Tolerances (u = 2^-24, half a step of float32).  A row is a sum over its actions in which a lane adds a chain of `chain(A)` terms before lanes are joined
(fewer than 24 more additions, exponentials and products, each off by at most 2 u): its softmax and its log S are off by E = u (chain + 24), a term by
another 2 u |t| for the rounding of its exponent t.  What is rounded to the logits' type adds half a step of that type."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from rlgymppo_cpp_amd import _lib, ops

U = 2.0 ** -24
FLOOR = math.log(1e-11)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
gpu = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def chain(A):
    return min(A, 128) + A / 1024


# ---- the definitions in 64 bits (on the CPU) -------------------------------------------------------------------------------------------------------------

def ref_rows(logits, actions, mask=None, temperature=1.0, floor=FLOOR):
    """dict of float64: z, s, lp (per action), logp, H, on (rows that count), floored"""
    z = logits.double().cpu() / temperature
    lowest = torch.finfo(logits.dtype).min
    ok = torch.ones_like(z, dtype=torch.bool) if mask is None else mask.cpu().bool()
    z = torch.where(ok, z, -math.inf)
    a = actions.cpu().long()
    some = (ok & ~(logits.double().cpu() <= lowest)).any(1)
    on = some & (a >= 0) & (a < z.shape[1])
    m = torch.where(some, z.amax(1), 0.0)[:, None]
    e = torch.exp(z - m)
    S = e.sum(1, keepdim=True)
    s = torch.where(some[:, None], e / S, 0.0)           # (a row with nothing allowed: 0 / 0)
    lp = torch.where(some[:, None], (z - m) - torch.log(S), 0.0)
    H = -torch.where(s > 0, s * lp, s).sum(1)
    lpa = lp.gather(1, a.clamp(0, z.shape[1] - 1)[:, None])[:, 0]
    zero = torch.zeros_like(H)
    return {"z": z, "s": s, "lp": lp, "logp": torch.where(on, lpa.clamp(min=floor), zero), "H": torch.where(on, H, zero), "on": on, "floored": lpa < floor,
            "a": a, "t": torch.where(some[:, None], (z - m).clamp(min=-1e30), 0.0)}


def ref_gradient(r, c, h, temperature):
    """d(c logp + h H) / d logits"""
    lp = r["lp"].clamp(min=-1e30)
    d = -r["s"] * (c[:, None] + h[:, None] * (lp + r["H"][:, None]))
    n = torch.arange(len(c))[r["on"]]
    d[n, r["a"][r["on"]]] += c[r["on"]]
    d[~r["on"]] = 0
    return d / temperature


def ref_loss(logits, actions, old, adv, ref=None, mask=None, weights=None, clip=0.2, high=None, ent=0.0, kl=0.0, temperature=1.0, scale=1.0):
    r = ref_rows(logits, actions, mask, temperature)
    w = torch.ones(len(old), dtype=torch.float64) if weights is None else weights.double().cpu()
    on = r["on"] & (w != 0)
    x, adv = r["logp"] - old.double().cpu(), adv.double().cpu()
    high = clip if high is None else high
    rho = torch.exp(x)
    clipped = rho.clamp(1 - clip, 1 + high) * adv
    surr = rho * adv
    d = torch.zeros_like(x) if ref is None else ref.double().cpu() - r["logp"]
    value = -torch.minimum(surr, clipped) + kl * (torch.expm1(d) - d) - ent * r["H"]
    c = torch.where(clipped < surr, 0.0, -surr) - kl * torch.expm1(d)
    c = torch.where(r["floored"] | ~on, 0.0, c * w * scale)
    h = torch.where(on, -ent * w * scale, 0.0)
    r["on"] = on
    per_row = torch.stack([r["H"], torch.expm1(x) - x, ((rho < 1 - clip) | (rho > 1 + high)).double(), rho, torch.expm1(d) - d, torch.ones_like(x), value * w * scale, w])
    per_row = torch.where(on, per_row, 0.0)
    return r, rho, d, w, c, h, per_row


# ---- tolerances ------------------------------------------------------------------------------------------------------------------------------------------

def tol_logp(r, A):
    ta = r["t"].gather(1, r["a"].clamp(0, A - 1)[:, None])[:, 0]
    return U * (chain(A) + 24) + 2 * U * ta.abs().clamp(max=200) + U * r["logp"].abs()


def tol_entropy(r, A):
    # ln2 (L - W / S): both parts off by E relative, each at most log A + the entropy
    return U * (chain(A) + 24) * (2 + 2 * math.log(max(A, 2))) + 4 * U * (r["s"] * r["t"] ** 2).nan_to_num(0).sum(1)


def tol_gradient(r, c, h, dc, want, dtype, temperature):
    """dc: how far c itself may be off"""
    A = want.shape[1]
    s, lp = r["s"], r["lp"].clamp(min=-1e30)
    one = torch.zeros_like(s)
    n = torch.arange(len(c))[r["on"]]
    one[n, r["a"][r["on"]]] = 1
    size = c.abs()[:, None] * (one + s) + h.abs()[:, None] * s * (lp.abs().clamp(max=1e4) + r["H"][:, None] + 1)
    rel = U * (chain(A) + 32) + 2 * U * r["t"].abs().clamp(max=1e4)
    # the hardware's 2^t is 0 where it would be under float32's smallest normal, 2^-126: that much of s, times what s is multiplied by
    tiny = 2.0 ** -25 if dtype is torch.float16 else 2.0 ** -126
    tiny = tiny + 2.0 ** -126 * (c.abs()[:, None] + h.abs()[:, None] * (lp.abs().clamp(max=1e4) + r["H"][:, None] + 1)) / temperature
    return ((size * rel + dc[:, None] * (one + s)) / temperature) * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + tiny


def check(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, 0.0, (got - want).abs())
    bad = ~(off <= tol)
    if bad.any():
        i = int(torch.argmax(torch.where(bad, (off / tol).nan_to_num(math.inf), 0.0).reshape(-1)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, e.g. [{i}] got {got.reshape(-1)[i]!r}, want {want.reshape(-1)[i]!r}, tol {torch.as_tensor(tol).expand_as(off).reshape(-1)[i]!r}")


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------------------------

def make(rows, A, dtype, seed=0, masked=False, temperature=1.0, pad=0, spread=2.0):
    """logits with a row stride of A + pad, actions, mask (the action itself allowed in most rows), on the CPU generator"""
    g = torch.Generator().manual_seed(1000 * seed + A + rows)
    buf = (torch.randn((rows, A + pad), generator=g) * spread * temperature).to(dtype)
    logits = buf[:, pad:]
    actions = torch.randint(0, A, (rows,), generator=g).to(torch.int32)
    actions[::3] = (logits.double()[::3] + torch.randn((len(actions[::3]), A), generator=g)).argmax(1).to(torch.int32)     # likely ones too
    mask = None
    if masked:
        mask = torch.rand((rows, A), generator=g) < 0.6
        keep = torch.arange(rows) % 5 != 0
        mask[torch.arange(rows)[keep], actions.long()[keep]] = True
    return buf, logits, actions, mask, g


def loss_inputs(rows, g, logp):
    """old / ref log-probabilities around logp and advantages: ratios at least 2 % off the borders 0.8 and 1.2"""
    x = torch.tensor([-0.9, -0.3, -0.1, 0.0, 0.02, 0.12, 0.25, 0.7]).repeat(rows // 8 + 1)[:rows]
    old = (logp - x.double()).float()
    ref = (logp + 0.4 * torch.randn(rows, generator=g).double()).float()
    return old, torch.randn(rows, generator=g), ref


def to_gpu(buf, A):
    """the same row stride on the GPU"""
    b = buf.cuda()
    return b[:, b.shape[1] - A:]


SIZES = [1, 2, 3, 7, 8, 16, 33, 63, 64, 65, 90, 127, 128, 129, 255, 257, 511, 512, 513, 1000, 1025, 2047, 2049, 4099, 8191, 8193, 16385, 32771, 65537, 131072, 140001]


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("A", SIZES)
def test_against_64_bits(A, dt, masked):
    dtype = DTYPES[dt]
    rows = 67 if A < 300 else (19 if A < 5000 else 5)
    temperature = 0.7 if A % 2 else 1.0
    buf, logits, actions, mask, g = make(rows, A, dtype, masked=masked, temperature=temperature, pad=3 if A % 3 == 0 else 0)
    x, act, m = to_gpu(buf, A), actions.cuda(), None if mask is None else mask.cuda()
    r = ref_rows(logits, actions, mask, temperature)
    logp, H = ops.action_logp(x, act, m, temperature=temperature)
    check(logp, r["logp"], tol_logp(r, A), "logp")
    check(H, r["H"], tol_entropy(r, A), "entropy")
    # backward
    dl, dh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    c = torch.where(r["floored"] | ~r["on"], 0.0, dl.double())
    h = torch.where(r["on"], dh.double(), 0.0)
    zero = torch.zeros(rows, dtype=torch.float64)
    for have_h in (True, False):
        hh = h if have_h else zero
        want = ref_gradient(r, c, hh, temperature)
        got = ops.action_logp_backward(x, act, dl.cuda(), dh.cuda() if have_h else None, m, temperature=temperature)
        assert got.dtype is dtype
        check(got, want, tol_gradient(r, c, hh, zero, want, dtype, temperature), f"dlogits (entropy {have_h})")
    # the loss
    old, adv, ref = loss_inputs(rows, g, r["logp"])
    w = (torch.arange(rows) % 4 != 1).float() * 1.5
    for kl, ent, weights in ((0.0, 0.01, None), (0.1, 0.0, w), (0.1, 0.01, w)):
        r, rho, d, ww, c, h, per_row = ref_loss(logits, actions, old, adv, ref if kl else None, mask, weights, ent=ent, kl=kl, temperature=temperature, scale=0.5)
        got = ops.policy_loss(x, act, old.cuda(), adv.cuda(), ref.cuda() if kl else None, m, None if weights is None else weights.cuda(), ent_coef=ent, kl_coef=kl,
                              temperature=temperature, scale=0.5)
        tl = tol_logp(r, A)
        check(got.logp, torch.where(r["on"], r["logp"], 0.0), tl, "loss: logp")
        want = ref_gradient(r, c, h, temperature)
        # c = w scale (-rho A - kl expm1 d): rho and exp d are off by what logp is off, the roundings of old / ref - logp and of the products
        step = tl + 8 * U + U * (old.double().abs() + ref.double().abs() + r["logp"].abs())
        on = r["on"].double()
        size = rho * adv.double().abs() + (kl * (torch.exp(d) + 1) if kl else 0.0)
        dc = on * 0.5 * ww * size * step
        check(got.dlogits, want, tol_gradient(r, c, h, dc, want, dtype, temperature), f"loss: dlogits (kl {kl}, ent {ent})")
        th = tol_entropy(r, A)
        lr = torch.log(rho)
        tol = torch.stack([on * th, on * ((rho - 1).abs() * step + 16 * U * rho * lr.abs().clamp(min=0.01)), 0 * on, on * rho * step,
                           on * ((torch.exp(d) - 1).abs() * step + 16 * U * (torch.exp(d) + 1) * d.abs().clamp(min=0.01)), 0 * on, dc + on * 0.5 * ww * ent * th, on * U * ww])
        check(got.stats, per_row.sum(1), tol.sum(1) + U * per_row.abs().sum(1), f"loss: stats (kl {kl}, ent {ent})")
        alone = ops.policy_loss(x, act, old.cuda(), adv.cuda(), ref.cuda() if kl else None, m, None if weights is None else weights.cuda(), ent_coef=ent, kl_coef=kl,
                                temperature=temperature, scale=0.5, grad=False)
        assert alone.dlogits is None and torch.equal(alone.stats, got.stats) and torch.equal(alone.logp, got.logp)


# the ends of the register sets a row may be held in (in 16-byte pieces): full, full with single values behind, and one piece more
PIECES = [8, 16, 24, 32, 64, 96, 128, 192, 256, 384, 512, 768, 1024, 1536, 2048, 2560, 3071, 3073, 4096, 6144, 8192, 13312, 16384]


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("pieces", PIECES)
def test_ends_of_the_register_sets(pieces, dt, masked):
    dtype = DTYPES[dt]
    n = 4 if dt == "f32" else 8
    for A in (pieces * n + 1, pieces * n + n - 1, pieces * n + n):
        rows = 131 if pieces > 4096 else 21               # (fewer rows of so many would be split)
        _, logits, actions, mask, g = make(rows, A, dtype, seed=6, masked=masked)
        x, act, m = logits.cuda(), actions.cuda(), None if mask is None else mask.cuda()
        some = torch.tensor([0, 1, 2, 5, rows // 2, rows - 1])
        r = ref_rows(logits[some], actions[some], None if mask is None else mask[some])
        logp, H = ops.action_logp(x, act, m)
        check(logp[some], r["logp"], tol_logp(r, A), f"logp {A}")
        check(H[some], r["H"], tol_entropy(r, A), f"entropy {A}")
        dl, dh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
        zero = torch.zeros(len(some), dtype=torch.float64)
        c, h = torch.where(r["floored"] | ~r["on"], 0.0, dl[some].double()), torch.where(r["on"], dh[some].double(), 0.0)
        want = ref_gradient(r, c, h, 1.0)
        got = ops.action_logp_backward(x, act, dl.cuda(), dh.cuda(), m)
        check(got[some], want, tol_gradient(r, c, h, zero, want, dtype, 1.0), f"dlogits {A}")
        # the loss with old = logp: c = -adv r, the gradient of logp alone, and r = 1 but for what either logp is off by
        loss = ops.policy_loss(x, act, logp, -dl.cuda(), None, m, clip_range=0.5)
        want = ref_gradient(r, c, zero, 1.0)
        check(loss.logp[some], r["logp"], tol_logp(r, A), f"loss: logp {A}")
        check(loss.dlogits[some], want, tol_gradient(r, c, zero, c.abs() * (2 * tol_logp(r, A) + 8 * U), want, dtype, 1.0), f"loss: dlogits {A}")


@gpu
@pytest.mark.parametrize("rows", [1, 127, 128, 129, 300])
@pytest.mark.parametrize("A", [2500, 20011, 70001])
def test_few_rows_and_many(A, rows):
    """A row over several workgroups, or a workgroup a row: the same numbers, also where the gradient overwrites the logits."""
    _, logits, actions, mask, g = make(rows, A, torch.bfloat16, seed=4, masked=True)
    x, act, m = logits.cuda().contiguous(), actions.cuda(), mask.cuda()
    r = ref_rows(logits, actions, mask)
    logp, H = ops.action_logp(x, act, m)
    check(logp, r["logp"], tol_logp(r, A), "logp")
    check(H, r["H"], tol_entropy(r, A), "entropy")
    dl, dh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    zero = torch.zeros(rows, dtype=torch.float64)
    c, h = torch.where(r["floored"] | ~r["on"], 0.0, dl.double()), torch.where(r["on"], dh.double(), 0.0)
    want = ref_gradient(r, c, h, 1.0)
    got = ops.action_logp_backward(x, act, dl.cuda(), dh.cuda(), m)
    check(got, want, tol_gradient(r, c, h, zero, want, torch.bfloat16, 1.0), "dlogits")
    old, adv = torch.full((rows,), -5.0, device="cuda"), dl.cuda()
    loss = ops.policy_loss(x, act, old, adv, None, m, ent_coef=0.01)
    for _ in range(3):
        y = x.clone()
        assert torch.equal(ops.action_logp_backward(y, act, dl.cuda(), dh.cuda(), m, out=y), got)
        y = x.clone()
        again = ops.policy_loss(y, act, old, adv, None, m, ent_coef=0.01, out=y)
        assert torch.equal(y, loss.dlogits) and torch.equal(again.stats, loss.stats) and torch.equal(again.logp, loss.logp)


@gpu
@pytest.mark.parametrize("A,dt,rows", [(33001, "bf16", r) for r in (1, 2, 3, 5, 31, 64, 65, 127, 128, 129)] + [(17001, "f32", 6), (90, "f32", 1), (90, "f32", 32), (90, "f32", 33),
                                       (700, "f16", 3), (2000, "bf16", 4), (9000, "f32", 1)])
def test_statistics_of_few_rows(A, dt, rows):
    """The sums over the rows wherever they are formed: one workgroup, a row over several, more of both; rows that do not count are among them."""
    _, logits, actions, mask, g = make(rows, A, DTYPES[dt], seed=rows, masked=True)
    w = torch.rand(rows, generator=g) + 0.5
    w[2::5] = 0.0
    actions[3::7] = -1
    mask[4::9] = False
    first = ref_rows(logits, actions, mask)
    old, adv, ref = loss_inputs(rows, g, first["logp"])
    old[2::5] = math.nan                                    # (weight 0: nothing else is looked at)
    clean = torch.where(w == 0, torch.zeros_like(old), old)
    r, rho, d, ww, c, h, per_row = ref_loss(logits, actions, clean, adv, ref, mask, w, ent=0.01, kl=0.1, scale=0.5)
    x, args = logits.cuda().contiguous(), (actions.cuda(), old.cuda(), adv.cuda(), ref.cuda(), mask.cuda(), w.cuda())
    got = ops.policy_loss(x, *args, ent_coef=0.01, kl_coef=0.1, scale=0.5)
    tl, th, on = tol_logp(r, A), tol_entropy(r, A), r["on"].double()
    # as for the loss above: what logp is off by, the roundings of old / ref - logp and of the products
    step = tl + 8 * U + U * (clean.double().abs() + ref.double().abs() + r["logp"].abs())
    dc = on * 0.5 * ww * (rho * adv.double().abs() + 0.1 * (torch.exp(d) + 1)) * step
    lr = torch.log(rho)
    tol = torch.stack([on * th, on * ((rho - 1).abs() * step + 16 * U * rho * lr.abs().clamp(min=0.01)), 0 * on, on * rho * step,
                       on * ((torch.exp(d) - 1).abs() * step + 16 * U * (torch.exp(d) + 1) * d.abs().clamp(min=0.01)), 0 * on, dc + on * 0.5 * ww * 0.01 * th, on * U * ww])
    check(got.stats, per_row.sum(1), tol.sum(1) + U * per_row.abs().sum(1), "stats")
    for _ in range(2):
        alone = ops.policy_loss(x, *args, ent_coef=0.01, kl_coef=0.1, scale=0.5, grad=False)
        assert torch.equal(alone.stats, got.stats) and torch.equal(alone.logp, got.logp)


@gpu
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("A", [6, 90, 700, 9001])
def test_rows_with_nothing_to_learn(A, dt):
    """Rows left out, masks in every form, infinities and NaN in masked places, actions at the floor."""
    dtype = DTYPES[dt]
    low = torch.finfo(dtype).min
    R = 14
    g = torch.Generator().manual_seed(A)
    x = torch.randn((R, A), generator=g).to(dtype)
    mask = torch.ones((R, A), dtype=torch.bool)
    act = torch.full((R,), 1, dtype=torch.int32)
    w = torch.ones(R)
    adv, old, ref = torch.ones(R), torch.full((R,), -1.0), torch.full((R,), -1.5)
    mask[0] = False                                         # 0: nothing allowed
    mask[1] = False; x[1] = math.nan                        # 1: nothing allowed, NaN behind the mask
    x[2] = -math.inf                                        # 2: all -inf
    x[3] = low                                              # 3: all at the type's lowest value
    act[4] = -1                                             # 4, 5: no such action
    act[5] = A
    w[6] = 0.0; x[6] = math.nan; adv[6] = old[6] = ref[6] = math.nan     # 6: padding
    w[7] = 0.0; act[7] = -2147483648                        # 7: padding with garbage
    left_out = list(range(8))
    x[8, 2:] = -math.inf                                    # 8: two actions by logits
    mask[9, 2:] = False; x[9, 2:] = math.inf; x[9, 3] = math.nan         # 9: two by the mask, +inf and NaN behind it
    mask[10, 1] = False                                     # 10: the action itself is not allowed: at the floor
    x[11] = 0.0; x[11, 1] = -200.0                          # 11: below the floor by its logit
    x[12, 2:] = low                                         # 12: masked by the lowest value
    x[13] = 0.0; x[13, 1] = 60.0                            # 13: the action has all of the probability
    ref[10] = ref[11] = FLOOR + 0.5                         # (a reference that is at the floor there as well)
    c = lambda t: t.cuda()
    r = ref_rows(torch.where(mask, x, torch.zeros_like(x)), act, mask)
    r["on"][6] = r["on"][7] = False
    logp, H = ops.action_logp(c(x), c(act), c(mask))
    for i in left_out[:6] + [7]:
        assert logp[i] == 0 and H[i] == 0
    assert math.isnan(logp[6]) and math.isnan(H[6])         # (this call knows no weights)
    keep = [8, 9, 10, 11, 12, 13]
    check(logp[keep], r["logp"][keep], tol_logp(r, A)[keep], "logp")
    check(H[keep], r["H"][keep], tol_entropy(r, A)[keep], "entropy")
    assert logp[10] == np.float32(FLOOR) and logp[11] == np.float32(FLOOR)
    dl, dh = torch.ones(R), torch.full((R,), 0.5)
    dl[:6] = dh[:6] = math.nan                              # (left out: whatever they are)
    d = ops.action_logp_backward(c(x), c(act), c(dl), c(dh), c(mask))
    assert (d[left_out[:6] + [7]] == 0).all() and not d[keep].isnan().any()
    assert (d[9, 2:] == 0).all() and (d[10, 1] == 0)
    for kl in (0.0, 0.2):
        got = ops.policy_loss(c(x), c(act), c(old), c(adv), c(ref) if kl else None, c(mask), c(w), ent_coef=0.3, kl_coef=kl)
        assert (got.dlogits[left_out] == 0).all() and (got.logp[left_out] == 0).all() and got.stats[ops.STAT_ROWS] == 6 and got.stats[ops.STAT_WEIGHT] == 6
        xs, os_, as_, rs = (torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (torch.where(mask, x, torch.zeros_like(x)), old, adv, ref))
        xs = torch.where(mask & (x == -math.inf), x, xs)
        rr, rho, dd, ww, cc, hh, per_row = ref_loss(xs, act, os_, as_, rs if kl else None, mask, w, ent=0.3, kl=kl)
        want = ref_gradient(rr, cc, hh, 1.0)
        step = tol_logp(rr, A) + 8 * U + U * 60
        dc = ww * (rho + kl * (torch.exp(dd) + 1)) * step
        check(got.dlogits, want, tol_gradient(rr, cc, hh, torch.where(rr["floored"], 0.0, dc), want, dtype, 1.0), "dlogits")
        check(got.stats[ops.STAT_LOSS], per_row[6].sum(), float((dc + 0.3 * tol_entropy(rr, A)).sum() + U * per_row[6].abs().sum()), "loss")


@gpu
@pytest.mark.parametrize("A,R,dt", [(5, 300001, "f32"), (90, 150001, "f32"), (250, 70001, "bf16"), (400, 50003, "bf16"), (700, 40001, "f16"), (1500, 30001, "bf16"), (5000, 9001, "bf16"),
                                    (20000, 3001, "f32"), (40000, 4003, "bf16"), (70001, 4201, "f16"), (140001, 1301, "bf16"), (140001, 301, "f32")])
def test_many_rows(A, R, dt):
    """Workgroups that take row after row, padding and left-out rows among them, and calls that go past the caches: the same bits as in blocks of few rows, some
    rows against 64 bits."""
    dtype = DTYPES[dt]
    g = torch.Generator(device="cuda").manual_seed(A)
    x = (torch.randn((R, A), generator=g, device="cuda", dtype=torch.float32) * 2).to(dtype)
    act = torch.randint(-1, A + 1, (R,), generator=g, device="cuda").to(torch.int32)        # a few out of range
    act[::5] = x[::5].argmax(1).to(torch.int32)
    at = torch.arange(R, device="cuda")
    w = (at % 512 < torch.randint(1, 513, (R // 512 + 1,), generator=g, device="cuda")[at // 512]).float()
    old, adv = torch.randn(R, generator=g, device="cuda") * 0.1 - 2, torch.randn(R, generator=g, device="cuda")
    old[w == 0] = math.nan
    dh = torch.randn(R, generator=g, device="cuda")

    def calls(k, out=None):
        lp, h = ops.action_logp(x[k], act[k])
        d = ops.action_logp_backward(x[k], act[k], adv[k], dh[k])
        r = ops.policy_loss(x[k], act[k], old[k], adv[k], None, None, w[k], ent_coef=0.01, scale=0.5)
        return lp, h, d, r.logp, r.dlogits, r.stats
    whole = calls(slice(0, R))
    stats = torch.zeros(8, dtype=torch.float64, device="cuda")
    step = max(129, min(3001, R // 3))
    edges = list(range(0, R - 129, step)) + [R]                       # (blocks of more than 128 rows: fewer would be split)
    for a, b in zip(edges, edges[1:]):
        part = calls(slice(a, b))
        for name, u, v in zip(("logp", "entropy", "backward", "loss logp", "loss dlogits"), whole, part):
            assert torch.equal(u[a:b], v), f"{name}: rows {a} to {b}"
        stats += part[5].double()
    # each block's statistics are rounded once to float32, the workgroups' parts once a row
    assert torch.allclose(whole[5].double(), stats, rtol=1e-5, atol=1e-5 * R)
    assert whole[5][ops.STAT_ROWS] == ((act >= 0) & (act < A) & (w != 0)).sum()
    some = torch.cat([torch.arange(4), torch.randint(0, R, (24,), generator=torch.Generator().manual_seed(1)), torch.arange(R - 4, R)])
    r = ref_rows(x[some], act[some])
    check(whole[0][some], r["logp"], tol_logp(r, A), "logp")
    c, h = torch.where(r["floored"] | ~r["on"], 0.0, adv[some].double().cpu()), torch.where(r["on"], dh[some].double().cpu(), 0.0)
    want = ref_gradient(r, c, h, 1.0)
    check(whole[2][some], want, tol_gradient(r, c, h, 0 * c, want, dtype, 1.0), "dlogits")


@gpu
@pytest.mark.parametrize("how", ["mask", "lowest", "-inf", "-1e30", "-8e36"])
@pytest.mark.parametrize("temperature", [0.01, 1.0, 2.0, 100.0])
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("A", [7, 90, 255, 1000, 9000, 140001])
def test_all_but_a_few_masked(A, dt, temperature, how):
    """Masks, by the mask or by the logits, that leave one to three actions anywhere in the row (most lanes have nothing), and coefficients far from 1."""
    dtype = DTYPES[dt]
    if dtype is torch.float16 and how in ("-1e30", "-8e36"):
        how = "-inf"
    R = 6
    _, logits, _, _, g = make(R, A, dtype, seed=8, temperature=temperature)
    keep = torch.zeros((R, A), dtype=torch.bool)
    act = torch.randint(0, A, (R,), generator=g)
    for i in range(R):
        keep[i, act[i]] = True
        keep[i, torch.randint(0, A, (i % 3,), generator=g)] = True
    act = act.to(torch.int32)
    x, mask = logits.clone(), None
    if how == "mask":
        x[~keep] = math.nan
        mask = keep
    else:
        x[~keep] = {"lowest": torch.finfo(dtype).min, "-inf": -math.inf, "-1e30": -1e30, "-8e36": -8e36}[how]
    r = ref_rows(torch.where(keep, logits, torch.zeros_like(logits)), act, keep, temperature)
    m = None if mask is None else mask.cuda()
    logp, H = ops.action_logp(x.cuda(), act.cuda(), m, temperature=temperature)
    check(logp, r["logp"], tol_logp(r, A), "logp")
    check(H, r["H"], tol_entropy(r, A), "entropy")
    zero = torch.zeros(R, dtype=torch.float64)
    for size in (1e-3, 1.0, 1e3):
        c, h = torch.full((R,), 0.5 * size).double(), torch.full((R,), size).double()
        if dtype is torch.float16:
            c, h = c * min(1.0, temperature), h * min(1.0, temperature)        # (float16 holds 65504)
        c, h = c.float().double(), h.float().double()
        want = ref_gradient(r, torch.where(r["floored"], 0.0, c), h, temperature)
        got = ops.action_logp_backward(x.cuda(), act.cuda(), c.float().cuda(), h.float().cuda(), m, temperature=temperature)
        check(got, want, tol_gradient(r, c, h, zero, want, dtype, temperature), f"dlogits {size}")
        assert (got[~keep.cuda()] == 0).all()


@gpu
@pytest.mark.parametrize("base", [1e4, 1e6, 1e9, 1e30, -1e7, -1e9, -1e30])
@pytest.mark.parametrize("temperature", [1e-4, 1.0])
@pytest.mark.parametrize("A,rows", [(5, 9), (90, 9), (700, 9), (20000, 3), (20000, 200)])
def test_far_logits(A, rows, temperature, base):
    """Logits whose exponents are far from 0, spread over a few of float32's steps there."""
    g = torch.Generator().manual_seed(A)
    step = max(abs(base) * 2.0 ** -23, temperature)
    x = (base + torch.randint(-4, 5, (rows, A), generator=g).double() * step).float()
    act = x.argmax(1).to(torch.int32)
    act[1] = x[1].argmin()
    r = ref_rows(x, act, None, temperature)
    logp, H = ops.action_logp(x.cuda(), act.cuda(), temperature=temperature)
    check(logp, r["logp"], tol_logp(r, A), "logp")
    check(H, r["H"], tol_entropy(r, A), "entropy")
    c, h, zero = (torch.full((rows,), v).double() for v in (0.5, 0.25, 0.0))
    want = ref_gradient(r, torch.where(r["floored"], 0.0, c), h, temperature)
    got = ops.action_logp_backward(x.cuda(), act.cuda(), c.float().cuda(), h.float().cuda(), temperature=temperature)
    check(got, want, tol_gradient(r, c, h, zero, want, torch.float32, temperature), "dlogits")


@gpu
@pytest.mark.parametrize("A", [5, 90, 3000])
def test_nan_and_infinite_logits_show(A):
    x = torch.zeros((4, A))
    x[0, 2] = math.nan; x[1] = math.nan; x[2, 3] = math.inf
    act = torch.ones(4, dtype=torch.int32)
    logp, H = ops.action_logp(x.cuda(), act.cuda())
    d = ops.action_logp_backward(x.cuda(), act.cuda(), torch.ones(4).cuda())
    for i in range(3):
        assert math.isnan(logp[i]) and math.isnan(H[i]) and d[i].isnan().all()
    assert abs(float(logp[3]) + math.log(A)) < 1e-5 and not d[3].isnan().any()


@gpu
@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("A", [3, 90, 1003, 20001])
def test_layouts(A, dt):
    """Row strides, unaligned rows, one mask row for all, in place, the other half of a buffer; what lies beside a row stays."""
    dtype = DTYPES[dt]
    R = 9
    buf, logits, actions, _, g = make(R, A, dtype, seed=3)
    x, act = logits.cuda().contiguous(), actions.cuda()
    one = (torch.rand(A, generator=g) < 0.7)
    one[0] = True
    full = one.expand(R, A).contiguous().cuda()
    dl, dh = torch.randn(R, generator=g).cuda(), torch.randn(R, generator=g).cuda()
    want_lp, want_h = ops.action_logp(x, act, full)
    want = ops.action_logp_backward(x, act, dl, dh, full)
    lp, h = ops.action_logp(x, act, one.cuda().expand(R, A))
    assert torch.equal(lp, want_lp) and torch.equal(h, want_h)
    for pad, off in ((1, 0), (5, 1), (8, 3)):
        wide = torch.full((R, A + pad), 7.0, dtype=dtype, device="cuda")
        wide[:, off:off + A] = x
        wm = torch.zeros((R, A + pad), dtype=torch.uint8, device="cuda")
        wm[:, off:off + A] = full * 3                       # any value but 0 allows
        lp, h = ops.action_logp(wide[:, off:off + A], act, wm[:, off:off + A])
        assert torch.equal(lp, want_lp) and torch.equal(h, want_h)
        got = ops.action_logp_backward(wide[:, off:off + A], act, dl, dh, wm[:, off:off + A], out=wide[:, off:off + A])
        assert torch.equal(got, want) and got.data_ptr() == wide[:, off:].data_ptr()
        rest = torch.ones(A + pad, dtype=torch.bool, device="cuda"); rest[off:off + A] = False
        assert (wide[:, rest] == 7.0).all()
    halves = torch.full((R, 2 * A), 5.0, dtype=dtype, device="cuda")
    halves[:, :A] = x
    ops.action_logp_backward(halves[:, :A], act, dl, dh, full, out=halves[:, A:])
    assert torch.equal(halves[:, :A], x) and torch.equal(halves[:, A:], want)
    # a vector of the batch that starts anywhere
    long = torch.randn(R + 3, generator=g).cuda(); long[2:2 + R] = dl
    assert torch.equal(ops.action_logp_backward(x, act, long[2:2 + R], dh, full), want)


@gpu
def test_a_reference_that_is_only_watched():
    """kl_coef 0: the reference's log-probabilities are a statistic, whatever they are."""
    x, a = torch.zeros((3, 5), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    old, adv = torch.full((3,), -math.log(5.0), device="cuda"), torch.ones(3, device="cuda")
    plain = ops.policy_loss(x, a, old, adv)
    r = ops.policy_loss(x, a, old, adv, torch.tensor([-1.0, -math.inf, math.nan], device="cuda"))
    assert torch.equal(r.dlogits, plain.dlogits) and r.stats[ops.STAT_LOSS] == plain.stats[ops.STAT_LOSS]


@gpu
def test_no_rows_and_one_row():
    e = torch.empty(0, device="cuda")
    none = ops.action_logp(torch.empty((0, 5), device="cuda"), e.to(torch.int32))
    assert none[0].shape == (0,) and none[1].shape == (0,)
    assert ops.action_logp_backward(torch.empty((0, 5), device="cuda"), e.to(torch.int32), e).shape == (0, 5)
    r = ops.policy_loss(torch.empty((0, 5), device="cuda"), e.to(torch.int32), e, e)
    assert (r.stats == 0).all() and r.dlogits.shape == (0, 5)
    one = torch.tensor([[0.3]], device="cuda")
    lp, h = ops.action_logp(one, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert lp[0] == 0 and h[0] == 0


@gpu
def test_offsets_past_32_bits():
    """40 000 rows of 131 072 actions in 16 bits: 5.2 G elements, 10.5 GB, in place."""
    R, A = 40000, 131072
    x = torch.empty((R, A), dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, 16383, 16384, 16385, 32767, 32768, 32769, R - 2, R - 1]
    x.fill_(0.0)
    g = torch.Generator().manual_seed(5)
    some = (torch.randn((len(rows), A), generator=g) * 2).bfloat16()
    x[rows] = some.cuda()
    act = torch.full((R,), A - 1, dtype=torch.int32)
    r = ref_rows(some, act[rows])
    dl = torch.zeros(R); dl[rows] = 1.0
    logp, H = ops.action_logp(x, act.cuda())
    check(logp[rows], r["logp"], tol_logp(r, A), "logp")
    assert (logp.cpu()[5:16000] - (-math.log(A))).abs().max() < 1e-4
    out = ops.action_logp_backward(x, act.cuda(), dl.cuda(), out=x)
    one, zero = torch.ones(len(rows), dtype=torch.float64), torch.zeros(len(rows), dtype=torch.float64)
    want = ref_gradient(r, one, zero, 1.0)
    check(out[rows], want, tol_gradient(r, one, zero, zero, want, torch.bfloat16, 1.0), "dlogits")
    assert (out[2:16000:97] == 0).all()


@gpu
@pytest.mark.parametrize("A", [4, 11])
def test_gradient_against_differences(A):
    """Central differences of the 64-bit loss in every logit (step 1e-5: 1e-10 of curvature and 1e-11 of rounding beside the tolerance of the kernel)."""
    R = 8
    _, logits, actions, mask, g = make(R, A, torch.float32, seed=9, masked=True)
    logp = ref_rows(logits, actions, mask, 0.8)["logp"]
    old, adv, ref = loss_inputs(R, g, logp)
    w = torch.rand(R, generator=g) + 0.5
    kw = dict(ent=0.2, kl=0.3, temperature=0.8, scale=0.7)

    def total(z):
        return float(ref_loss_64(z, actions, old, adv, ref, mask, w, **kw))
    base = logits.double()
    num = torch.zeros_like(base)
    for i in range(R):
        for j in range(A):
            up, down = base.clone(), base.clone()
            up[i, j] += 1e-5; down[i, j] -= 1e-5
            num[i, j] = (total(up) - total(down)) / 2e-5
    got = ops.policy_loss(logits.cuda(), actions.cuda(), old.cuda(), adv.cuda(), ref.cuda(), mask.cuda(), w.cuda(), ent_coef=0.2, kl_coef=0.3, temperature=0.8, scale=0.7)
    r, rho, d, ww, c, h, _ = ref_loss(logits, actions, old, adv, ref, mask, w, **kw)
    step = tol_logp(r, A) + 8 * U + U * 60
    dc = 0.7 * ww * (rho * adv.double().abs() + 0.3 * (torch.exp(d) + 1)) * step
    check(got.dlogits, num, tol_gradient(r, c, h, dc, num, torch.float32, 0.8) + 1e-8, "dlogits")


def ref_loss_64(z, *a, **kw):
    return ref_loss(z, *a, **kw)[6][6].sum()


def test_the_reference_gradient_is_the_derivative():
    """The oracle against itself: its gradient formula and autograd through its loss, in 64 bits."""
    R, A = 16, 9
    _, logits, actions, mask, g = make(R, A, torch.float32, seed=1, masked=True)
    old, adv, ref = loss_inputs(R, g, ref_rows(logits, actions, mask, 1.3)["logp"])
    z = logits.double().requires_grad_()
    kw = dict(ent=0.1, kl=0.2, temperature=1.3, scale=0.25)
    p = torch.where(mask, z / 1.3, -math.inf)
    lp = torch.log_softmax(p, 1)
    on = ref_rows(logits, actions, mask, 1.3)
    H = -(lp.exp() * torch.where(mask, lp, 0.0)).sum(1)
    lpa = lp.gather(1, actions.long()[:, None])[:, 0].clamp(min=FLOOR)
    rho = torch.exp(lpa - old.double())
    d = ref.double() - lpa
    loss = -torch.minimum(rho * adv.double(), rho.clamp(0.8, 1.2) * adv.double()) + 0.2 * (torch.exp(d) - 1 - d) - 0.1 * H
    keep = on["on"]
    (loss[keep].sum() * 0.25).backward()
    r, _, _, _, c, h, per_row = ref_loss(logits, actions, old, adv, ref, mask, None, **kw)
    want = ref_gradient(r, c, h, 1.3)
    assert torch.allclose(z.grad.nan_to_num(0)[keep], want[keep], rtol=0, atol=1e-12)
    assert abs(float((per_row[6].sum() - loss[keep].sum() * 0.25).detach())) < 1e-12


@gpu
def test_it_is_the_learner_s_loss():
    """policy_loss and action_logp against PPOCore on one minibatch of the same MLP (fp32): its gradients come back through the logits."""
    from rlgymppo_cpp_amd.ppo import PPOCore
    D, A, R = 21, 90, 512
    core = PPOCore(D, A, (64, 64), (32,), ent_coef=0.01, clip_range=0.2, temperature=1.0, max_rows=R, seed=7)
    flat = torch.from_numpy(core.get_params(0)).cuda()
    params, at = [], 0
    for ws, bs in core.layer_shapes(0):
        for shape in (ws, bs):
            n = int(np.prod(shape)); params.append(flat[at:at + n].view(shape).clone().requires_grad_()); at += n
    g = torch.Generator().manual_seed(2)
    obs = torch.randn((R, D), generator=g).cuda()
    acts, logp0 = torch.empty(R, dtype=torch.int32, device="cuda"), torch.empty(R, device="cuda")
    core.act(obs, acts, logp0)
    x = obs
    for i in range(0, len(params), 2):
        x = torch.nn.functional.linear(x, params[i], params[i + 1])
        x = x.relu() if i + 2 < len(params) else x
    logp, _ = ops.action_logp(x.detach(), acts)
    # both forward passes are fp32 sums of up to 64 products of O(1): a few 1e-6
    assert (logp - logp0).abs().max() < 2e-5
    x_shift = torch.tensor([-0.9, -0.3, -0.1, 0.0, 0.02, 0.12, 0.25, 0.7], device="cuda").repeat(R // 8)
    old, adv = logp0 - x_shift, torch.randn(R, generator=g).cuda()
    vals = core.value(obs)
    metrics = torch.zeros(8, device="cuda")
    core.zero_grads()
    core.minibatch(obs, acts, old, adv, vals, None, R, 1.0, metrics)
    r = ops.policy_loss(x.detach(), acts, old, adv, ent_coef=0.01, scale=1.0 / R)
    x.backward(r.dlogits)
    mine = torch.cat([p.grad.reshape(-1) for p in params])
    his = torch.from_numpy(core.get_grads(0)).cuda()
    assert (mine - his).norm() < 1e-4 * his.norm()
    assert torch.allclose(r.stats[:4], metrics[:4], rtol=1e-4, atol=1e-3)
    assert r.stats[ops.STAT_CLIPPED] == metrics[2]
    norm = ops.clip_grad_norm([p.grad for p in params], 0.5)
    assert abs(float(norm) - float(his.double().norm())) < 1e-4 * float(norm)
    core.close()


@gpu
def test_one_update_of_a_network_of_one_s_own():
    """As they are used together: a network in bfloat16 on the framework's envs, its old and reference log-probabilities, loss, gradients, clip, and the same in 64 bits."""
    from rlgymppo_cpp_amd.env import BatchedEnv
    env = BatchedEnv(64, 1)
    obs = env.reset(True).clone()
    R, A = env.n_agents, env.n_actions
    g = torch.Generator(device="cuda").manual_seed(11)
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Linear(env.obs_size, 128), torch.nn.LayerNorm(128), torch.nn.ReLU(), torch.nn.Linear(128, A)).cuda().bfloat16()
    with torch.no_grad():
        old_logits = net(obs.bfloat16())
    mask = torch.rand((R, A), generator=g, device="cuda") < 0.9
    mask[:, 0] = True
    noise = torch.empty((R, A), device="cuda").exponential_(generator=g)
    acts = torch.where(mask, old_logits.float() - noise.log(), -math.inf).argmax(1).to(torch.int32)
    nobs, rew, done = torch.empty_like(obs), torch.empty(R, device="cuda"), torch.empty(R, dtype=torch.int32, device="cuda")
    env.step(acts, nobs, rew, done); env.sync()
    adv = torch.randn(R, generator=g, device="cuda") + rew
    old_logp, _ = ops.action_logp(old_logits, acts, mask)
    old_logp += 0.05 * torch.randn(R, generator=g, device="cuda")
    ref_logp = (old_logp - 0.1).contiguous()
    logits = net(obs.bfloat16())
    r = ops.policy_loss(logits, acts, old_logp, adv, ref_logp, mask, ent_coef=0.01, kl_coef=0.1, scale=1.0 / R)
    logits.backward(r.dlogits)
    _, rho, d, w, c, h, per_row = ref_loss(logits.detach(), acts, old_logp, adv, ref_logp, mask, ent=0.01, kl=0.1, scale=1.0 / R)
    want = ref_gradient(ref_rows(logits.detach(), acts, mask), c, h, 1.0)
    assert (r.dlogits.double().cpu() - want).norm() <= (half_step(torch.bfloat16) + 1e-4) * want.norm()
    grads = [p.grad for p in net.parameters()]
    before = [p.clone() for p in grads]
    norm = ops.clip_grad_norm(grads, 0.01)
    exact = math.sqrt(sum(float((b.double() ** 2).sum()) for b in before))
    assert abs(float(norm) - exact) <= 2 * U * exact and exact > 0.01
    for a, b in zip(grads, before):
        check(a, b.double().cpu() * (0.01 / (exact + 1e-6)), (half_step(torch.bfloat16) + 4 * U) * b.double().cpu().abs() * (0.01 / exact) + 1e-40, "clipped")


# ---- clip ------------------------------------------------------------------------------------------------------------------------------------------------

def clip_reference(grads, max_norm, scale):
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads)) * scale
    return norm, scale * min(1.0, max_norm / (norm + 1e-6))


def check_clip(grads, max_norm, scale=1.0):
    before = [t.clone() for t in grads]
    norm, f = clip_reference(before, max_norm, scale)
    got = ops.clip_grad_norm(grads, max_norm, scale)
    assert got.dtype is torch.float32 and got.shape == ()
    # summed in 64 bits: one rounding to float32, one of the scale, far less from the sum
    assert abs(float(got) - norm) <= 2 * U * norm
    for a, b in zip(grads, before):
        tiny = 2.0 ** -25 if a.dtype is torch.float16 else 2.0 ** -133
        check(a, b.double().cpu() * f, (half_step(a.dtype) + 4 * U) * b.double().cpu().abs() * f + tiny, "clipped")


@gpu
@pytest.mark.parametrize("dt", list(DTYPES) + ["mixed"])
@pytest.mark.parametrize("counts", [[1], [7], [0, 5, 0], [16384], [16383, 1, 16385], [100003, 0, 3, 64, 65537], [3] * 700, [0, 0]])
@pytest.mark.parametrize("scale", [1.0, 0.125])
def test_clip_sizes(counts, dt, scale):
    g = torch.Generator().manual_seed(len(counts))
    kinds = list(DTYPES.values()) if dt == "mixed" else [DTYPES[dt]]
    grads = [torch.randn(n, generator=g).to(kinds[i % len(kinds)]).cuda() for i, n in enumerate(counts)]
    total = math.sqrt(sum(counts))
    check_clip(list(t.clone() for t in grads), 0.1 * total, scale)       # clipped
    check_clip([t.clone() for t in grads], 10 * total + 1, scale)    # below
    check_clip([t.clone() for t in grads], math.inf, scale)
    check_clip([t.clone() for t in grads], 0.0, scale)


@gpu
def test_clip_many_tensors_and_a_large_one():
    """More tensors than a few launches hold, in the order they come; a large one among them; one that is a generator's."""
    g = torch.Generator(device="cuda").manual_seed(3)
    grads = [torch.randn(1 + i % 7, generator=g, device="cuda").to(list(DTYPES.values())[i % 3]) for i in range(5003)]
    grads.insert(2000, torch.randn(30_000_001, generator=g, device="cuda"))
    grads.insert(4500, torch.randn(9_000_001, generator=g, device="cuda").bfloat16())
    before = [t.clone() for t in grads]
    exact = math.sqrt(sum(float((t.double() ** 2).sum()) for t in before))
    n = ops.clip_grad_norm((t for t in grads), 1.0)
    assert abs(float(n) - exact) <= 2 * U * exact
    f = 1.0 / (exact + 1e-6)
    for i in [0, 1, 2, 159, 160, 161, 1999, 2000, 2001, 4500, 5003, 5004]:
        a, b = grads[i], before[i].double().cpu() * f
        check(a, b, (half_step(a.dtype) + 4 * U) * b.abs() + 2.0 ** -25, "clipped")
    assert all(torch.equal(a, (b.float() * f).to(a.dtype)) or (a.float() - b.float() * f).abs().max() <= 2 * half_step(a.dtype) * (b.float() * f).abs().max() + 2.0 ** -25 for a, b in zip(grads, before))


@gpu
def test_clip_views_and_what_lies_beside():
    """Views that start at any element of a buffer, permuted and multi-dimensional tensors, None; nothing beside them is written."""
    for dtype in DTYPES.values():
        buf = torch.arange(40000, dtype=torch.float32).sin().to(dtype).cuda()
        keep = buf.clone()
        views = [buf[3:1000], buf[1001:1002], buf[1003:18500], buf[20000:20000], buf[20001:39999]]
        check_clip(views, 1.0)
        rest = torch.ones(40000, dtype=torch.bool, device="cuda")
        for a, b in ((3, 1000), (1001, 1002), (1003, 18500), (20001, 39999)):
            rest[a:b] = False
        assert torch.equal(buf[rest], keep[rest]) and not torch.equal(buf, keep)
    w = torch.randn((5, 7, 3), device="cuda").permute(2, 0, 1)
    conv = torch.randn((2, 8, 3, 3), device="cuda").to(memory_format=torch.channels_last)
    check_clip([w, conv, torch.tensor(3.0, device="cuda")], 0.5)
    n = ops.clip_grad_norm([None, torch.full((4,), 2.0, device="cuda"), None])
    assert float(n) == 4.0
    same = torch.ones(8, device="cuda")
    assert float(ops.clip_grad_norm([same, same])) == 4.0            # the norm alone may see a tensor twice


@gpu
def test_clip_norm_that_is_not_finite():
    for bad in (math.nan, math.inf, -math.inf):
        a, b = torch.ones(1000, device="cuda"), torch.ones(70000, dtype=torch.bfloat16, device="cuda")
        b[69999] = bad
        keep = [a.clone(), b.clone()]
        n = ops.clip_grad_norm([a, b], 0.5, 0.25)
        assert not math.isfinite(float(n)) and torch.equal(a, keep[0]) and torch.equal(b.nan_to_num(7.0), keep[1].nan_to_num(7.0))


@gpu
def test_clip_norm_past_float32():
    """Finite gradients whose norm is inf as a float32: what the caller is told is not finite, so they stay; scaled into range they are clipped."""
    for dtype in (torch.float32, torch.bfloat16):
        a = torch.full((5,), 3e38, device="cuda").to(dtype)
        keep = a.clone()
        assert float(ops.clip_grad_norm([a], 0.5)) == math.inf and torch.equal(a, keep)
        check_clip([a], 0.5, 2.0 ** -10)


@gpu
def test_clip_range_of_the_sum():
    """Squares that pass float32's range on both sides: the sum has 64 bits."""
    big = torch.full((1000,), 1e30, device="cuda")
    check_clip([big], 1.0)
    small = torch.full((1000,), 1e-30, device="cuda")
    n = ops.clip_grad_norm([small])
    assert abs(float(n) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6


@gpu
def test_clip_past_32_bits():
    n = (1 << 32) + 12345
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[0], t[(1 << 31) + 5], t[n - 1] = 3.0, 4.0, 12.0
    assert float(ops.clip_grad_norm([t], 6.5)) == 13.0
    # 13 + 1e-6 in the denominator: half of each to 1e-7, which bfloat16 rounds to the half itself
    assert (float(t[0]), float(t[(1 << 31) + 5]), float(t[n - 1])) == (1.5, 2.0, 6.0)


# ---- streams, graphs, repetition ---------------------------------------------------------------------------------------------------------------------------

def everything(x, act, mask, dl, dh, old, adv, ref, w, grads):
    lp, h = ops.action_logp(x, act, mask)
    d = ops.action_logp_backward(x, act, dl, dh, mask)
    r = ops.policy_loss(x, act, old, adv, ref, mask, w, ent_coef=0.01, kl_coef=0.1, scale=1.0 / len(act))
    out = [t.clone() for t in grads]
    return [lp, h, d, *r, *out, ops.clip_grad_norm(out, 0.3)]


def everything_inputs(R, A, dtype, seed):
    _, logits, actions, mask, g = make(R, A, dtype, seed=seed, masked=True)
    old, adv, ref = loss_inputs(R, g, ref_rows(logits, actions, mask)["logp"])
    v = [t.cuda() for t in (logits.contiguous(), actions, mask, torch.randn(R, generator=g), torch.randn(R, generator=g), old, adv, ref, (torch.rand(R, generator=g) < 0.8).float())]
    return v + [[torch.randn(n, generator=g).to(dtype).cuda() for n in (5, 70001, 0, 333)]]


@gpu
@pytest.mark.parametrize("R,A,dt", [(300, 90, "f32"), (7, 40003, "bf16"), (1, 131072, "f16"), (600, 1200, "bf16")])
def test_graphs_streams_and_repetition(R, A, dt):
    """The same bits on every call, on another stream, and on every replay of two graphs that live side by side, with eager work between the replays."""
    sets = [everything_inputs(R, A, DTYPES[dt], seed) for seed in (1, 2)]
    want = [everything(*s) for s in sets]
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(everything(*s), w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    # a size that no call has seen before the capture
    fresh = torch.randn((5, 700 + R), device="cuda")
    first = torch.zeros(5, dtype=torch.int32, device="cuda")
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        lp = ops.action_logp(fresh, first)[0]
    gr.replay()
    assert torch.equal(lp, ops.action_logp(fresh, first)[0])
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(everything(*s))
        graphs.append(gr)
    for k in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        for gr in graphs:
            gr.replay()
        eager = everything(*sets[k % 2])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[k % 2]))
    # both at once, each on a stream of its own
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream()); side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs[0].replay()
    with torch.cuda.stream(other):
        graphs[1].replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


# ---- refusals (no GPU needed) ------------------------------------------------------------------------------------------------------------------------------

def _row_args(R=4, A=6, dtype=torch.float32):
    return torch.zeros((R, A), dtype=dtype), torch.zeros(R, dtype=torch.int32), torch.zeros(R), torch.zeros(R)


def test_refusals_of_rows():
    x, a, old, adv = _row_args()
    cases = [
        (dict(logits=x.double()), "logits"), (dict(logits=x[0]), "logits"), (dict(logits=x.t()), "adjacent"), (dict(logits=torch.zeros((4, 0))), "actions"),
        (dict(logits=x[:1].expand(4, 6)), "overlap"), (dict(actions=a.long()), "actions"), (dict(actions=a[:3]), "actions"), (dict(actions=a[:, None]), "actions"),
        (dict(actions=torch.zeros(8, dtype=torch.int32)[::2]), "adjacent"), (dict(mask=torch.ones((4, 5), dtype=torch.bool)), "mask"), (dict(mask=torch.ones((4, 6))), "mask"),
        (dict(mask=torch.ones((6, 4), dtype=torch.bool).t()), "adjacent"), (dict(temperature=0.0), "temperature"), (dict(temperature=math.nan), "temperature"),
        (dict(temperature=math.inf), "temperature"), (dict(min_prob=0.0), "min_prob"), (dict(min_prob=1.0), "min_prob"), (dict(), "GPU"),
    ]
    for change, text in cases:
        kw = dict(logits=x, actions=a, mask=None, temperature=1.0, min_prob=1e-11)
        kw.update(change)
        with pytest.raises(ValueError, match=text):
            ops.action_logp(kw["logits"], kw["actions"], kw["mask"], temperature=kw["temperature"], min_prob=kw["min_prob"])
        with pytest.raises(ValueError, match=text):
            ops.policy_loss(kw["logits"], kw["actions"], old, adv, None, kw["mask"], temperature=kw["temperature"], min_prob=kw["min_prob"])


@gpu
def test_refusals_of_the_loss_and_the_gradient():
    x, a, old, adv = (t.cuda() for t in _row_args())
    for kw, text in ((dict(clip_range=1.0), "clip"), (dict(clip_range=-0.1), "clip"), (dict(clip_high=-1.0), "clip"), (dict(clip_range=math.nan), "clip"), (dict(kl_coef=0.1), "ref_logp"),
                     (dict(weights=adv.half()), "weights"), (dict(ref_logp=adv[:2]), "ref_logp"), (dict(out=x.half()), "out"), (dict(out=x[:2]), "out"), (dict(grad=False, out=x), "out"),
                     (dict(ref_logp=adv.cpu()), "cpu")):
        with pytest.raises(ValueError, match=text):
            ops.policy_loss(x, a, old, adv, **kw)
    for kw in (dict(ent_coef=math.nan), dict(scale=math.inf), dict(min_prob=1e-60)):
        with pytest.raises(_lib.RlgpuError):
            ops.policy_loss(x, a, old, adv, **kw)
    big = torch.zeros(64, device="cuda")
    with pytest.raises(_lib.RlgpuError, match="overlap"):
        ops.action_logp_backward(big[:24].view(4, 6), a, old, out=big[1:25].view(4, 6))
    with pytest.raises(_lib.RlgpuError, match="overlap"):
        ops.action_logp_backward(big[:28].view(4, 7)[:, :6], a, old, out=big[3:31].view(4, 7)[:, :6])
    with pytest.raises(_lib.RlgpuError, match="overlap"):
        ops.clip_grad_norm([big[:10], big[9:20]], 1.0)
    with pytest.raises(_lib.RlgpuError, match="overlap"):
        ops.clip_grad_norm([big, big], 1.0)


def test_refusals_of_the_clip():
    t = torch.zeros(4)
    for grads, kw, text in (([], {}, "no tensor"), ([None], {}, "no tensor"), ([t.double()], {}, "float64"), ([3.0], {}, "tensors"), ([torch.zeros(8)[::2]], {}, "strided"),
                            ([torch.zeros(1).expand(4)], {}, "strided"), ([t], dict(max_norm=-1.0), "max_norm"), ([t], dict(max_norm=math.nan), "max_norm"),
                            ([t], dict(grad_scale=0.0), "grad_scale"), ([t], dict(grad_scale=math.inf), "grad_scale"), ([t], {}, "GPU")):
        with pytest.raises(ValueError, match=text):
            ops.clip_grad_norm(grads, **kw)


def test_refusals_of_the_library():
    """The C entry points check what the Python ones do, before any GPU call: the pointers here are never looked at."""
    lib = _lib.load()
    P = 1 << 20

    def rows(**kw):
        p = _lib.PolicyRows(logits=P, ld=6, mask=None, ld_mask=0, actions=P, dtype=0, rows=4, n_actions=6, temperature=1.0, min_prob=1e-11)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def loss(**kw):
        l = _lib.PolicyLossC(old_logp=P, adv=P, ref_logp=None, weights=None, clip_low=0.2, clip_high=0.2, ent_coef=0.0, kl_coef=0.0, scale=1.0, logp=None, stats=P,
                             dlogits=None, ld_dlogits=0)
        for k, v in kw.items():
            setattr(l, k, v)
        return l
    N = 1 << 20
    bad_rows = [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=(1 << 30) + 1), dict(n_actions=0), dict(n_actions=(1 << 28) + 1), dict(temperature=0.0), dict(temperature=math.nan),
                dict(temperature=1e-45), dict(min_prob=0.0), dict(min_prob=1.0), dict(logits=None), dict(actions=None), dict(ld=5), dict(ld=1 << 31), dict(mask=P, ld_mask=5), dict(mask=P, ld_mask=1 << 31),
                dict(logits=P + 2), dict(actions=P + 1), dict(dtype=1, logits=P + 1)]
    for kw in bad_rows:
        p = rows(**kw)
        assert lib.rlgpu_action_logp(0, C.byref(p), P, None, P, N, None) == -1 and lib.rlgpu_ops_last_error()
        assert lib.rlgpu_action_logp_backward(0, C.byref(p), P, None, 2 * P, 6, P, N, None) == -1
        assert lib.rlgpu_policy_loss(0, C.byref(p), C.byref(loss()), P, N, None) == -1
    p = rows()
    assert lib.rlgpu_policy_workspace(7, 4, 6, 0) < 0 and lib.rlgpu_policy_workspace(0, -1, 6, 0) < 0 and lib.rlgpu_policy_workspace(0, 4, 0, 1) < 0
    assert lib.rlgpu_policy_workspace(0, 4, (1 << 28) + 1, 1) < 0 and lib.rlgpu_policy_workspace(0, 4, 6, 0) == 0
    long = rows(n_actions=40000, ld=40000)                  # four rows of many actions: in parts
    for ws, miss in ((None, 0), (P + 8, 0), (P, 1)):
        assert lib.rlgpu_policy_loss(0, C.byref(p), C.byref(loss()), ws, lib.rlgpu_policy_workspace(0, 4, 6, 1) - miss, None) == -1
        assert lib.rlgpu_action_logp(0, C.byref(long), P, None, ws, lib.rlgpu_policy_workspace(0, 4, 40000, 0) - miss, None) == -1
        assert lib.rlgpu_action_logp_backward(0, C.byref(long), P, None, 2 * P, 40000, ws, lib.rlgpu_policy_workspace(0, 4, 40000, 0) - miss, None) == -1
    assert lib.rlgpu_action_logp(0, None, P, None, P, N, None) == -1
    assert lib.rlgpu_action_logp(0, C.byref(p), None, None, P, N, None) == -1
    for d, ld in ((None, 6), (2 * P, 5), (2 * P + 1, 6), (P + 4, 6), (P - 8, 6)):
        assert lib.rlgpu_action_logp_backward(0, C.byref(p), P, None, d, ld, P, N, None) == -1
    assert lib.rlgpu_action_logp_backward(0, C.byref(p), None, None, 2 * P, 6, P, N, None) == -1
    for kw in (dict(stats=None), dict(old_logp=None), dict(adv=None), dict(adv=P + 2), dict(clip_low=1.0), dict(clip_low=-0.1), dict(clip_high=math.inf), dict(ent_coef=math.nan),
               dict(kl_coef=math.inf), dict(scale=math.nan), dict(kl_coef=0.1), dict(dlogits=P + 4, ld_dlogits=6)):
        assert lib.rlgpu_policy_loss(0, C.byref(p), C.byref(loss(**kw)), P, N, None) == -1, kw
    assert lib.rlgpu_policy_loss(0, C.byref(p), None, P, N, None) == -1

    def clip(ptrs=(P,), counts=(4,), kinds=(0,), max_norm=1.0, scale=1.0, norm=P, ws=P, n=N):
        k = len(ptrs)
        return lib.rlgpu_clip_grad_norm(0, k, (C.c_void_p * k)(*ptrs), (C.c_int64 * k)(*counts), (C.c_int32 * k)(*kinds), max_norm, scale, norm, ws, n, None)
    assert clip(kinds=(5,)) == -1 and clip(counts=(-1,)) == -1 and clip(counts=(1 << 41,)) == -1 and clip(ptrs=(None,)) == -1 and clip(ptrs=(P + 2,)) == -1
    assert clip(max_norm=-1.0) == -1 and clip(max_norm=math.nan) == -1 and clip(scale=0.0) == -1 and clip(scale=math.inf) == -1 and clip(norm=None) == -1
    assert clip(ws=None) == -1 and clip(ws=P + 8) == -1 and clip(n=8) == -1
    assert clip(ptrs=(P, P + 8), counts=(4, 4), kinds=(0, 0)) == -1 and b"overlap" in lib.rlgpu_ops_last_error()
    assert lib.rlgpu_clip_grad_norm(0, -1, None, None, None, 1.0, 1.0, P, P, N, None) == -1
    assert lib.rlgpu_clip_grad_norm(0, 1, None, None, None, 1.0, 1.0, P, P, N, None) == -1
    assert lib.rlgpu_clip_grad_workspace(-1) < 0 and lib.rlgpu_clip_grad_workspace(0) > 0
