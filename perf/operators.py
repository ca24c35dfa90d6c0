"""The operators that a program with a policy network of its own puts around the network's matrix products, as cases that can be timed and checked:

  logp       log-probability and entropy of given actions under (masked) logits       rlgymppo_cpp_amd.ops.action_logp
  logp_grad  its gradient with respect to the logits                                  rlgymppo_cpp_amd.ops.action_logp_backward
  loss       clipped policy loss with a KL term and an entropy term, and d(logits)    rlgymppo_cpp_amd.ops.policy_loss
  clip       global norm over many gradient tensors, and clipping in place            rlgymppo_cpp_amd.ops.clip_grad_norm

listed() names the cases, draw() makes more of the same ranges, prepare() makes a case's inputs from a seed, run() is one pass: in elementary torch
operations, or (own = True) through the framework.  exact() is the same from the definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

MIN_PROB = 1e-11                                    # the framework's floor of a probability (clamp(softmax, 1e-11, 1))
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LARGEST = 4096 * 131072                             # logits of the largest case


def _policy(name, op, rows, actions, dtype, mask=False, ref=False, padded=False, temperature=1.0, ent=0.005):
    return {"name": name, "op": op, "rows": rows, "actions": actions, "dtype": dtype, "mask": mask, "ref": ref, "padded": padded,
            "temperature": temperature, "ent": ent}


def _clip(name, tensors, values, dtype, above):
    return {"name": name, "op": "clip", "tensors": tensors, "values": values, "dtype": dtype, "above": above}


def listed():
    return [
        # one decision of a policy with a large vocabulary of actions: its log-probability while it is served
        _policy("logp_one_row", "logp", 1, 131072, "bf16"),
        # one gym step's actions of 4 096 1v1 arenas, with the actions that are not available masked
        _policy("logp_agents", "logp", 8192, 90, "f32", mask=True),
        # the old or reference log-probabilities of a batch of token rows, odd sizes
        _policy("logp_tokens", "logp", 6001, 50021, "f16", temperature=0.7),
        # a user's own loss over the learner's minibatch, through the log-probability and the entropy
        _policy("logp_grad_minibatch", "logp_grad", 65536, 90, "f32"),
        # the same over token rows
        _policy("logp_grad_tokens", "logp_grad", 2048, 131072, "bf16"),
        # the learner's minibatch: 65 536 rows of the 90-action table
        _policy("loss_minibatch", "loss", 65536, 90, "f32"),
        # a combined action table with unavailable actions, a reference policy and padded trajectories
        _policy("loss_masked", "loss", 16385, 1847, "f32", mask=True, ref=True, padded=True),
        # token rows of padded sequences against a reference policy: the largest
        _policy("loss_tokens", "loss", 4096, 131072, "bf16", ref=True, padded=True),
        # the few rows of one short sequence
        _policy("loss_few_rows", "loss", 23, 128003, "f16", ref=True),
        # the learner's own two 256 x 3 networks
        _clip("clip_networks", 16, 332635, "f32", True),
        # several hundred tensors of both types, as a sequence policy has them
        _clip("clip_mixed", 701, 60000013, "mixed", True),
        # the gradients of a large network in 16 bits
        _clip("clip_large", 290, 536870912, "bf16", True),
    ]


def draw(rng):
    op = rng.choice(("logp", "logp_grad", "loss", "loss", "clip"))
    if op == "clip":
        values = int(math.exp(rng.uniform(math.log(1000), math.log(400e6))))
        tensors = min(values, int(math.exp(rng.uniform(0, math.log(701)))))
        return {"op": op, "tensors": tensors, "values": values, "dtype": rng.choice(("f32", "bf16", "f16", "mixed")), "above": rng.random() < 0.8}
    actions = int(math.exp(rng.uniform(math.log(2), math.log(131072))))
    most = min(65536, LARGEST // actions // 2)
    rows = int(math.exp(rng.uniform(0, math.log(most))))
    return {"op": op, "rows": rows, "actions": actions, "dtype": rng.choice(tuple(TYPES)), "mask": rng.random() < 0.3, "ref": rng.random() < 0.5,
            "padded": rng.random() < 0.3, "temperature": rng.choice((1.0, 1.0, 0.7, 1.5)), "ent": rng.choice((0.0, 0.005, 0.01))}


def _sizes(case):
    """How many values each tensor has: a few large matrices, many small vectors, some empty; the same for every seed."""
    rng = random.Random(case["tensors"] * 1000003 + case["values"])
    parts = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(case["tensors"])]
    left, sizes = case["values"], []
    for p in parts:
        sizes.append(int(case["values"] * p / sum(parts)))
    left -= sum(sizes)
    sizes[0] += left
    return sizes


def _prepare_clip(case, g, dev):
    kinds = ("f32", "bf16") if case["dtype"] == "mixed" else (case["dtype"],)
    sizes = _sizes(case)
    # views into one buffer a type, as gradient buckets have them: a tensor starts wherever the one before it ends
    flat = {k: torch.randn(max(1, sum(sizes[i::len(kinds)])), generator=g, device=dev, dtype=TYPES[k]).mul_(0.02) for i, k in enumerate(kinds)}
    cut = {k: flat[k].split(sizes[i::len(kinds)]) if sum(sizes[i::len(kinds)]) else [flat[k][:0]] for i, k in enumerate(kinds)}
    grads = [cut[kinds[i % len(kinds)]][i // len(kinds)] for i in range(len(sizes))]
    norm = 0.02 * math.sqrt(case["values"])          # nearly the norm of these gradients
    # above: the sum is first scaled from the rows that were there to the rows that count, and clipped, in every pass anew; else the norm stays below
    return {"op": "clip", "grads": grads, "flat": flat, "max_norm": norm * (0.1 if case["above"] else 10.0), "scale": 1.25 if case["above"] else 1.0}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "clip":
        return _prepare_clip(case, g, dev)
    R, A, t = case["rows"], case["actions"], TYPES[case["dtype"]]
    f = dict(generator=g, device=dev)
    temperature = case["temperature"]
    logits = torch.randn((R, A), dtype=torch.float32, **f).mul_(2.0 * temperature).to(t)
    z = logits.float() / temperature
    mask = None
    if case["mask"]:
        mask = torch.rand((R, A), **f) < 0.75
        if R > 8:
            mask[R // 3] = False                     # a row in which nothing is allowed
        z.masked_fill_(~mask, -math.inf)
    noise = torch.empty((R, A), dtype=torch.float32, device=dev).exponential_(generator=g)
    actions = (z - noise.log_()).argmax(1)           # sampled from the softmax of what is allowed
    del noise
    logp = torch.log_softmax(z, 1).gather(1, actions[:, None])[:, 0].nan_to_num_(0.0, 0.0, 0.0)
    del z
    s = {"op": case["op"], "logits": logits, "actions": actions.to(torch.int32), "mask": mask, "temperature": temperature}
    loss_scale = 4096.0 if case["dtype"] == "f16" else 1.0   # five bits of exponent need one, as in any training in this type
    if case["op"] == "logp_grad":
        s["d_logp"] = torch.randn(R, **f).mul_(loss_scale / R)
        s["d_entropy"] = torch.full((R,), -case["ent"] * loss_scale / R, device=dev)
    if case["op"] == "loss":
        # most rows moved little since they were sampled, one in ten far enough to be clipped
        far = torch.rand(R, **f) < 0.1
        step = torch.where(far, (torch.rand(R, **f) * 0.6 + 0.4) * torch.where(torch.rand(R, **f) < 0.5, -1.0, 1.0), torch.randn(R, **f).mul_(0.04))
        s["old_logp"] = logp - step
        s["adv"] = torch.randn(R, **f)
        s["ref_logp"] = (logp + torch.randn(R, **f).mul_(0.3)).clamp_(max=0.0) if case["ref"] else None
        s["weights"] = None
        if case["padded"]:                           # sequences of up to 512 rows, each padded behind its own length
            at = torch.arange(R, device=dev)
            length = torch.randint(1, 513, ((R + 511) // 512,), **f)
            s["weights"] = (at % 512 < length[at // 512]).float()
        s["ent"], s["kl"] = case["ent"], 0.05 if case["ref"] else 0.0
        s["scale"] = loss_scale / R                  # the mean over the rows
    return s


def _plain_rows(s):
    """(log-probabilities of all actions, of the given ones, entropy, which rows count, whether the floor holds)"""
    z = s["logits"].float() / s["temperature"]
    if s["mask"] is not None:
        z = torch.where(s["mask"], z, -math.inf)
    m = z.amax(1, keepdim=True)
    live = m[:, 0] > -math.inf
    z = z - torch.where(live[:, None], m, 0.0)
    S = z.exp().sum(1, keepdim=True)
    lp = torch.where(live[:, None], z - S.log(), 0.0)
    H = -torch.where(lp > -math.inf, lp.exp() * lp, 0.0).sum(1)
    H = torch.where(live, H, 0.0)
    lpa = lp.gather(1, s["actions"].long()[:, None])[:, 0]
    logp = lpa.clamp(min=math.log(MIN_PROB))
    return lp, torch.where(live, logp, 0.0), H, live, lpa < math.log(MIN_PROB)


def _plain_grad(s, lp, H, live, c, h):
    p = lp.exp()
    dz = torch.where(lp > -math.inf, -p * (c[:, None] + h[:, None] * (lp + H[:, None])), 0.0)
    dz.scatter_add_(1, s["actions"].long()[:, None], c[:, None])
    return (torch.where(live[:, None], dz, 0.0) / s["temperature"]).to(s["logits"].dtype)


def _plain_loss(s):
    lp, logp, H, live, floored = _plain_rows(s)
    w = (live if s["weights"] is None else torch.where(live, s["weights"], 0.0)).double()
    on = w != 0
    x = logp.double() - s["old_logp"].double()       # what belongs to a row is next to the border of the clip: in 64 bits
    ratio, adv = x.exp(), s["adv"].double()
    clipped = ratio.clamp(0.8, 1.2) * adv
    through = ratio * adv <= clipped
    value = -torch.minimum(ratio * adv, clipped) - s["ent"] * H.double()
    c = -torch.where(through, ratio * adv, 0.0)
    ref_kl = torch.zeros_like(ratio)
    if s["ref_logp"] is not None:
        d = s["ref_logp"].double() - logp.double()
        ref_kl = torch.expm1(d) - d
        value, c = value + s["kl"] * ref_kl, c - s["kl"] * torch.expm1(d)
    c = torch.where(floored | ~on, 0.0, c * w * s["scale"])
    rows = torch.stack([H.double(), torch.expm1(x) - x, ((ratio - 1.0).abs() > 0.2).double(), ratio, ref_kl, torch.ones_like(ratio), value * w * s["scale"], w])
    stats = torch.where(on, rows, 0.0).sum(1).float()
    h = torch.where(on, -s["scale"] * s["ent"] * w, 0.0)
    return {"stats": stats, "logp": torch.where(on, logp, 0.0), "dlogits": _plain_grad(s, lp, H, live, c.float(), h.float())}


def _plain_clip(s):
    sums = torch.stack([g.float().square().sum() for g in s["grads"]])
    norm = sums.sum().sqrt() * s["scale"]
    coef = torch.where(norm.isfinite(), s["scale"] * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0), 1.0)
    [g.copy_(g.float() * coef) for g in s["grads"]]
    return {"norm": norm, **s["flat"]}


def run(s):
    if own:
        from rlgymppo_cpp_amd import ops
        if s["op"] == "clip":
            return {"norm": ops.clip_grad_norm(s["grads"], s["max_norm"], s["scale"]), **s["flat"]}
        if s["op"] == "logp":
            logp, entropy = ops.action_logp(s["logits"], s["actions"], s["mask"], temperature=s["temperature"])
            return {"logp": logp, "entropy": entropy}
        if s["op"] == "logp_grad":
            return {"dlogits": ops.action_logp_backward(s["logits"], s["actions"], s["d_logp"], s["d_entropy"], s["mask"], temperature=s["temperature"])}
        r = ops.policy_loss(s["logits"], s["actions"], s["old_logp"], s["adv"], s["ref_logp"], s["mask"], s["weights"], clip_range=0.2, ent_coef=s["ent"],
                            kl_coef=s["kl"], temperature=s["temperature"], scale=s["scale"])
        return {"stats": r.stats, "logp": r.logp, "dlogits": r.dlogits}
    if s["op"] == "clip":
        return _plain_clip(s)
    if s["op"] == "loss":
        return _plain_loss(s)
    lp, logp, H, live, floored = _plain_rows(s)
    if s["op"] == "logp":
        return {"logp": logp, "entropy": H}
    return {"dlogits": _plain_grad(s, lp, H, live, torch.where(floored, 0.0, s["d_logp"]), s["d_entropy"])}


def work(case):
    if case["op"] == "clip":
        kinds = ("f32", "bf16") if case["dtype"] == "mixed" else (case["dtype"],)
        sizes = _sizes(case)
        total = sum(sum(sizes[i::len(kinds)]) * TYPES[k].itemsize for i, k in enumerate(kinds))
        return {"bytes": total * (2 if case["above"] else 1) + 4, "flops": case["values"] * (3 if case["above"] else 2)}
    n, size = case["rows"] * case["actions"], TYPES[case["dtype"]].itemsize
    read = n * (size + (1 if case["mask"] else 0)) + 4 * case["rows"]
    if case["op"] == "logp":
        return {"bytes": read + 8 * case["rows"], "flops": 7 * n}
    per_row = 8 if case["op"] == "logp_grad" else 12 + 4 * case["ref"] + 4 * case["padded"]
    return {"bytes": read + n * size + per_row * case["rows"], "flops": 13 * n}


# ---- the same in 64 bits, by the definitions -------------------------------------------------------------------------------------------------------------

def _exact_clip(s):
    total = sum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in s["grads"] if g.numel())
    norm = math.sqrt(total) * s["scale"]
    factor = s["scale"] * min(1.0, s["max_norm"] / (norm + 1e-6))
    return {"norm": np.float64(norm), **{k: v.double() * factor for k, v in s["flat"].items()}}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        return _exact_clip(s)
    R, A = s["logits"].shape
    out = {"logp": torch.zeros(R, dtype=torch.float64, device="cuda"), "entropy": torch.zeros(R, dtype=torch.float64, device="cuda")}
    dlogits = None if case["op"] == "logp" else torch.zeros((R, A), dtype=torch.float64, device="cuda")
    stats = torch.zeros(8, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // A)
    for r in range(0, R, step):
        k = slice(r, min(R, r + step))
        z = s["logits"][k].double() / s["temperature"]
        z = z if s["mask"] is None else z.masked_fill(~s["mask"][k], -math.inf)
        some = z.amax(1) > -math.inf
        lse = torch.where(some, torch.logsumexp(z, 1), 0.0)
        p = torch.exp(z - lse[:, None])              # rows with nothing allowed: all zero
        entropy = torch.special.entr(p).sum(1)
        a = s["actions"][k].long()[:, None]
        raw = z.gather(1, a)[:, 0] - lse
        logp = raw.clamp(min=math.log(MIN_PROB))
        on = some
        if case["op"] == "logp_grad":
            to_logp, to_entropy = s["d_logp"][k].double(), s["d_entropy"][k].double()
        if case["op"] == "loss":
            w = torch.ones_like(logp) if s["weights"] is None else s["weights"][k].double()
            on = some & (w != 0)
            x, adv = logp - s["old_logp"][k].double(), s["adv"][k].double()
            rho = torch.exp(x)
            bound = torch.where(adv > 0, 1.2, 0.8)   # the side on which the minimum is the clipped term
            cut = torch.where(adv > 0, rho > bound, rho < bound)
            surrogate = torch.where(cut, bound, rho) * adv
            d = (s["ref_logp"][k].double() - logp) if s["ref_logp"] is not None else torch.zeros_like(logp)
            kl = torch.expm1(d) - d
            value = w * s["scale"] * (s["kl"] * kl - surrogate - s["ent"] * entropy)
            to_logp = w * s["scale"] * (torch.where(cut, 0.0, -rho * adv) - s["kl"] * torch.expm1(d))
            to_entropy = -w * s["scale"] * s["ent"]
            per_row = (entropy, torch.expm1(x) - x, ((rho < 0.8) | (rho > 1.2)).double(), rho, kl, torch.ones_like(rho), value, w)
            stats += torch.stack([torch.where(on, v, 0.0).sum() for v in per_row])
        out["logp"][k] = torch.where(on, logp, 0.0)
        out["entropy"][k] = torch.where(on, entropy, 0.0)
        if dlogits is not None:
            to_logp = torch.where((raw < math.log(MIN_PROB)) | ~on, 0.0, to_logp)
            to_entropy = torch.where(on, to_entropy, 0.0)
            plogp = -torch.special.entr(p)           # p log p, 0 where p is 0
            g = -to_logp[:, None] * p - to_entropy[:, None] * (plogp + p * entropy[:, None])
            g[torch.arange(len(a), device=g.device), a[:, 0]] += to_logp
            dlogits[k] = g / s["temperature"]
    if case["op"] == "logp":
        return out
    return {"dlogits": dlogits} if case["op"] == "logp_grad" else {"stats": stats, "logp": out["logp"], "dlogits": dlogits}
