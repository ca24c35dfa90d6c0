"""The operators of include/rlgpu.h for a policy network of the caller's own (rlgpu_action_logp, rlgpu_policy_loss, rlgpu_clip_grad_norm): what stands
around such a network's matrix products in an update, where PPOCore does the same inside the library's own MLPs (the reference's DiscretePolicy and
PPOLearner: PPO/DiscretePolicy.cpp:44-75, PPO/PPOLearner.cpp:148-215, 273-288).

    r = ops.policy_loss(logits, actions, old_logp, adv, ref_logp, mask, weights, clip_range=0.2, ent_coef=0.005, kl_coef=0.05, scale=1 / rows)
    logits.backward(r.dlogits)                                  # the rest of the network's backward pass
    norm = ops.clip_grad_norm([p.grad for p in network.parameters()], 0.5)

Tensors live on one GPU; the work goes to that device's current torch stream, and the outputs are new tensors of it.  Nothing synchronises and nothing is
kept between calls, so a call may be captured into a graph.  The gradients are explicit calls, not autograd nodes: outputs carry no graph, also where the
logits require a gradient (a loss that is added to another sends its dlogits through logits.backward by itself).  What is written in place (out=, clipped
gradients) counts as modified for autograd, as after torch's own in-place operations: a graph that kept it for its backward pass raises there.  Arguments
that do not fit raise ValueError before anything runs; an error of the library raises RlgpuError.
"""
import ctypes as C
from array import array
from typing import NamedTuple, Optional

import torch

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # RLGPU_F32, RLGPU_BF16, RLGPU_F16
MIN_PROB = 1e-11                                                    # the floor rlgpu_policy_act puts under a probability (PPO/DiscretePolicy.h:27-32)

# PolicyLoss.stats: sums over the rows that count (not left out)
STAT_ENTROPY, STAT_KL, STAT_CLIPPED, STAT_RATIO, STAT_REF_KL, STAT_ROWS, STAT_LOSS, STAT_WEIGHT = range(8)


class PolicyLoss(NamedTuple):
    stats: torch.Tensor                 # [8] float32, STAT_*; stats[STAT_LOSS] is the loss
    logp: torch.Tensor                  # [rows] float32: log-probability of each row's action (0 for rows left out)
    dlogits: Optional[torch.Tensor]     # [rows, n_actions], the logits' type: d(loss) / d(logits)


def _fail(rc):
    raise _lib.RlgpuError(f"rlgpu error {rc}: {_lib.load().rlgpu_ops_last_error().decode()}")


def _vector(name, t, rows, dtype, dev):
    try:
        if isinstance(t, torch.Tensor) and t.dtype is dtype and t.dim() == 1 and t.numel() == rows and t.is_contiguous() and t.device == dev:
            return t.data_ptr()
    except RuntimeError:                                    # a sparse tensor has neither strides nor memory of its own
        raise ValueError(f"{name}: a strided tensor is needed") from None
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.dim() != 1 or t.numel() != rows:
        raise ValueError(f"{name}: a {str(dtype)[6:]} tensor of {rows} rows is needed")
    if t.device != dev:
        raise ValueError(f"{name}: on {t.device}, the logits are on {dev}")
    raise ValueError(f"{name}: its rows have to be adjacent")


def _row_stride(name, t, rows, n):
    try:
        ld, one = t.stride()
    except RuntimeError:
        raise ValueError(f"{name}: a strided tensor is needed") from None
    if n > 1 and one != 1:
        raise ValueError(f"{name}: the actions of a row have to be adjacent")
    return ld if rows > 1 else n


def _rows(logits, actions, mask, temperature, min_prob):
    """The RlgpuPolicyRows of a call, checked, its rows and its device."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits: a float32, bfloat16 or float16 tensor [rows, n_actions] is needed")
    rows, n = logits.shape
    if n < 1 or n > 1 << 28 or rows > 1 << 30:
        raise ValueError(f"logits: {rows} rows of {n} actions")
    if not 0.0 < temperature < float("inf"):
        raise ValueError(f"temperature: {temperature}")
    if not 0.0 < min_prob < 1.0:
        raise ValueError(f"min_prob: {min_prob} is not between 0 and 1")
    dev = logits.device
    ld = _row_stride("logits", logits, rows, n)
    if rows > 1 and ld < n:
        raise ValueError("logits: its rows overlap (an expanded tensor)")
    at = _vector("actions", actions, rows, torch.int32, dev)
    mask_at, ld_mask = None, 0
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype not in (torch.bool, torch.uint8) or mask.shape != logits.shape:
            raise ValueError(f"mask: a bool or uint8 tensor [{rows}, {n}] is needed (one row for all: mask.expand({rows}, {n}))")
        if mask.device != dev:
            raise ValueError(f"mask: on {mask.device}, the logits are on {dev}")
        ld_mask = _row_stride("mask", mask, rows, n)
        if rows > 1 and 0 < ld_mask < n:
            raise ValueError("mask: its rows overlap")
        mask_at = mask.data_ptr()
    if dev.type != "cuda":
        raise ValueError("logits: the operators run on a GPU (there is no CPU path)")
    return _lib.PolicyRows(logits.data_ptr(), ld, mask_at, ld_mask, at, _DTYPES[logits.dtype], rows, n, temperature, min_prob), rows, dev


def _gradient(out, logits):
    if out is None:
        return torch.empty_like(logits, memory_format=torch.contiguous_format)
    if not isinstance(out, torch.Tensor) or out.shape != logits.shape or out.dtype is not logits.dtype or out.device != logits.device or out.layout is not torch.strided:
        raise ValueError("out: a strided tensor of the logits' shape, type and device is needed")
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("out: its rows overlap")
    if out.requires_grad and out.is_leaf and torch.is_grad_enabled():
        raise ValueError("out: a leaf that requires a gradient (write over it under torch.no_grad())")
    return out


_written = torch.autograd.graph.increment_version    # of a tensor or several: the kernels write behind autograd's back
_PLAIN = {torch.Tensor}
_stream = torch._C._cuda_getCurrentRawStream    # (device index) -> hipStream_t; torch.cuda.current_stream(device).cuda_stream without the object around it: 2 us less a call


def action_logp(logits, actions, mask=None, *, temperature=1.0, min_prob=MIN_PROB):
    """(logp, entropy) per row: log max(softmax(logits / temperature)[action], min_prob) and the softmax's entropy over the actions that `mask` (True =
    allowed) lets through; logits of -9.97e36 or less (float16: -65504) count as not allowed too.  actions: int32; one outside [0, n_actions) leaves its row
    out, as a row in which nothing is allowed is: logp = entropy = 0."""
    p, rows, dev = _rows(logits, actions, mask, temperature, min_prob)
    lib = _lib.load()
    n = lib.rlgpu_policy_workspace(p.dtype, rows, p.n_actions, 0)
    # one allocation: the workspace in front (none for most sizes), then the outputs
    buf = torch.empty(n // 4 + 2 * rows, dtype=torch.float32, device=dev)
    _, logp, entropy = buf.split_with_sizes((n // 4, rows, rows))
    entropy = entropy.data                              # (its own version counter: what is done to logp is no change of it)
    at = buf.data_ptr()
    rc = lib.rlgpu_action_logp(dev.index, C.byref(p), at + n, at + n + 4 * rows, at, n, _stream(dev.index))
    if rc:
        _fail(rc)
    return logp, entropy


def action_logp_backward(logits, actions, d_logp, d_entropy=None, mask=None, *, temperature=1.0, min_prob=MIN_PROB, out=None):
    """The gradient of sum(d_logp * logp + d_entropy * entropy) with respect to the logits, in the logits' type.  A logp at the floor passes none, rows left
    out and actions that are not allowed get 0.  out: where to write it; `logits` itself may be given, unless the layer behind it keeps its output (a tanh, a softmax)."""
    p, rows, dev = _rows(logits, actions, mask, temperature, min_prob)
    c = _vector("d_logp", d_logp, rows, torch.float32, dev)
    h = _vector("d_entropy", d_entropy, rows, torch.float32, dev) if d_entropy is not None else None
    d = _gradient(out, logits)
    ld = _row_stride("out", d, rows, logits.shape[1])
    lib = _lib.load()
    n = lib.rlgpu_policy_workspace(p.dtype, rows, p.n_actions, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    rc = lib.rlgpu_action_logp_backward(dev.index, C.byref(p), c, h, d.data_ptr(), ld, ws.data_ptr() if n else None, n, _stream(dev.index))
    if rc:
        _fail(rc)
    if out is not None:
        _written(out)
    return d


def policy_loss(logits, actions, old_logp, adv, ref_logp=None, mask=None, weights=None, *, clip_range=0.2, clip_high=None, ent_coef=0.0, kl_coef=0.0,
                temperature=1.0, min_prob=MIN_PROB, scale=1.0, grad=True, out=None):
    """scale * sum over rows of w (-min(r A, clip(r, 1 - clip_range, 1 + clip_high) A) + kl_coef (exp(d) - 1 - d) - ent_coef entropy) with
    r = exp(logp - old_logp), d = ref_logp - logp, and its gradient with respect to the logits, in one pass: a PolicyLoss.  clip_high defaults to
    clip_range.  A row with weight 0 is left out as in action_logp, and nothing else of it is looked at (padding may hold anything).  grad=False: no gradient.
    out: where to write the gradient; `logits` itself may be given."""
    p, rows, dev = _rows(logits, actions, mask, temperature, min_prob)
    old_at, adv_at = _vector("old_logp", old_logp, rows, torch.float32, dev), _vector("adv", adv, rows, torch.float32, dev)
    if ref_logp is None and kl_coef != 0.0:
        raise ValueError("kl_coef: needs ref_logp")
    ref_at = _vector("ref_logp", ref_logp, rows, torch.float32, dev) if ref_logp is not None else None
    weights_at = _vector("weights", weights, rows, torch.float32, dev) if weights is not None else None
    clip_high = clip_range if clip_high is None else clip_high
    if not 0.0 <= clip_range < 1.0 or not 0.0 <= clip_high < float("inf"):
        raise ValueError(f"clip range: {clip_range} below and {clip_high} above 1")
    dlogits, to, ld = None, None, 0
    if grad:
        dlogits = _gradient(out, logits)
        to, ld = dlogits.data_ptr(), _row_stride("out", dlogits, rows, logits.shape[1])
    elif out is not None:
        raise ValueError("out: without a gradient there is nothing to write")
    lib = _lib.load()
    n = lib.rlgpu_policy_workspace(p.dtype, rows, p.n_actions, 1)
    # one allocation: the workspace in front, then the statistics and the log-probabilities
    buf = torch.empty(n // 4 + 8 + rows, dtype=torch.float32, device=dev)
    _, stats, logp = buf.split_with_sizes((n // 4, 8, rows))
    stats = stats.data                                  # (its own version counter)
    ws_at = buf.data_ptr()
    l = _lib.PolicyLossC(old_at, adv_at, ref_at, weights_at, clip_range, clip_high, ent_coef, kl_coef, scale, ws_at + n + 32, ws_at + n, to, ld)
    rc = lib.rlgpu_policy_loss(dev.index, C.byref(p), C.byref(l), ws_at, n, _stream(dev.index))
    if rc:
        _fail(rc)
    if out is not None:
        _written(out)
    return PolicyLoss(stats, logp, dlogits)


def clip_grad_norm(grads, max_norm=float("inf"), grad_scale=1.0):
    """grad_scale * sqrt(sum of the squares of all the tensors' values) as a float32 tensor of one value; the tensors are multiplied in place by
    grad_scale * min(1, max_norm / (norm + 1e-6)), as PPOCore.clip_adam_step does.  max_norm = inf with grad_scale = 1 only takes the norm.  A norm that is
    not finite leaves the tensors as they are: look at it before the step.  grads: dense tensors (contiguous, or a permutation of it) of one GPU in float32,
    bfloat16 or float16, in any mix; None entries (parameters without a gradient) are passed over.  Tensors that overlap, and parameters in the place of their
    gradients, are refused when they are written."""
    grads = [grads] if isinstance(grads, torch.Tensor) else [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grads: no tensor")
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm: {max_norm}")
    if not 0.0 < grad_scale < float("inf"):
        raise ValueError(f"grad_scale: {grad_scale}")
    writes = max_norm < float("inf") or grad_scale != 1.0
    if writes and not _PLAIN.issuperset(map(type, grads)) and any(isinstance(g, torch.nn.Parameter) for g in grads):
        raise ValueError("grads: a parameter is among them (the gradients are its .grad)")
    # a pass over the list for each thing asked, with nothing but the tensor's own method in it: a network has hundreds of tensors, and a GPU that waits
    try:
        ptrs, counts = array("Q", map(torch.Tensor.data_ptr, grads)), array("q", map(torch.Tensor.numel, grads))
        dense = all(map(torch.Tensor.is_contiguous, grads)) or all(map(_dense, grads))
        devices = set(map(torch.Tensor.get_device, grads))
    except TypeError:
        raise ValueError("grads: tensors (or None) are needed") from None
    except RuntimeError:
        raise ValueError("grads: strided tensors are needed (a sparse one is among them)") from None
    try:
        kinds = array("i", [_DTYPES[g.dtype] for g in grads])
    except KeyError as e:
        raise ValueError(f"grads: {e.args[0]} is none of float32, bfloat16, float16") from None
    if not dense:
        raise ValueError("grads: a tensor is a strided view (its elements have to fill its memory)")
    if len(devices) > 1:
        raise ValueError("grads: the tensors are on several devices")
    dev = grads[0].device
    if dev.type != "cuda":
        raise ValueError("grads: the operators run on a GPU (there is no CPU path)")
    lib = _lib.load()
    n = len(grads)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = lib.rlgpu_clip_grad_workspace(n)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    rc = lib.rlgpu_clip_grad_norm(dev.index, n, ptrs.buffer_info()[0], counts.buffer_info()[0], kinds.buffer_info()[0], max_norm, grad_scale, norm.data_ptr(),
                                  ws.data_ptr(), size, _stream(dev.index))
    if rc:
        _fail(rc)
    if writes:
        _written(grads)
    return norm


def _dense(t):
    """Whether the elements fill the memory they span once: a permutation of a contiguous tensor."""
    want = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s > 1), key=lambda x: x[1]):
        if stride != want:
            return False
        want *= size
    return True
