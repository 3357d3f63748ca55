"""From a policy's action scores to the actions of `env.step()`, and back: operators on rows of logits, as hand-written HIP kernels
(include/mgx_policy.h).

  * `sample_actions` draws one action per env on the device, with random numbers the caller gives: what a rollout calls per env-step
    (`BaseEnv.step_policy` is the two together);
  * `action_log_probs` says how likely given actions are -- a demonstration's, a rollout's --, how spread the policy is, and what it
    would rather do; its backward pass gives the gradient to the logits.  Behaviour cloning's loss is
    `-(out.log_prob + c * out.entropy).mean()`, a policy gradient's `-(advantage * out.log_prob + c * out.entropy).mean()`;
    `saved_trajectories.replay_demos(policy=...)` scores a policy on demonstrations.

A row holds the logits of one choice among n: 18 for one env-step, 18 ** c for a policy that answers with c env-steps at once, a
vocabulary for one that answers in tokens.  Logits are float32, float16 or bfloat16 tensors [..., n] on the GPU, of any strides (a last
dimension that is not dense is copied first); `mask` is a bool tensor that broadcasts to them, False = ruled out; the distribution is
softmax(logits / temperature) over the actions that are open (not ruled out, logit above -inf).  Results are float32 whatever the
logits' type.  Rows with nothing open give log probability -inf, entropy 0 and action -1 with gradient 0; rows with NaN or +inf among
the open logits give NaN and action -1.  Calls run on torch's current stream of the logits' device; they can be captured into a HIP graph.
"""
import ctypes as C
import math
from typing import NamedTuple, Optional

import torch

from . import _native as nat

__all__ = ['ActionLogProbs', 'SampledActions', 'action_log_probs', 'sample_actions', 'MAX_TOP']

MAX_TOP = 64                     # MGX_POLICY_MAX_TOP
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # mgx_real
_LOG_PROBS, _SAMPLE = 0, 1       # mgx_policy_op


class ActionLogProbs(NamedTuple):
    log_prob: torch.Tensor                    # f32 [...]: log p of the given action
    entropy: torch.Tensor                     # f32 [...]
    top_log_probs: Optional[torch.Tensor]     # f32 [..., top], best first (None if top == 0); no gradient
    top_actions: Optional[torch.Tensor]       # i32 [..., top]; -1 where a row has no more open actions


class SampledActions(NamedTuple):
    action: torch.Tensor       # i32 [...]; -1 where nothing is open
    log_prob: torch.Tensor     # f32 [...]
    entropy: torch.Tensor      # f32 [...]


def _check(rc):
    if rc < 0:
        raise nat.MgxError(f'mgx error {rc}: {nat.lib().mgx_policy_last_error().decode()}')


def _rows(logits, mask, temperature):
    """The arguments (dtype, logits, rows, n, row stride, mask, mask's row stride, temperature) of the C calls and the tensors that
    have to live until then."""
    if not torch.is_tensor(logits):
        raise TypeError('logits: a tensor')
    dtype = _DTYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f'logits: float32, float16 or bfloat16, got {logits.dtype}')
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f'logits: [..., n] with n >= 1, got {tuple(logits.shape)}')
    n = logits.shape[-1]
    x = logits if logits.dim() == 2 else logits.reshape(-1, n)
    if n > 1 and x.stride(1) != 1:
        x = x.contiguous()
    rows = x.shape[0]
    mask_ptr, mask_stride = None, 0
    if mask is not None:
        if not torch.is_tensor(mask) or mask.dtype != torch.bool:
            raise TypeError('mask: a bool tensor')
        if mask.device != logits.device:
            raise ValueError(f'mask is on {mask.device}, logits on {logits.device}')
        try:
            whole = mask.expand(logits.shape)
        except RuntimeError:
            raise ValueError(f'mask {tuple(mask.shape)} does not broadcast to logits {tuple(logits.shape)}') from None
        mask = whole if whole.dim() == 2 else whole.reshape(-1, n)
        if n > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
        mask_ptr, mask_stride = mask.data_ptr(), mask.stride(0)
    temperature = float(temperature)
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f'temperature: positive and finite, got {temperature}')
    return (dtype, x.data_ptr(), rows, n, x.stride(0), mask_ptr, mask_stride, temperature), (x, mask)


def _stream(device):
    if device.type != 'cuda':
        raise nat.MgxError('magical_amd runs on an MI355X (torch device "cuda:N"); there is no CPU fallback')
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(op, args, top, device):
    size = nat.lib().mgx_policy_workspace_bytes(op, args[0], args[2], args[3], top)
    return (None, 0, None) if size <= 0 else _scratch(size, device)


def _scratch(size, device):
    t = torch.empty(size, dtype=torch.uint8, device=device)
    return t.data_ptr(), size, t


def _forward(logits, actions, mask, temperature, top, want_stats):
    args, kept = _rows(logits, mask, temperature)
    lead, dev = logits.shape[:-1], logits.device
    if not torch.is_tensor(actions) or actions.dtype not in (torch.int32, torch.int64):
        raise TypeError('actions: an int32 or int64 tensor')
    if actions.device != dev:
        raise ValueError(f'actions are on {actions.device}, logits on {dev}')
    if actions.shape != lead:
        raise ValueError(f'actions: one for each row of logits, {tuple(lead)}, got {tuple(actions.shape)}')
    top = int(top)
    if not 0 <= top <= min(args[3], MAX_TOP):
        raise ValueError(f'top: 0 ... min(n, {MAX_TOP}), got {top} for n = {args[3]}')
    stream = _stream(dev)
    actions = actions.contiguous()
    log_prob = torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    stats = torch.empty((args[2], 2), dtype=torch.float32, device=dev) if want_stats else None
    top_lp = torch.empty(lead + (top,), dtype=torch.float32, device=dev) if top else None
    top_a = torch.empty(lead + (top,), dtype=torch.int32, device=dev) if top else None
    ws, ws_bytes, ws_tensor = _workspace(_LOG_PROBS, args, top, dev)
    _check(nat.lib().mgx_policy_log_probs(
        dev.index, *args, actions.data_ptr(), actions.element_size(), top, log_prob.data_ptr(), entropy.data_ptr(),
        stats.data_ptr() if want_stats else None, top_lp.data_ptr() if top else None, top_a.data_ptr() if top else None,
        ws, ws_bytes, stream))
    return log_prob, entropy, top_lp, top_a, stats, actions


def _upstream(g):
    """(pointer, row stride, tensor) of an upstream gradient: f32, one value a row, or one for all (an expanded scalar's)."""
    if g is None:
        return None, 0, None
    g = g.reshape(-1)
    return g.data_ptr(), g.stride(0) if g.numel() > 1 else 1, g


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, mask, temperature, top):
        log_prob, entropy, top_lp, top_a, stats, actions = _forward(logits, actions, mask, temperature, top, True)
        ctx.save_for_backward(logits, actions, mask, stats, entropy)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if top_lp is not None:
            ctx.mark_non_differentiable(top_lp, top_a)
        return log_prob, entropy, top_lp, top_a

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_prob, g_entropy, _g_top_lp, _g_top_a):
        if g_log_prob is None and g_entropy is None:
            return None, None, None, None, None
        logits, actions, mask, stats, entropy = ctx.saved_tensors
        args, kept = _rows(logits, mask, ctx.temperature)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        lp_ptr, lp_stride, lp_kept = _upstream(g_log_prob)
        h_ptr, h_stride, h_kept = _upstream(g_entropy)
        _check(nat.lib().mgx_policy_log_probs_backward(
            logits.device.index, *args, actions.data_ptr(), actions.element_size(), stats.data_ptr(), entropy.data_ptr(),
            lp_ptr, lp_stride, h_ptr, h_stride, grad.data_ptr(), _stream(logits.device)))
        return grad, None, None, None, None


def action_log_probs(logits, actions, *, mask=None, temperature=1.0, top=0):
    """Log probabilities of given actions under softmax(logits / temperature), the distributions' entropies, and the `top` best
    alternatives of each row (best first, equal logits by the lower index).

    logits [..., n]; actions int32 / int64 [...]: a negative one marks a row in which none is given (a padded step: log probability 0,
    no gradient through it; entropy and alternatives are still there), one >= n gives NaN.  top: 0 ... min(n, 64).
    Differentiable to the logits through log_prob and entropy (once); the gradient has the logits' type and is 0 wherever an action is
    not open.  Returns ActionLogProbs."""
    if torch.is_grad_enabled() and torch.is_tensor(logits) and logits.requires_grad:
        return ActionLogProbs(*_ActionLogProbs.apply(logits, actions, mask, temperature, top))
    return ActionLogProbs(*_forward(logits, actions, mask, temperature, top, False)[:4])


def sample_actions(logits, uniforms, *, mask=None, temperature=1.0):
    """One action per row, drawn from softmax(logits / temperature) by the given random numbers: the first action j with
    p_0 + ... + p_j > u, the sums in 64 bits, so that it does not depend on how they are split.  uniforms: float32 / float64 [...] in
    [0, 1), one a row (`torch.rand`); numbers outside are taken as the nearest end.  Returns SampledActions (no gradient: for that,
    give the drawn actions to `action_log_probs`)."""
    args, kept = _rows(logits, mask, temperature)
    lead, dev = logits.shape[:-1], logits.device
    if not torch.is_tensor(uniforms) or uniforms.dtype not in (torch.float32, torch.float64):
        raise TypeError('uniforms: a float32 or float64 tensor')
    if uniforms.device != dev:
        raise ValueError(f'uniforms are on {uniforms.device}, logits on {dev}')
    if uniforms.shape != lead:
        raise ValueError(f'uniforms: one for each row of logits, {tuple(lead)}, got {tuple(uniforms.shape)}')
    stream = _stream(dev)
    uniforms = uniforms.contiguous()
    action = torch.empty(lead, dtype=torch.int32, device=dev)
    log_prob = torch.empty(lead, dtype=torch.float32, device=dev)
    entropy = torch.empty(lead, dtype=torch.float32, device=dev)
    ws, ws_bytes, ws_tensor = _workspace(_SAMPLE, args, 0, dev)
    _check(nat.lib().mgx_policy_sample(dev.index, *args, uniforms.data_ptr(), uniforms.element_size(), action.data_ptr(),
                                       log_prob.data_ptr(), entropy.data_ptr(), ws, ws_bytes, stream))
    return SampledActions(action, log_prob, entropy)
