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
softmax(logits / temperature), temperature in 1e-37 ... 1e37, over the actions that are open (not ruled out, logit above -inf).  Results are
float32 whatever the logits' type.  Rows with nothing open give log probability -inf, entropy 0 and action -1 with gradient 0; rows with NaN
or +inf among the open logits give NaN and action -1.  Calls run on torch's current stream of the logits' device.

Calls, and the backward pass with its forward call, can be captured into a HIP graph and replayed.  While a backward pass is captured, no
results of earlier calls on the same leaves (a logits tensor, a network's weights) and the default stream may be alive: torch would make that
stream part of the capture, which it cannot be, and end the process.  Where the backward pass would come to such a leaf by way of these
operators it is refused (MgxError; where the logits are one themselves, the forward call).
"""
from typing import TYPE_CHECKING, NamedTuple, Optional

from . import _native as nat

if TYPE_CHECKING:                # (the package is imported without torch, which comes with the first env or call)
    import torch

__all__ = ['ActionLogProbs', 'SampledActions', 'action_log_probs', 'sample_actions', 'MAX_TOP']

MAX_TOP = 64                     # MGX_POLICY_MAX_TOP
_ops = None                      # csrc/policy/mgx_policy_torch.cpp: argument checks, outputs, autograd, the C calls; loaded by the first call


def _load():
    global _ops
    import torch  # noqa: F401  (the module's types are torch's)
    _ops = nat.policy_ops()
    return _ops


class ActionLogProbs(NamedTuple):
    log_prob: 'torch.Tensor'                    # f32 [...]: log p of the given action
    entropy: 'torch.Tensor'                     # f32 [...]
    top_log_probs: Optional['torch.Tensor']     # f32 [..., top], best first (None if top == 0); no gradient
    top_actions: Optional['torch.Tensor']       # i32 [..., top]; -1 where a row has no more open actions


class SampledActions(NamedTuple):
    action: 'torch.Tensor'       # i32 [...]; -1 where nothing is open
    log_prob: 'torch.Tensor'     # f32 [...]
    entropy: 'torch.Tensor'      # f32 [...]


def action_log_probs(logits, actions, *, mask=None, temperature=1.0, top=0):
    """Log probabilities of given actions under softmax(logits / temperature), the distributions' entropies, and the `top` best
    alternatives of each row (best first, equal logits by the lower index).

    logits [..., n]; actions int32 / int64 [...]: a negative one marks a row in which none is given (a padded step: log probability 0,
    no gradient through it, whatever the row's logits; entropy and alternatives are still there), one >= n gives NaN, and NaN as gradient
    unless nothing flows back through its log probability.  top: 0 ... min(n, 64).
    Differentiable to the logits through log_prob and entropy (once, backwards; logits or upstream gradients with a forward-mode tangent
    are refused, NotImplementedError); the gradient has the logits' type and is 0 wherever an action is not open.  Returns ActionLogProbs.
    Refuses wrong types (TypeError), shapes, devices and ranges (ValueError), and to be traced (torch.jit.trace: NotImplementedError)."""
    return ActionLogProbs(*(_ops or _load()).log_probs(logits, actions, mask, temperature, top))


def sample_actions(logits, uniforms, *, mask=None, temperature=1.0):
    """One action per row, drawn from softmax(logits / temperature) by the given random numbers: the first action j with
    p_0 + ... + p_j > u, the sums in 64 bits (a u within some n * 2^-53 of a border between two actions can fall on either side of it, by the
    number of rows; a repeated call draws the same).  uniforms: float32 / float64 [...] in [0, 1), one a row (`torch.rand`); numbers outside
    are taken as the nearest end.  Returns SampledActions (no gradient, of any mode: for that, give the drawn actions to
    `action_log_probs`).  Other refusals are those of `action_log_probs`."""
    return SampledActions(*(_ops or _load()).sample(logits, uniforms, mask, temperature))
