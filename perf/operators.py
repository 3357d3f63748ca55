"""What is measured of the operators on a policy's action scores: log probabilities of given actions with the entropy and the best
alternatives (`action_log_probs`), the gradient of the two (its backward pass), and actions drawn with given random numbers
(`sample_actions`).

The scores are rows of `n` logits.  One env-step of every task chooses among n = 18 actions; a policy that answers with the next c
env-steps at once has n = 18^c classes (324, 5832, 104976); one that answers in tokens of a vocabulary has some ten thousand.  Rows are
envs (4096 in the benchmark's batches), demonstrations, or whole rollouts (4096 envs x 60 ... 240 env-steps)."""
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


def _case(name, op, rows, n, dtype, top=0, mask='none', layout='dense', temperature=1.0, padded=0.0):
    return {'name': name, 'op': op, 'rows': rows, 'n': n, 'dtype': dtype, 'top': top, 'mask': mask, 'layout': layout,
            'temperature': temperature, 'padded': padded}


def listed():
    return [
        # one env-step of a replay of a few dozen demonstrations: how likely was the recorded action, what would the policy rather do
        _case('score_replay_step', 'score', 61, 18, 'f32', top=3),
        # every (frame, action) pair of 4096 episodes of 80 env-steps: held-out likelihood and agreement with the best action
        _case('score_dataset', 'score', 327680, 18, 'bf16', top=1, padded=0.05),
        # chunks of three actions for every env of the batch, some chunks ruled out per env
        _case('score_chunks', 'score', 4096, 5832, 'bf16', top=5, mask='rows'),
        # a few requests of a policy that answers in tokens, twenty alternatives each
        _case('score_tokens_few', 'score', 7, 50021, 'f32', top=20),
        # one minibatch of an imitation learner
        _case('train_minibatch', 'train', 2048, 18, 'f32'),
        # a whole rollout of 4096 envs x 240 env-steps in one step of the learner
        _case('train_rollout', 'train', 983040, 18, 'f32'),
        # the same from a head that also gives a value: 18 of 19 columns, episodes padded to a common length
        _case('train_actor_critic', 'train', 245760, 18, 'f16', layout='head', padded=0.25),
        # chunks of two actions, 15 env-steps of 4096 envs, some chunks ruled out for all
        _case('train_chunks', 'train', 61440, 324, 'bf16', mask='shared'),
        # chunks of four actions: the largest
        _case('train_long_chunks', 'train', 1024, 104976, 'bf16'),
        # the rollout's own call: one action for each of 4096 envs
        _case('sample_step', 'sample', 4096, 18, 'f32'),
        # chunks of three actions for every env, at a lower temperature
        _case('sample_chunks', 'sample', 4096, 5832, 'bf16', temperature=0.7),
        # a few envs, chunks of four actions
        _case('sample_long_chunks', 'sample', 16, 104976, 'f32', mask='shared'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['score', 'train', 'sample'])
    n = rng.choice([18, 18, 324, 5832, 104976] + [_log_int(rng, 2, 110000)] * 5)
    rows = _log_int(rng, 1, max(1, min(983040, (48 << 20) // n)))
    return {'op': op, 'rows': rows, 'n': n, 'dtype': rng.choice(['f32', 'bf16', 'f16']),
            'top': min(n, rng.choice([0, 1, 3, 5, 20, 32])) if op == 'score' else 0,
            'mask': rng.choice(['none', 'none', 'shared', 'rows']), 'layout': rng.choice(['dense', 'dense', 'head']),
            'temperature': rng.choice([1.0, 1.0, 0.7, 2.0]), 'padded': rng.choice([0.0, 0.1]) if op != 'sample' else 0.0}


def _inputs(case, seed, device):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    rows, n, dt = case['rows'], case['n'], DTYPES[case['dtype']]
    wide = n + 1 if case['layout'] == 'head' else n
    # a policy's scores: spread by some units, and in half of the rows one of them well ahead of the others
    head = torch.randn((rows, wide), generator=g, device=device, dtype=torch.float32).mul_(2.5)
    best = torch.randint(0, n, (rows, 1), generator=g, device=device)
    ahead = torch.rand((rows, 1), generator=g, device=device).sub_(0.5).clamp_(min=0).mul_(24)
    head.scatter_add_(1, best, ahead)
    head = head.to(dt)
    actions = torch.where(torch.rand((rows, 1), generator=g, device=device) < 0.5, best,
                          torch.randint(0, n, (rows, 1), generator=g, device=device))[:, 0]
    pad = torch.rand((rows,), generator=g, device=device) < case['padded']
    actions = torch.where(pad, torch.full_like(actions, -1), actions)
    mask = None
    if case['mask'] == 'shared':      # an action that is ruled out for every env (the first one never is)
        mask = torch.rand((n,), generator=g, device=device) < 0.8
        mask[0] = True
    elif case['mask'] == 'rows':      # per env; in one row of 64 nothing is left
        mask = torch.rand((rows, n), generator=g, device=device) < 0.8
        mask &= torch.rand((rows, 1), generator=g, device=device) >= 1 / 64
    uniforms = torch.rand((rows,), generator=g, device=device)
    # a policy gradient's weights, and an entropy bonus
    grad_log_prob = torch.randn((rows,), generator=g, device=device)
    grad_entropy = torch.full((1,), -0.01, device=device).expand(rows)
    return {'logits': head[:, :n], 'actions': actions, 'mask': mask, 'uniforms': uniforms,
            'grad_log_prob': grad_log_prob, 'grad_entropy': grad_entropy}


def prepare(case, seed):
    state = _inputs(case, seed, 'cuda')
    state['logits'] = state['logits'].detach().requires_grad_(case['op'] == 'train')
    state['case'] = case
    return state


def run(state):
    case = state['case']
    if own:
        return _own(state, case)
    with torch.no_grad():
        if case['op'] == 'sample':
            return _plain_sample(state['logits'], state['uniforms'], state['mask'], case['temperature'])
        return _plain_score(state, case)


# ---------------------------------------------------------------------------------------------- the framework's calls
def _own(state, case):
    import magical_amd
    if case['op'] == 'sample':
        out = magical_amd.sample_actions(state['logits'], state['uniforms'], mask=state['mask'], temperature=case['temperature'])
        return {'action': out.action, 'log_prob': out.log_prob, 'entropy': out.entropy}
    out = magical_amd.action_log_probs(state['logits'], state['actions'], mask=state['mask'], temperature=case['temperature'],
                                       top=case['top'])
    if case['op'] == 'train':
        grad, = torch.autograd.grad((out.log_prob, out.entropy), (state['logits'],), (state['grad_log_prob'], state['grad_entropy']))
        return {'log_prob': out.log_prob.detach(), 'entropy': out.entropy.detach(), 'grad': grad}
    return {'log_prob': out.log_prob, 'entropy': out.entropy, 'top_log_probs': out.top_log_probs, 'top_actions': out.top_actions}


# ---------------------------------------------------------------------------------------------- the plain forms
def _plain_score(state, case):
    x, actions, mask = state['logits'].float(), state['actions'], state['mask']
    n, inv_t = x.shape[1], 1.0 / case['temperature']
    neg = float('-inf')
    if mask is not None:
        x = torch.where(mask, x, neg)
    top = x.amax(1, keepdim=True)
    some = top > neg                                          # rows in which something is allowed
    d = torch.where(x > neg, (x - top) * inv_t, neg)          # a row with nothing allowed: all of it -inf
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    t = torch.where(x > neg, e * d, 0.0).sum(1, keepdim=True)
    entropy = torch.where(some, log_s - t / s, 0.0)
    given = actions >= 0
    at = actions.clamp(min=0)[:, None]
    d_at = d.gather(1, at)
    log_prob = torch.where(given[:, None], torch.where(some, d_at - log_s, neg), 0.0)
    if case['op'] == 'train':
        p = torch.where(some, e / s, 0.0)
        log_p = torch.where(x > neg, d - log_s, 0.0)
        g_lp = torch.where(given, state['grad_log_prob'], 0.0)[:, None]
        g_h = state['grad_entropy'][:, None]
        grad = -p * (g_lp + g_h * (log_p + entropy))
        grad.scatter_add_(1, at, torch.where(d_at > neg, g_lp, 0.0))
        grad = (grad * inv_t).to(state['logits'].dtype)
        return {'log_prob': log_prob[:, 0], 'entropy': entropy[:, 0], 'grad': grad}
    k = case['top']
    if k == 0:
        return {'log_prob': log_prob[:, 0], 'entropy': entropy[:, 0], 'top_log_probs': None, 'top_actions': None}
    # the best k, ties to the lowest index: whole-number keys, the value's order first and then the index
    bits = (x + 0.0).contiguous().view(torch.int32).long()    # (+ 0.0: the two zeros are one value)
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))
    key = order * (1 << 31) + (n - 1 - torch.arange(n, device=x.device))
    top_actions = (n - 1) - (torch.topk(key, k, dim=1).values & 0x7fffffff)
    there = x.gather(1, top_actions) > neg
    top_log_probs = torch.where(there, d.gather(1, top_actions) - log_s, neg)
    return {'log_prob': log_prob[:, 0], 'entropy': entropy[:, 0], 'top_log_probs': top_log_probs,
            'top_actions': torch.where(there, top_actions, -1).int()}


def _plain_sample(logits, uniforms, mask, temperature):
    # in 64 bits: a running sum next to the drawn number decides which action it is
    x, neg = logits.double(), float('-inf')
    if mask is not None:
        x = torch.where(mask, x, neg)
    top = x.amax(1, keepdim=True)
    some = top > neg
    d = torch.where(x > neg, (x - top) * (1.0 / temperature), neg)
    e = torch.exp(d)
    c = e.cumsum(1)
    s = c[:, -1:]
    action = (c <= uniforms.double()[:, None] * s).sum(1, keepdim=True).clamp(max=x.shape[1] - 1)
    log_s = torch.log(s)
    t = torch.where(x > neg, e * d, 0.0).sum(1, keepdim=True)
    log_prob = torch.where(some, d.gather(1, action) - log_s, neg)
    entropy = torch.where(some, log_s - t / s, 0.0)
    action = torch.where(some, action, -1)
    return {'action': action[:, 0].int(), 'log_prob': log_prob[:, 0].float(), 'entropy': entropy[:, 0].float()}


# ---------------------------------------------------------------------------------------------- in 64 bits, from the definition
def exact(case, seed):
    inp = _inputs(case, seed, 'cuda')
    z = inp['logits'].double()
    neg = float('-inf')
    closed = torch.isneginf(z) if inp['mask'] is None else torch.isneginf(z) | ~inp['mask']
    dead = closed.all(1)
    z = z.requires_grad_(case['op'] == 'train')
    # log p = z / T - log sum exp(z / T); a dead row is computed as if nothing were closed in it and replaced afterwards
    shut = closed & ~dead[:, None]
    log_p = torch.log_softmax((z / case['temperature']).masked_fill(shut, neg), 1)
    kept = log_p.masked_fill(shut, 0.0)
    entropy = -(kept * kept.exp().masked_fill(shut, 0.0)).sum(1).masked_fill(dead, 0.0)
    if case['op'] == 'sample':
        cdf = log_p.exp().cumsum(1)
        found = torch.searchsorted(cdf, (inp['uniforms'].double() * cdf[:, -1])[:, None], right=True).clamp(max=case['n'] - 1)
        log_prob = log_p.gather(1, found)[:, 0].masked_fill(dead, neg)
        return {'action': found[:, 0].masked_fill(dead, -1).int(), 'log_prob': log_prob, 'entropy': entropy}
    acts, pad = inp['actions'].clamp(min=0)[:, None], inp['actions'] < 0
    log_prob = log_p.gather(1, acts)[:, 0].masked_fill(dead, neg).masked_fill(pad, 0.0)
    if case['op'] == 'train':
        # d/dz of sum(g_lp log p[a]) + sum(g_h H); an action that is closed contributes only through the others' sum
        at_closed = closed.gather(1, acts)[:, 0]
        chosen = torch.where(at_closed, -torch.logsumexp((z / case['temperature']).masked_fill(shut, neg), 1), log_p.gather(1, acts)[:, 0])
        chosen = chosen.masked_fill(pad | dead, 0.0)
        total = (inp['grad_log_prob'].double() * chosen).sum() + (inp['grad_entropy'].double() * entropy).sum()
        grad, = torch.autograd.grad(total, (z,))
        return {'log_prob': log_prob.detach(), 'entropy': entropy.detach(), 'grad': grad}
    k = case['top']
    if k == 0:
        return {'log_prob': log_prob, 'entropy': entropy, 'top_log_probs': None, 'top_actions': None}
    values, order = z.masked_fill(closed, neg).sort(dim=1, descending=True, stable=True)
    none = torch.isneginf(values[:, :k])
    return {'log_prob': log_prob, 'entropy': entropy, 'top_log_probs': log_p.gather(1, order[:, :k]).masked_fill(none, neg),
            'top_actions': order[:, :k].masked_fill(none, -1).int()}


def work(case):
    rows, n, size = case['rows'], case['n'], SIZE[case['dtype']]
    logits = rows * n * size
    mask = {'none': 0, 'shared': n, 'rows': rows * n}[case['mask']]
    if case['op'] == 'sample':      # logits, the drawn number; action, log probability, entropy
        return {'bytes': logits + mask + rows * (4 + 4 + 4 + 4), 'flops': 6 * rows * n}
    given = rows * (8 + 4 + 4)      # the action; log probability, entropy
    if case['op'] == 'train':       # ... the two upstream gradients (the entropy's is one number), the logits' gradient
        return {'bytes': 2 * logits + mask + given + rows * 4 + 4, 'flops': 12 * rows * n}
    return {'bytes': logits + mask + given + rows * case['top'] * (4 + 4), 'flops': 6 * rows * n}
