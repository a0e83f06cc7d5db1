"""A small recurrent policy trained with the training stages, end to end.

The task is recall: a sequence shows a token, then noise, and at every step the
policy is rewarded for naming the first token.  One layer holds a gated
recurrence on a residual branch with dropout; the products by its weights are
torch's, everything between them is hawk's, a traced kernel and its stages:

* the forward and its reverse: ``recurrence`` (sigmoid gates) and ``dropout``;
* rollouts: ``token_logp`` of the sampled actions; a traced kernel, a sample a
  step, turns rewards and ends into the planes of a reversed ``recurrence``, which
  sums the discounted rewards;
* the update: ``policy_loss`` (clipped, with a KL term to the first policy),
  its gradient in the same pass over the logits;
* then a few steps of ``preference_loss`` on pairs of answers;
* serving: the same recurrence a token at a time.

Run it on a ROCm device: ``python examples/recurrent_policy.py``.
"""

from __future__ import annotations

import sys
import tempfile
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import hawk_amd as hawk  # noqa: E402
from hawk_amd import Mutable, Param, Scalar  # noqa: E402

TOKENS, WIDTH, STEPS, SEQUENCES = 16, 64, 12, 250
DISCOUNT = 0.5


@hawk.kernel
def gains(reward: Scalar, ends: Scalar, baseline: Param, gate: Mutable[Scalar], x: Mutable[Scalar]):
    """One step's part of the discounted sum: what comes after an end is cut."""
    gate = DISCOUNT * (1.0 - ends)
    x = reward - baseline


class Policy:
    """``logits = (u + dropout(recurrence(u Wz, u Wx))) Wo`` of embedded tokens u."""

    def __init__(self, device, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(shape, generator=g, device=device) * scale
        self.embed = normal(TOKENS + 1, WIDTH)                   # the last row marks "shown, remember"
        self.weights = {"z": normal(WIDTH, WIDTH, scale=0.1), "x": normal(WIDTH, WIDTH, scale=0.2),
                        "o": normal(WIDTH, TOKENS, scale=0.05)}
        self.bias = torch.full((WIDTH,), 2.0, device=device)
        self.scan = hawk.stages.recurrence(gate="sigmoid")
        self.drop = hawk.stages.dropout(0.1)
        self.adam = torch.optim.Adam(list(self.weights.values()), lr=3e-3)
        self.seed, self.calls = 1234 + seed, 0

    def embedded(self, tokens):
        u = self.embed[tokens]
        u[:, 0] += self.embed[TOKENS]
        return u

    def forward(self, tokens, train: bool):
        """The logits of every step, and what the reverse needs."""
        u = self.embedded(tokens)
        z, x = u @ self.weights["z"] + self.bias, u @ self.weights["x"]
        h, y = torch.empty_like(x), torch.empty_like(x)
        hawk.run(self.scan, gate=z, x=x, h=h)
        self.calls += 1
        if train:
            hawk.run(self.drop, x=h, residual=u, y=y, seed=self.seed, offset=self.calls)
        else:
            torch.add(u, h, out=y)
        return (y @ self.weights["o"]).reshape(-1, TOKENS), (u, z, x, h, y, self.calls)

    def update(self, saved, bar_logits):
        """One step of the weights, from the gradient by the logits."""
        u, z, x, h, y, call = saved
        bar_logits = bar_logits.view(*u.shape[:2], TOKENS)
        bar_y = bar_logits @ self.weights["o"].t()
        bar_h, bar_z, bar_x = (torch.empty_like(h) for _ in range(3))
        hawk.run(self.drop.vjp, bar_y=bar_y, bar_x=bar_h, seed=self.seed, offset=call)
        hawk.run(self.scan.vjp, gate=z, x=x, h=h, bar_h=bar_h, bar_gate=bar_z, bar_x=bar_x)
        flat = u.reshape(-1, WIDTH).t()
        self.weights["z"].grad = flat @ bar_z.reshape(-1, WIDTH)
        self.weights["x"].grad = flat @ bar_x.reshape(-1, WIDTH)
        self.weights["o"].grad = y.reshape(-1, WIDTH).t() @ bar_logits.reshape(-1, TOKENS)
        self.adam.step()

    def answer(self, tokens):
        """Greedy actions a token at a time: the state alone is kept between steps."""
        u = self.embedded(tokens)
        state = torch.zeros(len(tokens), WIDTH, device=u.device)
        h, actions = torch.empty(len(tokens), 1, WIDTH, device=u.device), []
        for t in range(tokens.shape[1]):
            now = u[:, t:t + 1]
            hawk.run(self.scan, gate=now @ self.weights["z"] + self.bias, x=now @ self.weights["x"], h=h, h0=state,
                     last=state)
            actions.append(((now + h) @ self.weights["o"]).argmax(-1))
        return torch.cat(actions, 1)


def logp_of(logits, actions):
    out, lse = (torch.empty(len(actions), device=logits.device) for _ in range(2))
    hawk.run(hawk.stages.token_logp(), logits=logits, target=actions, logp=out, lse=lse)
    return out


def train(device="cuda:0", rounds: int = 60, seed: int = 0, tell=None) -> dict:
    """Policy optimisation, then preferences; what each reached."""
    g = torch.Generator(device=device).manual_seed(seed + 1)

    def episodes(n):
        return torch.randint(0, TOKENS, (n, STEPS), generator=g, device=device)
    policy, first = Policy(device, seed), Policy(device, seed)
    returns = hawk.stages.recurrence(reverse=True)
    loss_of = hawk.stages.policy_loss(clip=(0.2, 0.28), kl=0.01)
    with tempfile.TemporaryDirectory() as unit:
        hawk.build([gains], unit, mode="float32")
        step_gains = hawk.load(unit, "gains")
    ends, (gate, x) = torch.zeros(SEQUENCES, STEPS, 1, device=device), torch.empty(2, SEQUENCES, STEPS, 1, device=device)
    ends[:, -1] = 1.0                                            # the episode ends here
    rewards = []
    for k in range(rounds):
        tokens = episodes(SEQUENCES)
        logits, _ = policy.forward(tokens, train=False)
        actions = torch.multinomial(torch.softmax(logits, 1), 1, generator=g)[:, 0]
        reward = (actions.view(SEQUENCES, STEPS) == tokens[:, :1]).float()
        rewards.append(float(reward.mean()))
        hawk.run(step_gains, reward=reward.flatten(), ends=ends.flatten(), baseline=rewards[-1], gate=gate.flatten(),
                 x=x.flatten())
        gain = torch.empty_like(gate)
        hawk.run(returns, gate=gate, x=x, h=gain)
        planes = dict(target=actions, old_logp=logp_of(logits, actions), advantage=gain.flatten() / (gain.std() + 1e-6),
                      ref_logp=logp_of(first.forward(tokens, train=False)[0], actions))
        loss = torch.empty(1, device=device)
        for _ in range(4):
            logits, saved = policy.forward(tokens, train=True)
            bar = torch.empty_like(logits)
            hawk.run(loss_of, logits=logits, loss=loss, bar_logits=bar, **planes)
            policy.update(saved, bar)
        if tell and k % 10 == 0:
            tell(f"round {k}: reward {rewards[-1]:.3f}, loss {float(loss):.4f}")

    # pairs of answers to the same episode: the right one before a random one
    pairs = 64
    prefer = hawk.stages.preference_loss(beta=0.2, smoothing=0.05)
    offsets = torch.arange(0, 2 * pairs + 1, device=device) * STEPS
    margin, loss, lse = (torch.empty(n, device=device) for n in (pairs, 1, 2 * pairs * STEPS))
    losses = []
    for _ in range(20):
        tokens = episodes(pairs).repeat_interleave(2, 0)
        target = episodes(2 * pairs)
        target[0::2] = tokens[0::2, :1]
        target[:, 0] = -1                                        # the first step is the prompt
        target = target.flatten()
        reference = logp_of(first.forward(tokens, train=False)[0], target)
        logits, saved = policy.forward(tokens, train=True)
        bar = torch.empty_like(logits)
        planes = dict(logits=logits, target=target, offsets=offsets)
        hawk.run(prefer, ref_logp=reference, loss=loss, margin=margin, lse=lse, **planes)
        hawk.run(prefer.vjp, margin=margin, lse=lse, bar_logits=bar, **planes)
        policy.update(saved, bar)
        losses.append(float(loss))
    tokens = episodes(512)
    right = float((policy.answer(tokens) == tokens[:, :1]).float().mean())
    if tell:
        tell(f"preference loss {losses[0]:.4f} -> {losses[-1]:.4f}; greedy answers right: {right:.3f}")
    return {"rewards": rewards, "preference": losses, "right": right}


if __name__ == "__main__":
    train(tell=lambda line: print(line, flush=True))
