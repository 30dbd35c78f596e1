"""Train a small token policy with the package's training operators, then verify what it learned.

A policy reads a context of four tokens and answers with one of eight actions; the right one
follows from the context.  It is trained in two stages, as such policies are: sampled actions and the
clipped policy loss, then pairs of a right and a wrong action and the preference loss, with AdamW and its
moments in 8 bits.  Before them it may imitate right actions (--imitate), with dropout of the hidden layer and the
cross entropy of its head.  Before and after, the same contexts are verified: every perturbation of the embedded
context within a Linf ball has to leave the right action's logit the largest (CROWN bounds of
its margins).

    python examples/train_and_verify.py [--steps 120] [--contexts 512] [--eps 0.05] [--imitate 0]

Needs an MI355X and the built library (python -m boundflow_amd.build).
"""

from __future__ import annotations

import argparse
import copy
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from boundflow_amd import crown, frontend, training  # noqa: E402
from boundflow_amd import workloads as wl  # noqa: E402
from boundflow_amd.ir import BFTaskModule  # noqa: E402
from boundflow_amd.spec import InputSpec  # noqa: E402

VOCAB, CONTEXT, DIM, HIDDEN, ACTIONS = 97, 4, 24, 160, 8
SCALE = DIM ** 0.5     # of the looked-up rows


class Policy:
    """A token table (trained through the package's own lookup) and an MLP (through autograd)."""

    def __init__(self, device, seed: int = 0):
        g = torch.Generator().manual_seed(seed)
        self.table = (torch.randn(VOCAB, DIM, generator=g) / SCALE).to(device)
        torch.manual_seed(seed)
        self.net = torch.nn.Sequential(torch.nn.Linear(CONTEXT * DIM, HIDDEN), torch.nn.ReLU(),
                                       torch.nn.Linear(HIDDEN, ACTIONS)).to(device)
        self.params = [self.table, *self.net.parameters()]
        self.optimizer = training.AdamW(self.params, lr=5e-3, betas=(0.9, 0.98), weight_decay=1e-3, bits=8)

    def embed(self, contexts):
        return training.embed_tokens(self.table, contexts, scale=SCALE).flatten(1)

    def step(self, contexts, loss_of_logits):
        """One training step; ``loss_of_logits`` returns a loss result with ``grad_logits``."""
        x = self.embed(contexts).requires_grad_(True)
        logits = self.net(x)
        result = loss_of_logits(logits.detach())
        grads = torch.autograd.grad(logits, [x, *self.net.parameters()], result.grad_logits)
        table_grad = training.embed_tokens_grad(grads[0].view(-1, CONTEXT, DIM), contexts, VOCAB, scale=SCALE)
        self.optimizer.step([table_grad, *grads[1:]])
        return result

    def imitate(self, contexts, actions, drop: float):
        """One supervised step: the layers before the head through autograd, the dropped hidden layer and the head through
        the package.  (the loss result, the gradients in the parameters' order)"""
        x = self.embed(contexts).requires_grad_(True)
        *body, head = self.net
        hidden = torch.nn.Sequential(*body)(x)
        mask = {"seed": 7, "counter": self.optimizer.t}      # another mask each step
        result = training.vocabulary_loss(training.dropout(hidden.detach(), drop, **mask), head.weight.detach(), actions,
                                          bias=head.bias.detach())
        through = training.dropout_grad(result.grad_hidden, drop, **mask)
        grads = torch.autograd.grad(hidden, [x, *(p for layer in body for p in layer.parameters())], through)
        table_grad = training.embed_tokens_grad(grads[0].view(-1, CONTEXT, DIM), contexts, VOCAB, scale=SCALE)
        grads = [table_grad, *grads[1:], result.grad_weight, result.grad_bias]
        self.optimizer.step(grads)
        return result, grads

    def planned(self, example) -> BFTaskModule:
        """The MLP as the bound queries take it."""
        net = copy.deepcopy(self.net).cpu()
        tm = frontend.plan_interval_ibp_v0(frontend.import_torch(net, (example.cpu(),)))
        return BFTaskModule(tasks=tm.tasks, entry_task_id=tm.entry_task_id, storage_plan=tm.storage_plan,
                            bindings={**tm.bindings, "params": {k: v.to(example.device) for k, v in tm.params.items()}})


def right_action(contexts):
    return (contexts[:, 0] + 3 * contexts[:, -1]) % ACTIONS


def verify(policy: Policy, contexts, eps: float):
    """(share answered rightly, share certified within eps, mean lower margin)."""
    x = policy.embed(contexts)
    label = right_action(contexts)
    with torch.no_grad():
        right = float((policy.net(x).argmax(1) == label).float().mean())
    module = policy.planned(x[:2])
    C = wl.margin_spec(label.cpu(), ACTIONS).to(x.device)
    bounds = crown.run_crown_ibp_mlp(module, InputSpec.linf(value_name="input", center=x, eps=eps), linear_spec_C=C)
    margin = bounds.lower.min(1).values
    return right, float((margin > 0).float().mean()), float(margin.mean())


def train(policy: Policy, contexts, steps: int, g):
    """The last policy loss and preference loss."""
    label = right_action(contexts)
    n = contexts.shape[0]
    with torch.no_grad():
        ref_logp = torch.log_softmax(policy.net(policy.embed(contexts)), 1)
    reinforced = preferred = None
    for _ in range(steps):
        with torch.no_grad():
            logp = torch.log_softmax(policy.net(policy.embed(contexts)), 1)
        taken = torch.multinomial(logp.exp(), 1, generator=g)[:, 0]
        reward = (taken == label).float()
        old = logp.gather(1, taken[:, None])[:, 0]
        ref = ref_logp.gather(1, taken[:, None])[:, 0]
        for _pass in range(2):     # two updates on one set of samples
            reinforced = policy.step(contexts, lambda logits: training.policy_loss(
                logits, taken, old, reward - reward.mean(), ref_logp=ref, kl_weight=0.01, clip_high=0.28))
    with torch.no_grad():
        ref_logp = torch.log_softmax(policy.net(policy.embed(contexts)), 1)
    both = torch.cat([contexts, contexts])
    offsets = torch.arange(2 * n + 1, device=contexts.device)      # answers of one token each
    for _ in range(steps):
        wrong = (label + torch.randint(1, ACTIONS, (n,), device=label.device, generator=g)) % ACTIONS
        answers = torch.cat([label, wrong])
        ref = torch.cat([ref_logp, ref_logp]).gather(1, answers[:, None])[:, 0]
        preferred = policy.step(both, lambda logits: training.preference_loss(
            logits, answers, ref, offsets, beta=0.5, label_smoothing=0.02))
    return float(reinforced.loss), float(preferred.loss)


def imitate(policy: Policy, contexts, steps: int, drop: float = 0.1):
    """The losses of a supervised stage."""
    label = right_action(contexts)
    return [policy.imitate(contexts, label, drop)[0].loss for _ in range(steps)]


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=120)
    ap.add_argument("--contexts", type=int, default=512)
    ap.add_argument("--eps", type=float, default=0.05)
    ap.add_argument("--imitate", type=int, default=0, help="supervised steps before the two stages")
    a = ap.parse_args(argv)
    device = torch.device("cuda:0")
    g = torch.Generator(device=device).manual_seed(1)
    contexts = torch.randint(0, VOCAB, (a.contexts, CONTEXT), device=device, generator=g)
    policy = Policy(device)
    before = verify(policy, contexts, a.eps)
    imitated = [float(loss) for loss in imitate(policy, contexts, a.imitate)]
    losses = train(policy, contexts, a.steps, g)
    after = verify(policy, contexts, a.eps)
    for name, (right, certified, margin) in (("before", before), ("after", after)):
        print(f"{name:>6}: {100 * right:5.1f} % answered rightly, {100 * certified:5.1f} % certified within {a.eps}, "
              f"mean lower margin {margin:+.3f}", flush=True)
    if imitated:
        print(f"imitation: loss {imitated[0]:.4f} at first, {imitated[-1]:.4f} at last")
    print(f"last losses: policy {losses[0]:.4f}, preference {losses[1]:.4f}")
    return {"before": before, "after": after, "losses": losses, "imitated": imitated}


if __name__ == "__main__":
    main()
