"""Trains a policy over tokens on the loader's windows, distils it into a smaller one, and rolls that out from caches.

    python examples/train_token_model.py [--steps 200] [--batch 256]

A synthetic table of trajectories: observations of four numbers, given to the model in 64 bins each, and one of ten actions
that a fixed function of the observation prefers.  Windows of 16 steps with padding at the head and validity masks."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gear_amd.dataset import SharedDataset  # noqa: E402
from gear_amd.loader import OfflineLoader  # noqa: E402
from gear_amd.mpu import ModelParallelismUnit  # noqa: E402
from gear_amd.sequence import Rollouts, TokenModel  # noqa: E402
from gear_amd.specs import TableSpec  # noqa: E402

OBSERVATION, ACTIONS, BINS, SPAN, LENGTH = 4, 10, 64, 16, 48
VOCAB = ACTIONS + BINS  # actions first


def model(width=128, layers=2):
    return TokenModel(VOCAB, OBSERVATION + 1, width=width, layers=layers)


def bins(observation):
    """Numbers of O(1) -> tokens."""
    return ACTIONS + ((observation.clamp(-2.99, 2.99) + 3) * (BINS / 6)).long()


def preferred(observation):
    g = torch.Generator().manual_seed(1)
    return (observation @ torch.randn(OBSERVATION, ACTIONS, generator=g).to(observation.device)).argmax(-1)


def dataset(capacity=256, key=None):
    spec = TableSpec.create(trajectory_length=LENGTH, capacity=capacity, column_specs=[
        {"shape": [OBSERVATION], "dtype": torch.float32, "name": "observations"},
        {"shape": [], "dtype": torch.int64, "name": "actions"},
        {"shape": [], "dtype": torch.uint8, "name": "done"}])
    data = SharedDataset.create(spec, key=os.getpid() if key is None else key, placement="device")
    g = torch.Generator().manual_seed(0)
    for i in range(capacity):
        observations = torch.randn(LENGTH, OBSERVATION, generator=g)
        done = (torch.rand(LENGTH, generator=g) < 0.02).to(torch.uint8)
        data[i] = (1.0, int(torch.randint(5, LENGTH + 1, (1,), generator=g)), [observations, preferred(observations), done])
    return data


def loader(data, batch):
    window = dict(offset=-SPAN, length=SPAN, pad="head")
    return OfflineLoader(data, batch, ModelParallelismUnit(), "Uniform",
                         [dict(name=n, **window) for n in ("observations", "actions", "done")],
                         timesteps_on_device=True, with_mask=True)


def _train(policy, batches, steps, loss_of, lr):
    optimizer = torch.optim.AdamW(policy.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        _, (observations, actions, done) = next(batches)
        mask = batches.last_masks[0]
        tokens = torch.cat([bins(observations), actions[..., None]], -1)
        loss = loss_of(tokens, mask, done).sum() / mask.sum().clamp(min=1)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses)


def clone(policy, batches, steps, lr=2e-3, bonus=0.01):
    """Learns the table's actions, with a bonus for entropy."""
    def loss_of(*windows):
        log_probs, entropy = policy.log_probs(*windows)[:2]
        return -(log_probs + bonus * entropy)

    return _train(policy, batches, steps, loss_of, lr)


def distil(policy, teacher, batches, steps, lr=2e-3):
    """Learns a teacher's best actions and how probable it finds them."""
    return _train(policy, batches, steps, lambda *windows: policy.distilled(teacher, *windows, count=5), lr)


def act(policy, batch):
    """Whether the best action is the preferred one, [batch, SPAN]."""
    rollouts, action, right = Rollouts(policy, batch, SPAN * (OBSERVATION + 1)), None, []
    for _ in range(SPAN):
        observation = torch.randn(batch, OBSERVATION, device="cuda")
        _, _, best = policy.step(rollouts, bins(observation), action)
        action = best[:, 0]
        right.append(action == preferred(observation))
    return torch.stack(right, 1)


def main():
    args = argparse.ArgumentParser()
    args.add_argument("--steps", type=int, default=200)
    args.add_argument("--batch", type=int, default=256)
    args = args.parse_args()
    torch.manual_seed(0)
    batches = loader(dataset(), args.batch)
    teacher, student = model().cuda(), model(width=64, layers=1).cuda()
    losses = clone(teacher, batches, args.steps).tolist()
    print("cloning: loss first %.4f, last %.4f" % (losses[0], losses[-1]))
    losses = distil(student, teacher, batches, args.steps).tolist()
    print("distillation: loss first %.4f, last %.4f" % (losses[0], losses[-1]))
    print("preferred actions in rollouts: %.2f" % float(act(student, 64).float().mean()))


if __name__ == "__main__":
    main()
