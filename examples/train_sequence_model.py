"""Trains a small causal model on the loader's windows and rolls it out from caches.

    python examples/train_sequence_model.py [--steps 200] [--batch 256]

A synthetic table of trajectories of a linear system whose actions are a fixed function of its observations; windows of
20 steps with padding at the head, validity masks, and a `done` column that ends episodes inside trajectories."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gear_amd.dataset import SharedDataset  # noqa: E402
from gear_amd.loader import OfflineLoader  # noqa: E402
from gear_amd.mpu import ModelParallelismUnit  # noqa: E402
from gear_amd.sequence import Rollouts, WindowModel  # noqa: E402
from gear_amd.specs import TableSpec  # noqa: E402

OBSERVATION, ACTION, SPAN, LENGTH = 17, 6, 20, 64


def policy(observation):
    """What is to be learnt."""
    g = torch.Generator().manual_seed(1)
    w = torch.randn(OBSERVATION, ACTION, generator=g) / OBSERVATION ** 0.5
    return torch.tanh(observation @ w.to(observation.device))


def dataset(capacity=256, key=None):
    spec = TableSpec.create(trajectory_length=LENGTH, capacity=capacity, column_specs=[
        {"shape": [OBSERVATION], "dtype": torch.float32, "name": "observations"},
        {"shape": [ACTION], "dtype": torch.float32, "name": "actions"},
        {"shape": [], "dtype": torch.uint8, "name": "done"}])
    data = SharedDataset.create(spec, key=os.getpid() if key is None else key, placement="device")
    g = torch.Generator().manual_seed(0)
    for i in range(capacity):
        observations = torch.randn(LENGTH, OBSERVATION, generator=g)
        done = (torch.rand(LENGTH, generator=g) < 0.02).to(torch.uint8)
        data[i] = (1.0, int(torch.randint(5, LENGTH + 1, (1,), generator=g)), [observations, policy(observations), done])
    return data


def loader(data, batch):
    window = dict(offset=-SPAN, length=SPAN, pad="head")
    return OfflineLoader(data, batch, ModelParallelismUnit(), "Uniform",
                         [dict(name=n, **window) for n in ("observations", "actions", "done")],
                         timesteps_on_device=True, with_mask=True)


def train(model, batches, steps, lr=2e-3):
    """The losses, one a step."""
    optimizer = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        _, (observations, actions, done) = next(batches)
        mask = batches.last_masks[0]
        error = (model(observations, actions, mask, done) - actions).square().mean(-1)
        loss = (error * mask).sum() / mask.sum().clamp(min=1)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses)


def main():
    args = argparse.ArgumentParser()
    args.add_argument("--steps", type=int, default=200)
    args.add_argument("--batch", type=int, default=256)
    args = args.parse_args()
    torch.manual_seed(0)
    model = WindowModel(OBSERVATION, ACTION).cuda()
    losses = train(model, loader(dataset(), args.batch), args.steps).tolist()
    print("loss: first %.4f, last %.4f" % (losses[0], losses[-1]))
    rollouts, action = Rollouts(model, 64, 2 * SPAN), None
    for _ in range(SPAN):
        observation = torch.randn(64, OBSERVATION, device="cuda")
        action = model.step(rollouts, observation, action)
    print("error of a rollout's last actions: %.4f" % float((action - policy(observation)).square().mean()))


if __name__ == "__main__":
    main()
