"""A sequence policy learns to recall: every episode opens with a cue, ends at a
random step and may ask for its cue at any step; the policy answers with the
action that names it.  Whole sequences train at once (linear attention, gated
projections, AdamW with 8-bit moments, all in one replayed graph); then the
policy acts token by token and its answers are compared.

    python tt-rl_amd/examples/sequence_recall.py [--updates 300]
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

CUES = 4


def episodes(rng, T: int, B: int):
    """-> obs (T, B, CUES + 1) [cue | asked], starts (T, B, 1), the cue's
    one-hot (T, B, CUES) where it is asked for and zeros elsewhere."""
    starts = rng.random((T, B)) < 0.08
    starts[0] = True
    cue = rng.integers(0, CUES, (T, B))
    for t in range(1, T):
        cue[t] = np.where(starts[t], cue[t], cue[t - 1])
    asked = (rng.random((T, B)) < 0.25) & ~starts
    hot = np.eye(CUES, dtype=np.float32)[cue]
    obs = np.concatenate([hot * starts[..., None], asked[..., None]], axis=-1).astype(np.float32)
    return obs, starts[..., None].astype(np.float32), hot * asked[..., None]


def run(device, updates: int = 300, T: int = 48, B: int = 64, seed: int = 0, log=print) -> dict:
    from ttrl_amd.engine import AdamW, Tensor, TrainStep, no_grad
    from ttrl_amd.engine.ops import log_softmax, mul, split, sum_all
    from ttrl_amd.engine.tensor import bound_block
    from ttrl_amd.nets import SequencePolicy

    np.random.seed(seed)
    rng = np.random.default_rng(seed)
    policy = SequencePolicy(CUES + 1, CUES, device, features=64, blocks=2, heads=4, key=16, value=16, hidden=128,
                            kv_heads=2, horizon=64.0)
    optimizer = AdamW(list(policy.parameters()), lr=3e-3, state_bits=8)
    obs, starts, answers = episodes(rng, T, B)
    arrays, block = bound_block(device, [("obs", obs), ("starts", starts), ("answers", answers.reshape(T * B, CUES))])
    inputs = {name: Tensor(a) for name, a in arrays.items()} | {"_block": block}

    def loss_of(x):
        rows, _ = policy(x["obs"], starts=x["starts"])
        logits, _value = split(rows, (CUES, 1), dim=-1)
        loss = mul(sum_all(mul(log_softmax(logits), x["answers"])), -4.0 / (T * B))
        loss.backward()
        return {"loss": loss}

    losses = []
    with TrainStep(loss_of, inputs, device, optimizer=optimizer, mode="graph") as step:
        for i in range(updates):
            if i:
                obs, starts, answers = episodes(rng, T, B)
                step.load_input("obs", obs)
                step.load_input("starts", starts)
                step.load_input("answers", answers.reshape(T * B, CUES))
            losses.append(float(np.ravel(step.run()["loss"])[0]))
            if log and (i % 50 == 0 or i + 1 == updates):
                log(f"update {i + 1}: loss {losses[-1]:.4f}", flush=True)

    obs, starts, answers = episodes(rng, T, B)
    with no_grad():
        whole = policy(Tensor.from_numpy(obs, device), starts=Tensor.from_numpy(starts, device))[0].numpy()
        states = policy.initial_states(B)
        acted = np.stack([policy.step(Tensor.from_numpy(obs[t], device), states, Tensor.from_numpy(starts[t], device)).numpy()
                          for t in range(T)])
    asked = answers.any(-1)
    right = acted[..., :CUES].argmax(-1)[asked] == answers.argmax(-1)[asked]
    result = {"losses": losses, "recalled": float(right.mean()),
              "difference": float(np.abs(acted.reshape(whole.shape) - whole).max()), "size": float(np.abs(whole).max())}
    if log:
        log(f"recalled {100 * result['recalled']:.1f} % of the cues acting token by token; rows differ from the whole "
            f"sequence's by {result['difference']:.1e} of {result['size']:.1f} at most", flush=True)
    return result


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--updates", type=int, default=300)
    args = parser.parse_args()
    from ttrl_amd.engine import open_device

    run(open_device(0), args.updates)
