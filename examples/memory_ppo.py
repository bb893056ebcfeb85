"""Trains a policy with memory for a few iterations on the synthetic image:

    python examples/memory_ppo.py --envs 256 --steps 64 --iterations 3
"""
import argparse
import importlib.util
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAME = "fast_mario_env_b200"


def load():
    """The package; its directory name has hyphens, so it is loaded by path."""
    if NAME not in sys.modules:
        d = os.path.join(ROOT, "fast-mario-env_b200")
        spec = importlib.util.spec_from_file_location(NAME, os.path.join(d, "__init__.py"), submodule_search_locations=[d])
        sys.modules[NAME] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[NAME])
    return sys.modules[NAME]


def main(argv=None):
    p = argparse.ArgumentParser()
    p.add_argument("--envs", type=int, default=256)
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--iterations", type=int, default=3)
    p.add_argument("--minibatch-envs", type=int, default=64)
    a = p.parse_args(argv)
    fme = load()
    from fast_mario_env_b200 import memory, ppo
    from fast_mario_env_b200.synth_rom import build_rom
    dev = torch.device("cuda", torch.cuda.current_device())
    env = fme.CudaVecEnv("1-1", a.envs, device=dev, rom=build_rom(0), seed=0, sticky=0.25, noop_max=30, maxpool=True, max_steps=2000)
    cfg = ppo.PPOConfig(n_envs=a.envs, n_steps=a.steps, batch=a.minibatch_envs * a.steps, epochs=2, graph=False)
    trainer = memory.MemoryTrainer(env, cfg, dev)
    history = []
    for i in range(a.iterations):
        t = time.perf_counter()
        stats = trainer.iterate()
        history.append(stats)
        print(f"iteration {i}: {a.envs * a.steps / (time.perf_counter() - t):.0f} samples/s, " + ", ".join(f"{k} {v:.4f}" for k, v in stats.items()))
    env.check()
    return history


if __name__ == "__main__":
    main()
