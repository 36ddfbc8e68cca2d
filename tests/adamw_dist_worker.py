"""One rank of a short AdamW training session (gloo, CPU) for test_adamw.py:
writes its parameters and states to the path it is given."""

import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from aggregathor_amd import experiments
from aggregathor_amd.graph import Engine
from aggregathor_amd.parallel import WorkerGroup


def main():
    exp = experiments.instantiate("mnist", ["batch-size:16"])
    eng = Engine(exp, "krum", WorkerGroup(4, device="cpu"), nbbyzwrks=1,
                 optimizer="adamw",
                 optimizer_args=["clip-norm:0.5"] + sys.argv[2:])
    for _ in range(4):
        eng.step()
    torch.save([[p.detach()] + [v.float() for _, v in sorted(
        eng.optimizer.state[p].items())] for p in eng.params], sys.argv[1])


if __name__ == "__main__":
    main()
