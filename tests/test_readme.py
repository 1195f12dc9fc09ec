"""What the README shows runs."""
import os
import re
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def blocks():
    with open(os.path.join(ROOT, "README.md")) as f:
        return re.findall(r"```python\n(.*?)```", f.read(), re.S)


def test_the_package_has_what_the_readme_reaches_through_it():
    code = "import difflogic_b200 as difflogic\n" + "\n".join(sorted(set(re.findall(r"difflogic(?:\.\w+)+", "\n".join(blocks())))))
    assert "difflogic.optim.FlatMuon" in code and "difflogic.training.TrainStep" in code
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


@pytest.mark.gpu
def test_the_readmes_examples_run():
    torch.manual_seed(0)
    names = dict(x=torch.rand(100, 784, device="cuda"), y=torch.randint(0, 10, (100,), device="cuda"), weight=torch.randn(50, 784, device="cuda"),
                 bias=torch.randn(50, device="cuda"), residual=torch.randn(100, 50, device="cuda"), g=torch.randn(40, 60, device="cuda"))
    names.update(weights=[torch.randn(40, 60, device="cuda")], grads=[torch.randn(40, 60, device="cuda")], momenta=[torch.zeros(40, 60, device="cuda")])
    x, y = names["x"], names["y"]
    for block in blocks():
        exec(block, names)
    assert names["y"].shape == (100, 50) and names["o"].shape == (40, 60)
    model, step = names["model"], names["step"]
    before = [p.detach().clone() for p in model.parameters()]
    assert bool(torch.isfinite(step(x, y)))
    assert all(not torch.equal(p, q) for p, q in zip(before, model.parameters()))
    step.close()
