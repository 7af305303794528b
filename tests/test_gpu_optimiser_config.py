"""The runners train with the optimiser that the configuration names."""
import os

import pytest
import torch
import yaml

from gncde import run, train

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name,clip", [("sgd", True), ("sgd", False), ("adam", True)])
def test_update_is_the_named_optimisers(name, clip):
    """One step from known gradients: sgd moves by lr g, adam's first step is lr g / (|g| + 1e-8); both of the clipped g.
    Rounded in fp32: the clip's factor and product (8 u), the step's two or three operations, the parameter's half step."""
    m = torch.nn.Linear(20, 30).to("cuda")
    before = [p.detach().clone() for p in m.parameters()]
    opt = run._build_optimiser({"optimiser": {"name": name, "gradient_clipping": clip, "schedule": {"value": "1e-1"}}}, m)
    assert isinstance(opt, train.ClippedOptimiser) and opt.max_norm == (1.0 if clip else None)
    g = torch.Generator(device="cuda").manual_seed(0)
    gs = [torch.randn(p.shape, generator=g, device="cuda") for p in m.parameters()]
    train.make_step(opt, lambda: (sum((p * w).sum() for p, w in zip(m.parameters(), gs)), 1))
    n = torch.sqrt(sum((w.double() ** 2).sum() for w in gs)) if clip else 1.0
    for p, z, w in zip(m.parameters(), before, gs):
        d = w.double() / n
        step = 0.1 * (d if name == "sgd" else d / (d.abs() + 1e-8))
        want = z.double() - step
        assert bool(((p.detach().double() - want).abs() <= 32 * 2.0 ** -24 * (step.abs() + z.double().abs() + 0.1)).all())


@pytest.mark.parametrize("config,name,readout", [("heat_grid_small.yaml", "sgd", None), ("tgb_trade_small.yaml", "adam", "fused")])
def test_runner_trains_with_it(tmp_path, config, name, readout, monkeypatch):
    with open(os.path.join(ROOT, "configs", config)) as fh:
        cfg = yaml.safe_load(fh)
    cfg["optimiser"].update(name=name, weight_decay=0.0)
    cfg.update(checkpoint_dir=str(tmp_path), eval_freq=1, log_freq=1)
    steps = []
    real = train.ClippedOptimiser.step
    monkeypatch.setattr(train.ClippedOptimiser, "step", lambda self, *a: steps.append(type(self.optimiser)) or real(self, *a))
    if readout:
        cfg["dataset"]["num_snapshots"] = 16
        cfg["model"]["readout_loss"] = readout
        res = run.WindowTrainer(cfg, epochs=2).run()
    else:
        cfg["dataset"].update(num_nodes=16, time_tick=16, batch_size=3)
        res = run.Trainer(cfg, epochs=2, steps_per_interval=1).run()
    assert os.path.exists(res["checkpoint"])
    assert steps and set(steps) == {{"sgd": torch.optim.SGD, "adam": torch.optim.Adam}[name]}
