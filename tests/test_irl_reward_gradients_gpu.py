"""GPU: gradients of the reward network on a 256 x 256 MDP grid against the oracle in 64 bits, wherever its ReLUs' inputs lie.

Ten million ReLU inputs and pooling windows of one step hold some within fp32's rounding of the edge, and on which side of it an
implementation finds them is not defined to fp32; each moves the gradients by up to some percent.  So the 64-bit network takes the sides
that the HIP forward took: they may differ from its own only where an input lies at the edge, and with them every gradient has to
agree."""
import copy

import numpy as np
import pytest
import torch

from creste_public_amd import synth, train_ops
from creste_public_amd.config import maxent_irl_cfg
from tests.test_model_gpu import _irl_step, _rms, _with_eval_backbone, calibrate_bn

pytestmark = pytest.mark.gpu


class _Relu(torch.nn.Module):
    """ReLU with the sides of `y`, another forward's output.  far: how far the two differ where both are positive, at most; off_by: how far
    from the edge an input lies whose sides differ; top: the largest output"""

    def __init__(self, y):
        super().__init__()
        self.y = y.double()

    def forward(self, x):
        on, mine = self.y > 0, x.detach() > 0
        self.far = float(((self.y - x.detach()).abs() * (on & mine)).max())
        self.off_by = float((x.detach().abs() * (on != mine)).max())
        self.top = float(x.detach().max())
        return torch.where(on, x, torch.zeros_like(x))


class _Pool(torch.nn.Module):
    """2 x 2 maximum with a given element of each window; off_by: how much larger another one is"""

    def __init__(self, idx):
        super().__init__()
        self.idx = idx

    def forward(self, x):
        B, Cn, H, W = x.shape
        win = x.view(B, Cn, H // 2, 2, W // 2, 2).permute(0, 1, 2, 4, 3, 5).reshape(B, Cn, H // 2, W // 2, 4)
        y = win.gather(4, self.idx[..., None])[..., 0]
        self.off_by = float((win.detach().amax(4) - y.detach()).max())
        return y


def _with_sides_of(net, engine):
    """replace the ReLUs and pools of `net` by ones that decide as the engine's latest forward did -> the replacements"""
    new = []
    for name in ("prepool", "trunk", "skip", "postpool"):
        sides = []
        for op in getattr(engine, name).ops:
            if isinstance(op, train_ops.ReLUT) or (isinstance(op, train_ops.BNT) and op.relu):
                sides.append(_Relu(op.y.nchw()))
            elif isinstance(op, train_ops.PoolT):
                sides.append(_Pool(op.idx.permute(0, 3, 1, 2).long()))
        new += sides
        branch = getattr(net, name)
        for at in [n for n, m in branch.named_modules() if isinstance(m, (torch.nn.ReLU, torch.nn.MaxPool2d))]:
            above, _, child = at.rpartition(".")
            setattr(branch.get_submodule(above), child, sides.pop(0))
        assert not sides
    return new


def _gradients(net, lm, out, dev, dtype, expert, fov, cf):
    net.train()
    net.zero_grad()
    iv = out["input_view"].detach().to(dev, dtype).requires_grad_(True)
    r = net(iv)
    td = {"outputs/exp_svf": out["exp_svf"].to(dev, dtype), "outputs/traversability_preds": r, "outputs/input_view": iv,
          "inputs/traversability_label": expert.to(dev), "inputs/fov_mask": fov.to(dev), "inputs/counterfactuals_label": cf, "task": "irl"}
    ld, _ = lm(td)
    sum(w * v for w, v in ld.values()).backward()
    return {n: p.grad.detach().double().cpu() for n, p in net.named_parameters()}


@pytest.fixture(scope="module")
def step():
    """the oracle and its outputs for one step"""
    from oracle import irl as oirl
    Hh, Ww, Bb = 128, 192, 2
    kw = dict(map_size=(256, 256), map_ds=1, point_cloud_range=[-25.6, -12.8, -2, 25.6, 12.8, 1])
    bev = (512, 256)
    cfg = maxent_irl_cfg((Hh, Ww), solve_mdp=True, **kw)
    torch.manual_seed(77)
    oracle = oirl.MaxEntIRL(cfg)
    rgbd, p2p = synth.make_frames(Bb, Hh, Ww, seed=12)
    expert = synth.make_experts(Bb, 50, bev, seed=4)
    calibrate_bn(oracle, lambda: oracle((rgbd, p2p, expert)))
    with torch.no_grad():
        oracle.traversability_head.r.postpool[0].norm.weight.mul_(0.01)
        oracle.traversability_head.r.postpool[0].norm.bias.mul_(0.01)
    oracle = _with_eval_backbone(oracle)
    fov = torch.ones(Bb, max(bev[0], 512), max(bev[1], 512), dtype=torch.bool)
    rng = np.random.RandomState(1)
    c0 = np.array([[bev[0] / 2 - 28.0, bev[1] / 2.0]])
    cf = [dict(trajectories=(c0 + np.linspace(0, 1, 20)[None, :, None] *
                             rng.uniform(-0.3 * bev[1], 0.3 * bev[1], size=(3, 1, 2))).astype(np.float32),
               rank=np.array([0, 1, 2])), None]
    _, _, _, out, _ = _irl_step(copy.deepcopy(oracle), oirl.LossManager(cfg), "cpu", (rgbd, p2p, expert), cf, fov)
    return dict(cfg=cfg, kw=kw, size=(Hh, Ww), oracle=oracle, lm=oirl.LossManager(cfg), data=(expert, fov, cf), out=out)


@pytest.mark.parametrize("prec", ["f32", "f16x3", "bf16x6"])
def test_reward_gradients_with_the_sides_of_the_forward(step, prec):
    import creste_public_amd
    from creste_public_amd import LossManager, MaxEntIRL
    creste_public_amd.set_precision(prec)
    try:
        model = MaxEntIRL(maxent_irl_cfg(step["size"], solve_mdp=True, **step["kw"]))
        model.load_state_dict(step["oracle"].state_dict(), strict=True)
        net = model.cuda().traversability_head.r
        got = _gradients(net, LossManager(step["cfg"]).cuda(), step["out"], "cuda", torch.float32, *step["data"])
    finally:
        creste_public_amd.set_precision("f32")
    ref_net = copy.deepcopy(step["oracle"].traversability_head.r).cuda().double()
    sided = _with_sides_of(ref_net, net._train_engine)
    ref = _gradients(ref_net, step["lm"], step["out"], "cuda", torch.float64, *step["data"])
    far = 0.0
    for s in sided:                            # sides differ only as close to the edge as the forwards do elsewhere in the layer
        if isinstance(s, _Relu):
            far = s.far
            assert far <= 1e-4 * s.top         # (fp32 sums of up to 1000 products; some channels scaled up by their BatchNorm)
            assert s.off_by <= far
        else:
            assert s.off_by <= 2 * far
    assert far and set(got) == set(ref)
    for n in ref:
        assert _rms(got[n] - ref[n]) <= 2e-3 * max(_rms(ref[n]), 1e-8) + 1e-9, n
