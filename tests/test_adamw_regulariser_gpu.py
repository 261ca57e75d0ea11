"""The scale regulariser in the trainer's AdamW path: its gradient is added to the features' before the norm and the step, over one rank
or over owners of different points."""
import os
import socket
from types import SimpleNamespace

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

pytestmark = pytest.mark.gpu
DEV, WEIGHT = "cuda:0", 2.0


def _scene(seed=7, n=5003):
    gen = torch.Generator().manual_seed(seed)
    features = torch.randn(n, 56, generator=gen)
    features[:, 4:7] = features[:, 4:7] * 1.5 - 2
    mask = (torch.rand(n, generator=gen) < 0.3).to(torch.int8)
    return features, mask, torch.randn(n, 56, generator=gen) * 1e-3


def _trainer(features, mask, owner_sharded=False):
    from taichi_3d_gaussian_splatting_amd.GaussianPointTrainer import GaussianPointCloudTrainer as TRN
    trainer = TRN.__new__(TRN)
    trainer.scene = SimpleNamespace(point_cloud_features=torch.nn.Parameter(features.to(DEV)), point_invalid_mask=mask.to(DEV))
    trainer.loss_function = SimpleNamespace(config=SimpleNamespace(regularization_weight=WEIGHT))
    trainer.adaptive_controller = SimpleNamespace(mask_version=0)
    trainer.owner_sharded = owner_sharded
    return trainer


def _formula(features, mask):
    """Gradient of WEIGHT * mean over live rows of ||exp(s)||, s = columns 4..6, in 64 bits."""
    s = features[:, 4:7].double().requires_grad_(True)
    live = mask == 0
    (WEIGHT * s[live].exp().norm(dim=1).mean()).backward()
    whole = torch.zeros(features.shape, dtype=torch.float64)
    whole[:, 4:7] = s.grad
    return whole


def _bound(reg, total):
    """exp(s) of |s| <= 8: 8 u of its argument's rounding and 2 of its own; squared, summed, rooted, divided and scaled: 32 u in all;
    the sum with the gradient 1 u."""
    u = 2.0 ** -24
    return 32 * u * reg.abs() + u * total.abs() * 1.001 + 1e-38


@pytest.mark.parametrize("given", [True, False])
def test_gradient_is_the_formulas(given):
    features, mask, grad = _scene()
    trainer = _trainer(features, mask)
    if given:
        trainer.scene.point_cloud_features.grad = grad.to(DEV)
    trainer._add_regulariser_gradient()
    reg = _formula(features, mask)
    want = reg + (grad.double() if given else 0)
    off = (trainer.scene.point_cloud_features.grad.double().cpu() - want).abs()
    assert (off <= _bound(reg, want)).all(), float((off - _bound(reg, want)).max())
    assert (reg[mask == 0][:, 4:7] > 0).all()


def test_step_takes_the_gradient_that_the_fused_adam_takes():
    """Both optimisers' first moments after a step: a tenth of the same gradient, each within two roundings more."""
    from taichi_3d_gaussian_splatting_amd.optim import Adam, AdamW
    features, mask, grad = _scene()
    trainer = _trainer(features, mask)
    p, invalid = trainer.scene.point_cloud_features, trainer.scene.point_invalid_mask
    q = torch.nn.Parameter(features.to(DEV))
    a, b = AdamW([p], lr=1e-3, weight_decay=0.0), Adam([q], lr=1e-3)
    for opt, x in ((a, p), (b, q)):
        opt.set_row_mask(x, invalid)
        x.grad = grad.to(DEV)
    b.set_scale_regulariser(q, WEIGHT, invalid)
    trainer._add_regulariser_gradient()
    a.step()
    b.step()
    reg = _formula(features, mask)
    want = torch.where((mask == 0)[:, None], 0.1 * (reg + grad.double()), 0.0)
    bound = 0.1 * _bound(reg, reg + grad.double()) + 3 * 2.0 ** -24 * want.abs()
    for opt, x in ((a, p), (b, q)):
        assert ((opt.state[x]["exp_avg"].double().cpu() - want).abs() <= bound).all()


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _owner(rank, world, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY="0")
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        features, mask, grad = _scene()
        mask[:1700] = (torch.arange(1700) % 3 > 0).to(torch.int8)       # (blocks of different sizes and live shares)
        rows = slice(0, 1700) if rank == 0 else slice(1700, len(mask))
        trainer = _trainer(features[rows].clone(), mask[rows].clone(), owner_sharded=True)
        if rank == 0:                                                   # (the other one has seen no point)
            trainer.scene.point_cloud_features.grad = grad[rows].to(DEV)
        trainer._add_regulariser_gradient()
        reg = _formula(features, mask)[rows]
        want = reg + (grad[rows].double() if rank == 0 else 0)
        off = (trainer.scene.point_cloud_features.grad.double().cpu() - want).abs()
        # (the share of live rows is a double, its product with the weight rounded once more)
        assert (off <= _bound(reg, want) + 2.0 ** -23 * reg.abs()).all()
    finally:
        dist.destroy_process_group()


def test_gradient_over_owners_is_that_of_all_live_points():
    mp.spawn(_owner, args=(2, _free_port()), nprocs=2, join=True)


@pytest.mark.parametrize("backend", ["gloo", "nccl"])
def test_live_share_hands_device_memory_to_back_ends_that_take_it(monkeypatch, backend):
    """(a sum over two ranks that hold the same: doubled)"""
    features, mask, _ = _scene()
    trainer = _trainer(features, mask, owner_sharded=True)
    handed = []

    def all_reduce(value, *args, **kwargs):
        handed.append(value.device.type)
        value *= 2
    monkeypatch.setattr(dist, "get_backend", lambda group=None: backend)
    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    assert trainer._local_live_share() == 0.5
    assert handed == ["cpu" if backend == "gloo" else "cuda"]
    assert trainer._local_live_share() == 0.5 and len(handed) == 1      # (kept while the live set stays)
