"""optim.AdamW where it is used: the trainer (TrainConfig.optimizer = "adamw"), ranks that own different parameters, and the
whole set of operators together -- rows that die and come back, clipping, checkpoints, the moments' values."""
import os
import socket

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests import adamw_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _config(TRN, root, tag, iterations, **more):
    cfg = TRN.TrainConfig(
        train_dataset_json_path=os.path.join(root, "train.json"), val_dataset_json_path=os.path.join(root, "val.json"),
        pointcloud_parquet_path=os.path.join(root, "points.parquet"), num_iterations=iterations, val_interval=10 ** 6,
        feature_learning_rate=5e-3, position_learning_rate=5e-5, initial_downsample_factor=2,
        half_downsample_factor_interval=30, log_loss_interval=10, log_metrics_interval=10 ** 6, log_image_interval=10 ** 6,
        position_learning_rate_decay_interval=1, log_validation_image=False,
        summary_writer_log_dir=os.path.join(root, tag), num_data_loader_workers=0, **more)
    cfg.adaptive_controller_config.num_iterations_warm_up = 20
    cfg.adaptive_controller_config.num_iterations_densify = 20
    cfg.gaussian_point_cloud_scene_config.max_num_points_ratio = 3.0
    cfg.gaussian_point_cloud_scene_config.initial_alpha = 0.5
    return cfg


@pytest.mark.parametrize("bits,clip", [(32, 0.0), (8, 0.0), (8, 1e-4)])
def test_trainer_with_adamw(tmp_path, bits, clip):
    """Through two densifications: the live rows move and stay finite, the norm is there where it is asked for, the moments
    are held in the bits asked for, and the positions' rate (alone) decays."""
    from tests.test_training_gpu import _write_dataset
    from taichi_3d_gaussian_splatting_amd.GaussianPointTrainer import GaussianPointCloudTrainer as TRN
    root = str(tmp_path)
    _write_dataset(root, torch.device(DEV))
    cfg = _config(TRN, root, "logs", 51, optimizer="adamw", optimizer_state_bits=bits, weight_decay=1e-3, max_grad_norm=clip)
    cfg.to_yaml_file(os.path.join(root, "train.yaml"))
    trainer = TRN(TRN.TrainConfig.from_yaml_file(os.path.join(root, "train.yaml")))
    assert trainer.config.optimizer_state_bits == bits and trainer.config.max_grad_norm == clip
    made = []
    build = trainer._adamw
    trainer._adamw = lambda: made.append(build()) or made[0]
    first = trainer.scene.point_cloud_features.detach().clone()
    n_before = int((trainer.scene.point_invalid_mask == 0).sum())
    trainer.train()
    (optimizer,), _ = made[0]
    live = trainer.scene.point_invalid_mask == 0
    assert int(live.sum()) != n_before
    for p in (trainer.scene.point_cloud_features, trainer.scene.point_cloud):
        assert torch.isfinite(p.detach()[live]).all()
        state = optimizer.state[p]
        assert state["step"] == 51 and state["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
        m, v = optimizer.moments(p)
        assert torch.isfinite(m[live]).all() and (v[live] >= 0).all() and bool(v[live].any())
    assert not torch.equal(first, trainer.scene.point_cloud_features.detach())
    assert (optimizer.last_grad_norm is None) == (clip == 0.0)
    if clip:
        assert float(optimizer.last_grad_norm) > 0
    features, positions = optimizer.param_groups
    assert features["lr"] == 5e-3 and positions["lr"] == pytest.approx(5e-5 * 0.97 ** 51)


def test_first_step_of_the_trainer_is_the_same_with_either_optimiser(tmp_path):
    """Without decay, clipping and regulariser AdamW's first step is Adam's.  Each side is off by at most 12 units of 2^-24
    of the change (at most the rate: m / sqrt(v) is 1 at most there) and 3 of the parameter (adamw_plain.error_bounds)."""
    from tests.test_training_gpu import _write_dataset
    from taichi_3d_gaussian_splatting_amd.GaussianPointTrainer import GaussianPointCloudTrainer as TRN
    root = str(tmp_path)
    _write_dataset(root, torch.device(DEV))
    after = {}
    for name in ("adam", "adamw"):
        cfg = _config(TRN, root, name, 1, optimizer=name)
        cfg.loss_function_config.enable_regularization = False
        trainer = TRN(cfg)
        trainer.train()
        live = trainer.scene.point_invalid_mask == 0
        after[name] = [p.detach()[live].clone() for p in (trainer.scene.point_cloud_features, trainer.scene.point_cloud)]
    for a, b, rate in zip(after["adam"], after["adamw"], (5e-3, 5e-5)):
        assert ((a - b).abs() <= 2 * 2.0 ** -24 * (16 * rate + 3 * a.abs())).all()


def test_trainer_refuses_options_that_its_optimiser_does_not_take(tmp_path):
    from taichi_3d_gaussian_splatting_amd.GaussianPointTrainer import GaussianPointCloudTrainer as TRN
    for more in (dict(optimizer="sgd"), dict(optimizer_state_bits=8), dict(weight_decay=0.1), dict(max_grad_norm=1.0)):
        with pytest.raises(ValueError):
            TRN(_config(TRN, str(tmp_path), "logs", 1, **more))


def test_rows_die_and_come_back_through_clipped_steps_and_a_checkpoint():
    """The operators together, as a run uses them: a capacity whose rows are masked and revived with new parameters, clipped
    steps, the norm by itself, a checkpoint in the middle and the moments' values -- each step against 64 bits from the state
    before it (so rounding does not add up)."""
    from taichi_3d_gaussian_splatting_amd import optim
    gen = torch.Generator().manual_seed(4)
    n = 700
    mask = (torch.rand(n, generator=gen) < 0.5).to(torch.int8).to(DEV)
    params = [torch.nn.Parameter(torch.randn(n, w, generator=gen).to(DEV)) for w in (56, 3)]
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
    opt = optim.AdamW(params, state_bits=8, max_grad_norm=0.3, seed=11, **hyper)
    for p in params:
        opt.set_row_mask(p, mask)
    for t in range(1, 13):
        live = (mask == 0).cpu().numpy()
        for p in params:
            p.grad = (torch.randn(p.shape, generator=gen) * 10.0 ** (t % 3 - 2)).to(DEV)
            p.grad[mask != 0] = float("nan")
        before = []
        for p in params:
            state = opt.state.get(p)
            moments = [x.double().cpu().numpy() for x in opt.moments(p)] if state else [np.zeros(p.shape)] * 2
            stamps = state["last_step"].cpu().numpy() if state else np.zeros(n, int)
            before.append((p.detach().double().cpu().numpy(), p.grad.double().cpu().numpy(), *moments, stamps))
        norm = optim.grad_norm([p.grad for p in params], [mask, mask])
        opt.step()
        assert torch.equal(norm, opt.last_grad_norm)
        total = np.sqrt(sum((b[1][live] ** 2).sum() for b in before))
        assert abs(float(norm) - total) <= 2.0 ** -23 * total
        for p, (p0, g, m0, v0, stamps) in zip(params, before):
            want, m, v = plain.update(p0, np.where(live[:, None], g, 0), m0, v0, step=t, scale=min(1.0, 0.3 / (total + 1e-6)),
                                      missed=t - 1 - stamps, **hyper)
            ep, _, _ = plain.error_bounds(p0, want, np.where(live[:, None], g, 0), m0, m, v, step=t, **hyper)
            got = p.detach().double().cpu().numpy()
            assert (np.abs(got - want) <= ep)[live].all() and np.array_equal(got[~live], p0[~live])
            values = [x.double().cpu().numpy() for x in opt.moments(p)]
            for x, y, floor in ((values[0], m, 2.0 ** -17), (values[1], v, 2.0 ** -30)):
                # a code is within one step of the value: an eighth of it, or the smallest code's size
                top = np.abs(y).max(1, keepdims=True)
                assert (np.abs(x - y) <= np.abs(y) / 8 * 1.001 + floor * top)[live].all()
            assert np.array_equal(opt.state[p]["last_step"].cpu().numpy(), np.where(live, t, stamps))
        if t % 4 == 0:
            die = (torch.rand(n, generator=gen) < 0.2).to(DEV) & (mask == 0)
            back = (torch.rand(n, generator=gen) < 0.3).to(DEV) & (mask != 0)
            mask[die] = 1
            mask[back] = 0
            with torch.no_grad():
                for p in params:
                    p[back] = torch.randn(int(back.sum()), p.shape[1], generator=gen).to(DEV)
        if t == 6:
            saved = opt.state_dict()
            opt = optim.AdamW(params, state_bits=8, max_grad_norm=0.3, seed=11, **hyper)
            for p in params:
                opt.set_row_mask(p, mask)
            opt.load_state_dict(saved)


def _norm_group_worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY="0")
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from taichi_3d_gaussian_splatting_amd import optim
        gen = torch.Generator().manual_seed(8)
        whole = [torch.randn(600, 56, generator=gen), torch.randn(600, 3, generator=gen)]
        grads = [[torch.randn(600, 56, generator=gen), torch.randn(600, 3, generator=gen)] for _ in range(4)]
        rows = slice(0, 250) if rank == 0 else slice(250, 600)
        mine = [torch.nn.Parameter(x[rows].clone().to(DEV)) for x in whole]
        alone = [torch.nn.Parameter(x.clone().to(DEV)) for x in whole]
        a = optim.AdamW(mine, max_grad_norm=2.0, norm_group=dist.group.WORLD)
        b = optim.AdamW(alone, max_grad_norm=2.0)
        for it, g in enumerate(grads):
            # in the last step the second rank has no gradient: it takes part in the norm all the same
            gone = it == 3 and rank == 1
            for p, x in zip(mine, g):
                p.grad = None if gone else x[rows].to(DEV)
            for p, x in zip(alone, g):
                x = x.clone()
                if it == 3:
                    x[250:] = 0
                p.grad = x.to(DEV)
            a.step()
            b.step()
            total = float(b.last_grad_norm)
            assert abs(float(a.last_grad_norm) - total) <= 2.0 ** -23 * total, (it, float(a.last_grad_norm), total)
            if it < 3:
                # (the two coefficients are one unit in the last place apart at most: 2^-23 of a step of lr at most)
                for p, q in zip(mine, alone):
                    assert ((p - q[rows]).abs() <= 1e-3 * 2.0 ** -20 + 2.0 ** -23 * q[rows].abs()).all(), it
    finally:
        dist.destroy_process_group()


def test_clipping_by_the_norm_of_all_ranks(tmp_path):
    mp.spawn(_norm_group_worker, args=(2, _free_port(), str(tmp_path)), nprocs=2, join=True)


def _owner_worker(rank, world, port, root):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), HSA_ENABLE_IPC_MODE_LEGACY="0")
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from taichi_3d_gaussian_splatting_amd.GaussianPointTrainer import GaussianPointCloudTrainer as TRN
        cfg = _config(TRN, root, f"owner{rank}", 25, optimizer="adamw", optimizer_state_bits=8, max_grad_norm=1e-3,
                      distributed_mode="owner")
        trainer = TRN(cfg)
        made = []
        build = trainer._adamw
        trainer._adamw = lambda: made.append(build()) or made[0]
        trainer.train()
        (optimizer,), _ = made[0]
        norms = [None, None]
        dist.all_gather_object(norms, float(optimizer.last_grad_norm))
        assert norms[0] == norms[1] and norms[0] > 0
        live = trainer.scene.point_invalid_mask == 0
        assert torch.isfinite(trainer.scene.point_cloud_features.detach()[live]).all()
    finally:
        dist.destroy_process_group()


def test_trainer_with_adamw_and_owner_sharded_gaussians(tmp_path):
    from tests.test_training_gpu import _write_dataset
    root = str(tmp_path)
    _write_dataset(root, torch.device(DEV))
    mp.spawn(_owner_worker, args=(2, _free_port(), root), nprocs=2, join=True)
