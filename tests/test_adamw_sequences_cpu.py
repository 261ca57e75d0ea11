"""Sequences of calls of optim.AdamW that need no device: states that are loaded, masks that come and go, hooks.  The step itself
is replaced by the plain one in 64 bits (adamw_plain.py); what it is handed is what is tested."""
import ctypes

import numpy as np
import pytest
import torch

from taichi_3d_gaussian_splatting_amd import _lib, optim
from tests import adamw_plain as plain
from tests.test_adamw_cpu import _step

HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _plain_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas, eps, weight_decay, exponents=None, masters=None, row_masks=None,
                last_steps=None, grad_scale=None, seed=0, tensor_ids=None):
    """adamw_step_ for float32 host tensors with moments in 32 bits."""
    for i, p in enumerate(params):
        mask = None if row_masks is None else row_masks[i]
        missed = None if mask is None else step[i] - 1 - last_steps[i].numpy()
        state = [t.detach().double().numpy() for t in (p, grads[i], exp_avgs[i], exp_avg_sqs[i])]
        new = plain.update(*state, step=step[i], lr=lr[i], betas=betas, eps=eps, weight_decay=weight_decay[i], missed=missed)
        for t, value in zip((p, exp_avgs[i], exp_avg_sqs[i]), new):
            value = torch.from_numpy(value).float()
            t.copy_(value if mask is None else torch.where(mask[:, None] == 0, value, t))
        if mask is not None:
            last_steps[i].copy_(torch.where(mask == 0, torch.full_like(last_steps[i], step[i]), last_steps[i]))


@pytest.fixture
def host_steps(monkeypatch):
    """AdamW on host tensors: the plain step in the kernels' place."""
    monkeypatch.setattr(optim, "adamw_step_", _plain_step)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _masked_state(shape, step, stamps, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return {"state": {0: dict(step=step, exp_avg=torch.randn(shape, generator=gen), exp_avg_sq=torch.rand(shape, generator=gen),
                              last_step=torch.as_tensor(stamps, dtype=torch.int32))},
            "param_groups": [dict(params=[0], state_bits=32, **HYPER)]}


def test_stamps_of_rows_do_not_outlive_steps_without_a_mask(host_steps):
    """A state saved under a row mask goes on without one, and under one again: late rows are decayed by the first step that
    reaches them, and the steps without the mask owe no decay."""
    shape, stamps = (4, 3), [100, 97, 100, 60]
    p = torch.nn.Parameter(torch.ones(shape))
    opt = optim.AdamW([p], **HYPER)
    saved = _masked_state(shape, 100, stamps)
    opt.load_state_dict(saved)
    want = [np.ones(shape), *(saved["state"][0][k].double().numpy() for k in ("exp_avg", "exp_avg_sq"))]
    missed = 100 - np.array(stamps)
    gen = torch.Generator().manual_seed(1)
    for t in range(101, 113):
        if t == 106:
            opt.set_row_mask(p, torch.zeros(4, dtype=torch.int8))
        p.grad = torch.randn(shape, generator=gen)
        opt.step()
        want = plain.update(want[0], p.grad.double().numpy(), want[1], want[2], step=t, missed=missed, **HYPER)
        missed = None
        state = opt.state[p]
        # the host's step rounds each value to float32 once a step: t steps of half a spacing
        for got, value in zip((p.detach(), state["exp_avg"], state["exp_avg_sq"]), want):
            assert np.allclose(got.numpy(), value, rtol=20 * 2.0 ** -24, atol=20 * 2.0 ** -24), t
    assert (opt.state[p]["last_step"] == 112).all()


def test_stamps_are_not_taken_for_parameters_that_cannot_have_them():
    for p in (torch.zeros(4, 3, dtype=torch.bfloat16), torch.zeros(4, 65)):
        opt = optim.AdamW([torch.nn.Parameter(p)], master_weights=False, **HYPER)
        with pytest.raises(ValueError, match="last_step"):
            opt.load_state_dict(_masked_state(tuple(p.shape), 5, [5, 5, 3, 5]))


def _plain_state(shape=(4, 3), step=7, seed=0):
    saved = _masked_state(shape, step, [step] * shape[0], seed)
    del saved["state"][0]["last_step"]
    return saved


def test_hooks_of_load_state_dict_see_and_change_what_is_loaded():
    """As in torch: a hook before the load may return another state_dict, one behind it finds the loaded state and groups."""
    seen = []
    for kind in (torch.optim.AdamW, optim.AdamW):
        opt = kind([torch.nn.Parameter(torch.zeros(4, 3))], **HYPER)
        saved = _plain_state()
        kept = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in saved["state"][0].items()}

        def before(optimizer, state_dict):
            state = dict(state_dict["state"][0], step=77, exp_avg=state_dict["state"][0]["exp_avg"] + 1)
            return {"state": {0: state}, "param_groups": [dict(state_dict["param_groups"][0], lr=0.5)]}

        def after(optimizer):
            (state,) = optimizer.state.values()
            seen.append((int(state["step"]), optimizer.param_groups[0]["lr"], state["exp_avg"].clone(), "state_bits" in optimizer.param_groups[0]))
        handles = [opt.register_load_state_dict_pre_hook(before), opt.register_load_state_dict_post_hook(after)]
        opt.load_state_dict(saved)
        for name, value in kept.items():
            assert torch.equal(saved["state"][0][name], value) if isinstance(value, torch.Tensor) else saved["state"][0][name] == value
        for handle in handles:
            handle.remove()
        opt.load_state_dict(saved)
        (state,) = opt.state.values()
        assert int(state["step"]) == 7
        assert not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks
    assert [s[:2] for s in seen] == [(77, 0.5)] * 2 and torch.equal(seen[0][2], seen[1][2]) and seen[1][3]


def test_a_refused_state_dict_changes_nothing_and_leaves_no_hook():
    opt = optim.AdamW([torch.nn.Parameter(torch.zeros(4, 3))], **HYPER)
    opt.load_state_dict(_plain_state())
    (before,) = (dict(s) for s in opt.state.values())
    wrong_shape, two_groups = _plain_state(step=9), _plain_state(step=9)
    wrong_shape["state"][0]["exp_avg"] = torch.zeros(5, 3)
    two_groups["param_groups"] *= 2
    other_size = _plain_state(step=9)
    other_size["param_groups"] = [dict(other_size["param_groups"][0], params=[0, 1])]
    amsgrad = _plain_state(step=9)
    amsgrad["param_groups"][0]["amsgrad"] = True
    for bad in (wrong_shape, two_groups, other_size, amsgrad):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        (state,) = opt.state.values()
        assert state.keys() == before.keys() and all(state[k] is before[k] for k in before)
        assert not opt._optimizer_load_state_dict_pre_hooks


def test_options_that_a_saved_group_does_not_name_stay_the_groups_own(host_steps):
    """A state_dict of optim.Adam has no weight decay: the step takes the group's."""
    p = torch.nn.Parameter(torch.ones(4, 3))
    adam = optim.Adam([p], lr=2e-3)
    saved = {"state": _plain_state()["state"], "param_groups": adam.state_dict()["param_groups"]}
    opt = optim.AdamW([dict(params=[p], weight_decay=0.3)], lr=1e-3)
    opt.load_state_dict(saved)
    assert "weight_decay" not in saved["param_groups"][0]
    assert opt.param_groups[0]["lr"] == 2e-3 and opt.param_groups[0]["weight_decay"] == 0.3 and opt.param_groups[0]["state_bits"] == 32
    p.grad = torch.zeros(4, 3)
    m, v = (saved["state"][0][k].double().numpy() for k in ("exp_avg", "exp_avg_sq"))
    want = plain.update(np.ones((4, 3)), np.zeros((4, 3)), m, v, step=8, **{**HYPER, "lr": 2e-3, "weight_decay": 0.3})[0]
    opt.step()
    assert np.allclose(p.detach().numpy(), want, rtol=4 * 2.0 ** -24, atol=0)
    # groups without a state keep the form that they were made with
    opt = optim.AdamW([dict(params=[p], state_bits=8)], lr=1e-3)
    opt.load_state_dict({"state": {}, "param_groups": torch.optim.AdamW([p]).state_dict()["param_groups"]})
    assert opt.param_groups[0]["state_bits"] == 8


# Elements of the largest launch: gridDim.x * blockDim.x has to stay below 2^32, so 2^24 - 1 workgroups of 256 lanes, times what
# a workgroup takes of each form
WORKGROUPS = (1 << 24) - 1
LARGEST = [(dict(), 1024), (dict(dtype=1), 1024), (dict(dtype=2, master=1 << 47), 1024), (dict(x=1 << 46), 4096), (dict(x=1 << 46, dtype=1), 4096),
           (dict(x=1 << 46, dtype=1, row=56), 64 * 56), (dict(x=1 << 46, row=17), 128 * 17), (dict(x=1 << 46, row=2), 1024 * 2),
           (dict(mask=1 << 46, last=1 << 47, row=56), 64 * 56), (dict(mask=1 << 46, last=1 << 47, row=1), 1024)]


@pytest.mark.parametrize("change,share", LARGEST)
def test_a_step_that_no_launch_holds_is_refused(change, share):
    """At the limit the size is taken (what is said then is that these made-up buffers overlap), one row or element over it not."""
    row = change.get("row", 1)
    status, message = _step(numel=WORKGROUPS * share // row * row + row, **change)
    assert status == -1 and "too large" in message, message
    status, message = _step(numel=WORKGROUPS * share // row * row, **change)
    assert status == -1 and "overlap" in message, message


@pytest.mark.parametrize("dtype,row,share", [(0, 0, 4096), (1, 0, 4096), (1, 56, 64 * 56), (0, 56, 64 * 56), (0, 17, 128 * 17), (0, 3, 4096)])
def test_a_reading_of_moments_that_no_launch_holds_is_refused(dtype, row, share):
    lib = _lib.load()
    for rows_more, says in ((1, "too large"), (0, "overlaps")):
        n = WORKGROUPS * share // max(row, 1) * max(row, 1) + rows_more * max(row, 1)
        columns = [(ctypes.c_uint64 * 1)(0x10000 * (i + 1)) for i in range(5)]
        status = lib.gs_read_moments(1, *columns, (ctypes.c_int64 * 1)(n), (ctypes.c_int32 * 1)(row), dtype, None)
        assert status == -1 and says in lib.gs_last_error().decode(), lib.gs_last_error()


@pytest.mark.parametrize("change", [dict(step_dev=0x10010, ws=0x90000), dict(lr_dev=0x30000, ws=0x90000), dict(step_dev=0x40000 - 4, ws=0x90000),
                                    dict(lr_dev=0x50000, x=0x50000, ws=0x90000)])
def test_device_scalars_inside_written_buffers_are_refused(change):
    """The kernels read them while they write there."""
    status, message = _step(**change)
    assert status == -1 and "overlap" in message, message


def test_a_gradient_scale_inside_a_written_buffer_is_refused():
    u64 = ctypes.c_uint64
    lib = _lib.load()
    columns = [(u64 * 1)(x) for x in (0x10000, 0x20000, 0x30000, 0x40000)]
    for scale in (0x10000, 0x30000 + 4 * 63, 0x40010):
        status = lib.gs_adamw_step(1, *columns, None, None, None, None, (ctypes.c_int64 * 1)(64), (ctypes.c_int32 * 1)(0), (ctypes.c_int32 * 1)(0),
                                   (ctypes.c_int32 * 1)(0), (ctypes.c_double * 5)(1e-3, 0.9, 0.999, 1e-8, 0.0), (ctypes.c_int64 * 1)(1), None, None,
                                   scale, 0, None, None)
        assert status == -1 and "overlap" in lib.gs_last_error().decode(), (hex(scale), lib.gs_last_error())


def test_whether_a_graph_is_captured_is_asked_on_the_parameters_device(monkeypatch):
    """A step with a number for its count, of tensors on another device than the current one, whose stream is being captured."""
    import contextlib
    entered = []

    @contextlib.contextmanager
    def on(index):
        entered.append(index)
        yield
        entered.pop()

    class Host:
        PARAM = GRAD = FLOAT = CODE = EXPONENTS = MASTER = PARAM_MASK = STAMP = 0
        collect = staticmethod(lambda *lists: ((None,) * 8, b"", b"", b"", 1, []))
        scalars = staticmethod(lambda *numbers: (b"", b"", None, None, True))
    monkeypatch.setattr(optim, "_on", on)
    monkeypatch.setattr(optim._lib, "host", Host)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: entered == [1])
    one = [torch.zeros(8)]
    with pytest.raises(RuntimeError, match="same at every replay"):
        optim.adamw_step_(one, one, one, one, step=1)


def test_no_norm_stays_from_a_step_before_where_no_parameter_has_a_gradient():
    p = torch.nn.Parameter(torch.zeros(4))
    opt = optim.AdamW([p], max_grad_norm=1.0)
    opt.last_grad_norm = torch.tensor(3.0)
    opt.step()
    assert float(opt.last_grad_norm) == 0.0 and opt.last_grad_norm.dtype == torch.float32 and opt.last_grad_norm.shape == ()
    opt = optim.AdamW([p])
    opt.step()
    assert opt.last_grad_norm is None


@pytest.mark.parametrize("kind", [optim.AdamW, optim.Adam])
def test_a_mask_does_not_pass_on_to_a_parameter_that_takes_anothers_place(kind):
    """Parameters are replaced where points are added and removed; a new object may have the address of the one that went."""
    mask = torch.ones(4, dtype=torch.int8)
    for _ in range(100):
        opt = kind([torch.nn.Parameter(torch.zeros(4, 3))])
        opt.set_row_mask(opt.param_groups[0]["params"][0], mask)
        opt.param_groups[0]["params"][0] = None
        q = torch.nn.Parameter(torch.zeros(4, 3))
        opt.param_groups[0]["params"][0] = q
        assert not any(key is q or (isinstance(key, int) and key == id(q)) for key in opt._row_mask)
    # copies keep the masks of the parameters that are there
    if kind is optim.AdamW:
        import copy
        opt.set_row_mask(q, mask)
        twin = copy.deepcopy(opt)
        (r,) = twin.param_groups[0]["params"]
        assert [(key is r, bool(m.all())) for key, m in twin._row_mask.items()] == [(True, True)]
