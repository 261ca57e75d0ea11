"""optim.AdamW's operators without a device: refusals of the functions and of the C entry points, and the properties of the
8-bit moments' format and rounding (in the plain implementation that the device tests compare with)."""
import ctypes

import numpy as np
import pytest
import torch

from taichi_3d_gaussian_splatting_amd import _lib, optim
from tests import adamw_plain as plain


def test_every_code_and_exponent_of_the_format_is_its_own_value_and_fits_bfloat16():
    assert len(set(plain.M_TABLE)) == 127 and len(set(plain.V_TABLE)) == 256
    for table in (plain.M_TABLE, plain.V_TABLE):
        as_bf16 = torch.tensor(table, dtype=torch.float64).to(torch.bfloat16).double().numpy()
        assert np.array_equal(as_bf16, table)
    # steps: at most an eighth of the value (first moment: its normal codes), never none
    assert np.all(np.diff(plain.V_TABLE)[1:] / plain.V_TABLE[1:-1] <= 1 / 8 + 1e-15) and np.all(np.diff(plain.V_TABLE) > 0)
    assert np.all(np.diff(plain.M_TABLE)[8:] / plain.M_TABLE[8:-1] <= 1 / 8 + 1e-15)


def test_rounding_bits_are_even_and_independent_between_steps_and_elements():
    """Means of n uniform 16-bit numbers: within 5 standard deviations (1 / sqrt(12 n)) of one half; correlations of two such
    rows: within 5 / sqrt(n) of zero."""
    n = 1 << 16
    a, b, c = plain.noise(n, 0, 0, 1), plain.noise(n, 0, 0, 2), plain.noise(n, 0, 1, 1)
    def halves(x):
        return (x & np.uint64(0xFFFF)).astype(float) / 65536, (x >> np.uint64(16)).astype(float) / 65536
    for x in (a, b, c):
        for y in halves(x):
            assert abs(y.mean() - 0.5) < 5 / np.sqrt(12 * n)
            assert abs(np.corrcoef(y[:-1], y[1:])[0, 1]) < 5 / np.sqrt(n)
    for x, y in ((a, b), (a, c)):
        for k in range(2):
            assert abs(np.corrcoef(halves(x)[k], halves(y)[k])[0, 1]) < 5 / np.sqrt(n)
    assert abs(np.corrcoef(*halves(a))[0, 1]) < 5 / np.sqrt(n)
    # one element over many steps
    over = np.array([int(plain.noise(8, 0, 0, t)[5]) for t in range(1, 4097)], dtype=np.uint64)
    for y in halves(over):
        assert abs(y.mean() - 0.5) < 5 / np.sqrt(12 * 4096) and abs(np.corrcoef(y[:-1], y[1:])[0, 1]) < 5 / np.sqrt(4096)


def test_rounding_keeps_the_mean_and_a_positive_second_moment():
    """4096 roundings of one block: a rounding is within one code step s, so the mean is within 5 s / (2 sqrt(4096)) of the
    value (two outcomes: the standard deviation is at most s / 2)."""
    rng = np.random.default_rng(0)
    shape = (64,)
    m = rng.standard_normal(64) * 10.0 ** rng.uniform(-3, 0, 64)
    v = m * m * rng.uniform(0.5, 2, 64)
    v[3], v[4], m[5] = 0.0, v.max() * 2.0 ** -40, 0.0
    ms, vs = [], []
    for t in range(4096):
        mc, vc, x, _ = plain.encode(m, v, plain.noise(64, 7, 0, t + 1), shape)
        a, b = plain.decode(mc, vc, x, shape)
        ms.append(a)
        vs.append(b)
    ms, vs = np.array(ms), np.array(vs)
    step_m = np.maximum(np.abs(m) / 8, np.abs(m).max() * 2.0 ** -17)
    assert np.all(np.abs(ms.mean(0) - m) <= 5 * step_m / 2 / 64)
    inside = np.arange(64) != 4         # (v[4] lies below the smallest code: it is that code)
    assert np.all(np.abs(vs.mean(0) - v)[inside] <= 5 * v[inside] / 8 / 2 / 64)
    assert np.all(vs[:, 3] == 0) and np.all(vs[:, 4] > 0) and np.all(ms[:, 5] == 0)


def test_functions_refuse_host_tensors():
    p = torch.zeros(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.adamw_step_([p], [p.clone()], [p.clone()], [p.clone()], step=1)
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.grad_norm([p])
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.read_moments([torch.zeros(8, dtype=torch.uint8)], [torch.zeros(8, dtype=torch.uint8)], [torch.zeros(1, 2, dtype=torch.uint8)])
    q = torch.nn.Parameter(p)
    q.grad = p.clone()
    with pytest.raises(RuntimeError, match="HIP device"):
        optim.AdamW([q]).step()


def test_functions_refuse_wrong_lists_and_numbers():
    p = torch.zeros(8)
    one = [p], [p.clone()], [p.clone()], [p.clone()]
    with pytest.raises(ValueError, match="grads"):
        optim.adamw_step_([p], [], [p], [p], step=1)
    with pytest.raises(ValueError, match="come together"):
        optim.adamw_step_(*one, step=1, row_masks=[None])
    with pytest.raises(ValueError, match="positive"):
        optim.adamw_step_(*one, step=1, max_grad_norm=0.0)
    with pytest.raises(ValueError, match="positive"):
        optim.adamw_step_(*one, step=1, max_grad_norm=float("nan"))
    with pytest.raises(ValueError, match="exclude"):
        optim.adamw_step_(*one, step=1, max_grad_norm=1.0, grad_scale=p)
    with pytest.raises(ValueError, match="hyper"):
        optim.adamw_step_(*one, step=1, betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="no gradients"):
        optim.grad_norm([])
    with pytest.raises(ValueError):
        optim.new_moments(p, 16)
    assert optim.adamw_step_([], [], [], [], step=1) is None
    assert optim.read_moments([], [], []) == ([], [])
    for bad in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-0.1), dict(state_bits=4),
                dict(max_grad_norm=-1.0), dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(p.clone())], **bad)
    o = optim.AdamW([torch.nn.Parameter(torch.zeros(5, 65)), torch.nn.Parameter(torch.zeros(5, 3))])
    a, b = o.param_groups[0]["params"]
    with pytest.raises(ValueError):
        o.set_row_mask(a, torch.zeros(5, dtype=torch.int8))
    with pytest.raises(ValueError):
        o.set_row_mask(b, torch.zeros(4, dtype=torch.int8))
    with pytest.raises(TypeError):
        o.set_row_mask(b, torch.zeros(5, dtype=torch.bool))
    with pytest.raises(KeyError):
        o.moments(b)


@pytest.mark.parametrize("shape,blocks", [((0,), 0), ((1,), 1), ((64,), 1), ((65,), 2), ((7, 3), 7), ((7, 64), 7), ((7, 65), 8),
                                          ((2, 3, 4), 1), ((0, 5), 0), ((5, 0), 0), ((), 1)])
def test_new_moments_have_a_block_for_each_row_or_64_elements(shape, blocks):
    m, v, x = optim.new_moments(torch.zeros(shape), 8)
    assert m.shape == v.shape == torch.Size(shape) and m.dtype == v.dtype == x.dtype == torch.uint8 and x.shape == (blocks, 2)
    m, v, x = optim.new_moments(torch.zeros(shape, dtype=torch.bfloat16), 32)
    assert m.dtype == v.dtype == torch.float32 and x is None


def _step(**change):
    """Status and message of gs_adamw_step for one tensor whose arguments are changed (no launch is reached)."""
    u64, i64, i32, f64 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_int32, ctypes.c_double
    a = dict(n=1, param=0x10000, grad=0x20000, m=0x30000, v=0x40000, x=None, master=None, mask=None, last=None, numel=64, row=0,
             dtype=0, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1, step_dev=None, lr_dev=None, ws=None)
    a.update(change)
    ptr = lambda v: None if v is None else (u64 * 1)(v)  # noqa: E731
    lib = _lib.load()
    status = lib.gs_adamw_step(a["n"], ptr(a["param"]), ptr(a["grad"]), ptr(a["m"]), ptr(a["v"]), ptr(a["x"]), ptr(a["master"]),
                               ptr(a["mask"]), ptr(a["last"]), (i64 * 1)(a["numel"]), (i32 * 1)(a["row"]), (i32 * 1)(a["dtype"]),
                               (i32 * 1)(0), (f64 * 5)(a["lr"], a["b1"], a["b2"], a["eps"], a["wd"]), (i64 * 1)(a["step"]),
                               ptr(a["step_dev"]), ptr(a["lr_dev"]), None, 0, a["ws"], None)
    return status, lib.gs_last_error().decode()


@pytest.mark.parametrize("change,says", [
    (dict(n=-1), "tensors"), (dict(param=None), "null array"), (dict(param=0), "null tensor"), (dict(x=0), "null tensor"),
    (dict(numel=-1), "numel"), (dict(row=65, numel=65), "rows of 1..64"), (dict(row=3, numel=64), "rows of 1..64"),
    (dict(dtype=3), "dtype"), (dict(step=0), "step >= 1"), (dict(step=1 << 31), "step >= 1"), (dict(b1=1.0), "betas"),
    (dict(b2=float("nan")), "betas"), (dict(eps=-1.0), "betas"), (dict(mask=0x50000), "last steps"),
    (dict(mask=0x50000, last=0x60000), "row mask"), (dict(mask=0x50000, last=0x60000, row=4, dtype=1), "row mask"),
    (dict(master=0x50000), "master"), (dict(step_dev=0x50000), "workspace"), (dict(lr_dev=0x50000), "workspace"),
    (dict(param=0x10002), "multiple"), (dict(grad=0x20001, dtype=1), "multiple"), (dict(m=0x30002), "multiple"),
    (dict(grad=0x10000), "overlap"), (dict(m=0x10010), "overlap"), (dict(v=0x30000), "overlap"), (dict(x=0x30020), "overlap"),
    (dict(master=0x10000, dtype=1), "overlap"), (dict(mask=0x50000, last=0x40010, row=4), "overlap"),
    (dict(numel=1 << 62), "too large"),
])
def test_c_entry_of_the_step_refuses(change, says):
    status, message = _step(**change)
    assert status == -1 and says in message, (status, message)


def test_c_entries_with_nothing_to_do_or_missing_arguments():
    lib = _lib.load()
    assert lib.gs_adamw_step(0, *[None] * 17, 0, None, None) == 0
    assert lib.gs_read_moments(0, *[None] * 7, 0, None) == 0
    assert lib.gs_read_moments(1, *[None] * 7, 0, None) == -1
    assert lib.gs_grad_norm(0, *[None] * 5, 0.0, *[None] * 6) == -1
    assert lib.gs_clip_coefficient(None, 1.0, None, None, None) == -1
    assert lib.gs_adamw_workspace_bytes(3) >= 3 * 40 and lib.gs_adamw_workspace_bytes(-1) == 0
    assert lib.gs_grad_norm_workspace_bytes(3) >= 8 * 2003 and lib.gs_grad_norm_workspace_bytes(-1) == 0
