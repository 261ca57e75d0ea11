"""Rows beyond a workgroup's share and masked rows at odd addresses, against the plain implementation in 64 bits."""
import numpy as np
import pytest
import torch

from tests import adamw_plain as plain
from tests.test_adamw_gpu import DEV, HYPER, TYPES, _check_step, _inputs, _np, _optim, _place

pytestmark = pytest.mark.gpu
# (a workgroup takes 2048 / 1024 / 1024 / 512 rows of 1 / 2 / 3 / 4 elements; of longer rows at most 512)
NARROW = [(5003, 1), (3001, 2), (5003, 3), (1501, 4)]
# (and from 32768 rows on a lane has four quads at once: reading takes 4096 elements a workgroup)
MANY = [(40_003, 1), (35_001, 2), (40_003, 3), (33_001, 4), (1301, 5), (1301, 17)]


@pytest.mark.parametrize("dtype,with_master", TYPES)
@pytest.mark.parametrize("shapes,offset", [(NARROW, 0), (NARROW, 1), (MANY, 0), (MANY, 1)])
def test_short_rows_with_8_bits_in_later_workgroups(dtype, with_master, shapes, offset):
    o = _optim()
    tensors = [_inputs(s, dtype, 8, i, offset) for i, s in enumerate(shapes)]
    masters = [_place(t[0].float() * (1 + 2e-3), offset) for t in tensors] if with_master else None
    before = [((_np(masters[i]) if masters else _np(t[0])), *(_np(x) for x in t[1:])) for i, t in enumerate(tensors)]
    for out_dtype in (torch.float32, torch.bfloat16):
        for t, m, v in zip(tensors, *o.read_moments(*([t[k] for t in tensors] for k in (2, 3, 4)), dtype=out_dtype)):
            true_m, true_v = plain.decode(_np(t[2]), _np(t[3]), _np(t[4]), tuple(t[0].shape))
            normal = np.abs(true_m) >= 2.0 ** -126, true_v >= 2.0 ** -126
            assert np.array_equal(_np(m)[normal[0]], true_m[normal[0]]) and np.array_equal(_np(v)[normal[1]], true_v[normal[1]])
    o.adamw_step_(*[[t[k] for t in tensors] for k in range(4)], step=17, exponents=[t[4] for t in tensors], masters=masters, seed=5, **HYPER)
    for i, t in enumerate(tensors):
        _check_step(before[i], (t[0], t[2], t[3], t[4]), dtype, 17, 8, seed=5, tensor=i, master=masters[i] if masters else None)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("shape", [*NARROW, (1237, 5), (1237, 7), (1237, 16), (1237, 17), (601, 33), (601, 56), (601, 63)])
def test_masked_rows_at_odd_addresses_and_in_later_workgroups(bits, offset, shape):
    """Masked rows hold NaN; their bits, exponents and stamps stay, the others are stepped with their decay."""
    o = _optim()
    p, g, m, v, x = _inputs(shape, torch.float32, bits, shape[1], offset)
    gen = torch.Generator().manual_seed(shape[1])
    mask = (torch.rand(shape[0], generator=gen) < 0.4).to(torch.int8)
    stamps = 19 - torch.randint(0, 8, (shape[0],), generator=gen) * (torch.rand(shape[0], generator=gen) < 0.5)
    mask, stamps = _place(mask.to(DEV), offset), _place(stamps.to(torch.int32).to(DEV), offset)
    if x is not None:
        x = _place(x, offset)
    dead = mask != 0
    for t in (p, g) + ((m, v) if bits == 32 else ()):
        t[dead] = float("nan")
    if bits == 8:
        x[dead] = 255
    before = (_np(p), _np(g), _np(m), _np(v), None if x is None else _np(x))
    kept = [t.clone() for t in (p, m, v, stamps) + (() if x is None else (x,))]
    o.adamw_step_([p], [g], [m], [v], step=20, exponents=None if x is None else [x], row_masks=[mask], last_steps=[stamps], seed=4, **HYPER)
    bits_of = lambda t: t.view(torch.uint8 if t.dtype == torch.uint8 else torch.int32)  # noqa: E731
    for t, old in zip((p, m, v) + (() if x is None else (x,)), kept[:3] + kept[4:]):
        assert torch.equal(bits_of(t[dead]), bits_of(old[dead])), "a masked row was written"
    assert torch.equal(stamps, torch.where(dead, kept[3], torch.full_like(stamps, 20)))
    live, missed = ~dead.cpu().numpy(), 19 - kept[3].cpu().numpy()
    # (the comparison's own arrays: masked rows as zeros on both sides)
    clean = [None if b is None else np.where(live[:, None], b, 100 if k == 4 else 0) for k, b in enumerate(before)]
    after = [None if t is None else t.clone() for t in (p, m, v, x)]
    for k, t in enumerate(after):
        if t is not None:
            t[dead] = 100 if k == 3 else 0
    _check_step(tuple(clean), tuple(after), torch.float32, 20, bits, seed=4, missed=missed, live=live)
