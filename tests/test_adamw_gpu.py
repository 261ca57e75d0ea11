"""optim.AdamW and its operators on the device, against the plain implementation in 64 bits (adamw_plain.py)."""
import numpy as np
import pytest
import torch

from tests import adamw_plain as plain

pytestmark = pytest.mark.gpu
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
DEV = "cuda:0"


def _optim():
    from taichi_3d_gaussian_splatting_amd import optim
    return optim


def _np(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def _place(x, offset):
    """The tensor at `offset` elements past an aligned address."""
    buffer = torch.empty(x.numel() + offset, dtype=x.dtype, device=DEV)
    y = buffer[offset:].view(x.shape)
    y.copy_(x)
    return y


def _inputs(shape, dtype, bits, seed, offset=0):
    """Parameter, gradient and moments of a tensor in training: magnitudes over five orders, some gradients zero."""
    gen = torch.Generator().manual_seed(seed)
    n = int(np.prod(shape))
    scale = 10.0 ** (torch.rand(-(-n // 8) + 1, generator=gen) * 5 - 5).repeat_interleave(8)[:n].view(shape)
    g = torch.randn(shape, generator=gen) * scale * (torch.rand(shape, generator=gen) > 0.1)
    p = torch.randn(shape, generator=gen)
    m = 0.5 * g + 0.3 * scale * torch.randn(shape, generator=gen)
    v = (0.5 * g) ** 2 + 1.2 * m * m
    p, g = _place(p.to(dtype), offset), _place(g.to(dtype), offset)
    if bits == 32:
        return p, g, _place(m, offset), _place(v, offset), None
    mc, vc, x, _ = plain.encode(m.double().numpy(), v.double().numpy(), plain.noise(n, 3, 0, 1), shape)
    return (p, g, _place(torch.from_numpy(mc), offset), _place(torch.from_numpy(vc), offset), torch.from_numpy(x).to(DEV))


HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _assert_near(got, want, bound, what):
    off = np.abs(got - want)
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float((off / np.maximum(bound, 1e-300))[bad].max()), np.argwhere(bad)[:3].tolist())


def _check_step(before, after, dtype, step, bits, seed=0, tensor=0, scale=1.0, master=None, missed=None, live=None):
    """One tensor's state before and after the step: `before` (p or master, g, m, v, exponents) as numpy, `after` as tensors."""
    p0, g, m0, v0, x0 = before
    p1, m1, v1, x1 = after
    shape = p0.shape
    if p0.size == 0:
        return
    if bits == 8:
        code_m, code_v = m0, v0
        m0, v0 = plain.decode(m0, v0, x0, shape)
    p, m, v = plain.update(p0, g, m0, v0, step=step, scale=scale, missed=missed, **HYPER)
    ep, em, ev = plain.error_bounds(p0, p, g * scale, m0, m, v, step=step, **HYPER)
    keep = np.zeros(shape, bool) if live is None else np.broadcast_to(~live[:, None], shape)
    if master is not None:
        _assert_near(_np(master), np.where(keep, p0, p), np.where(keep, 0, ep), "master")
        assert torch.equal(p1, master.to(dtype))
    else:
        spacing = HALF[dtype] * np.abs(p) + (2.0 ** -25 if dtype == torch.float16 else 0) if dtype != torch.float32 else 0
        # (an error of ep before a rounding moves what it gives by at most ep and half a spacing more)
        _assert_near(_np(p1), np.where(keep, p0, p), np.where(keep, 0, ep * 1.01 + spacing * (1 + 1e-3)), "param")
    if bits == 32:
        _assert_near(_np(m1), np.where(keep, m0, m), np.where(keep, 0, em), "exp_avg")
        _assert_near(_np(v1), np.where(keep, v0, v), np.where(keep, 0, ev), "exp_avg_sq")
        return
    mc, vc, x, margins = plain.encode(m, v, plain.noise(p0.size, seed, tensor, step), shape)
    keep_blocks = np.zeros(len(x), bool) if live is None else ~live
    # exponents: the same, unless a block's largest value is within its error of the limit
    same_x = (x1.cpu().numpy() == np.where(keep_blocks[:, None], x0, x)).all(1)
    assert same_x.mean() > 1 - 1e-3 - 1.5 / len(x), (same_x.mean(), len(x))
    where = plain.blocks_of(shape)[0].reshape(shape)
    dm, dv = plain.decode(m1.cpu().numpy(), v1.cpu().numpy(), x1.cpu().numpy(), shape)
    wm, wv = plain.decode(mc, vc, x, shape)
    for got, want, code, old, table, err, true, margin, codes in (
            (dm, wm, m1, code_m, plain.M_TABLE, em, m, margins[0], mc), (dv, wv, v1, code_v, plain.V_TABLE, ev, v, margins[1], vc)):
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        same = np.where(keep, (code.cpu().numpy() == old), same)
        # an element may have the neighbouring code only where its rounding was within the error of the limit.  A code's
        # step is at least 1/16 of the value (second moment, first from 2^-6 up) or 2^-17 of the block's largest.
        largest = np.zeros(len(x))
        np.maximum.at(largest, where.reshape(-1), np.where(np.isfinite(true), np.abs(true), 0).reshape(-1))
        step_size = np.maximum(np.abs(true) / 16, largest[where] * 2.0 ** -18 if table is plain.M_TABLE else 0) + 1e-300
        near = margin <= err / step_size + 1e-9
        wrong = ~same & ~near & same_x[where] & ~keep
        assert not wrong.any(), (int(wrong.sum()), np.argwhere(wrong)[:3].tolist(), got[wrong][:3], want[wrong][:3], margin[wrong][:3])
        assert same[same_x[where]].mean() > 1 - 1e-4 - 1.5 / same.size


SHAPES = [(1,), (3,), (4,), (63,), (64,), (65,), (1003,), (40_001,), (5, 1), (301, 3), (50, 4), (33, 5), (33, 7), (9, 16), (31, 17),
          (257, 56), (20, 63), (40, 64), (40, 65), (2, 3, 5), (0,), (0, 7), ()]
TYPES = [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float16, True)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,with_master", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_step_of_many_shapes_against_64_bits(bits, dtype, with_master, offset):
    """All shapes in one call; at an offset of one element nothing is aligned."""
    o = _optim()
    tensors = [_inputs(s, dtype, bits, 100 + i, offset) for i, s in enumerate(SHAPES)]
    masters = None
    if with_master:
        masters = [_place(t[0].float() * (1 + 2e-3), offset) for t in tensors]
    before = [((_np(masters[i]) if masters else _np(t[0])), _np(t[1]), _np(t[2]), _np(t[3]), None if t[4] is None else _np(t[4]))
              for i, t in enumerate(tensors)]
    grads = [t[1].clone() for t in tensors]
    out = o.adamw_step_([t[0] for t in tensors], [t[1] for t in tensors], [t[2] for t in tensors], [t[3] for t in tensors], step=17,
                        exponents=[t[4] for t in tensors] if bits == 8 else None, masters=masters, seed=5, **HYPER)
    assert out is None
    for i, t in enumerate(tensors):
        assert torch.equal(t[1], grads[i]), "a gradient was written"
        _check_step(before[i], (t[0], t[2], t[3], t[4]), dtype, 17, bits, seed=5, tensor=i, master=masters[i] if masters else None)


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_types_in_one_call_and_more_tensors_than_a_batch_holds(bits):
    o = _optim()
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    shapes = [(1 + 37 * (i % 29),) if i % 4 else (3 + i % 11, 1 + i % 70) for i in range(130)]
    tensors = [_inputs(s, kinds[i % 3], bits, i, offset=i % 2) for i, s in enumerate(shapes)]
    masters = [t[0].float() if i % 3 == 1 and i % 2 else None for i, t in enumerate(tensors)]
    before = [(_np(t[0]), _np(t[1]), _np(t[2]), _np(t[3]), None if t[4] is None else _np(t[4])) for t in tensors]
    o.adamw_step_(*[[t[k] for t in tensors] for k in range(4)], step=[1 + i % 5 for i in range(130)], masters=masters,
                  exponents=[t[4] for t in tensors] if bits == 8 else None, **HYPER)
    for i, t in enumerate(tensors):
        _check_step(before[i], (t[0], t[2], t[3], t[4]), kinds[i % 3], 1 + i % 5, bits, tensor=i, master=masters[i])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("columns", [1, 3, 4, 7, 16, 17, 56, 64])
@pytest.mark.parametrize("share", [0.0, 0.4, 1.0])
def test_row_masks_leave_rows_alone_and_late_rows_decay(bits, columns, share):
    """Masked rows hold NaN and infinities everywhere, in the gradient too: nothing of them is touched, or seen by the norm."""
    o = _optim()
    shape = (1237, columns)
    p, g, m, v, x = _inputs(shape, torch.float32, bits, columns)
    gen = torch.Generator().manual_seed(columns)
    mask = (torch.rand(shape[0], generator=gen) < share).to(torch.int8)
    mask[mask != 0] = torch.randint(1, 3, (int((mask != 0).sum()),), generator=gen).to(torch.int8) * 2 - 3   # -1 and 1
    stamps = (20 - 1 - torch.randint(0, 8, (shape[0],), generator=gen) * (torch.rand(shape[0], generator=gen) < 0.5)).to(torch.int32)
    mask, stamps = mask.to(DEV), stamps.to(DEV)
    dead = mask != 0
    for t in (p, g) + ((m, v) if bits == 32 else ()):
        t[dead] = float("nan")
        t[dead.nonzero()[::2, 0]] = float("inf")
    if bits == 8:
        x[dead] = 255
    before = (_np(p), _np(g), _np(m), _np(v), None if x is None else _np(x))
    raw = [t.clone() for t in (p, m, v, stamps)] + ([x.clone()] if x is not None else [])
    live = ~dead.cpu().numpy()
    true = float(np.sqrt((np.where(live[:, None], before[1], 0) ** 2).sum()))
    norm = o.adamw_step_([p], [g], [m], [v], step=20, exponents=None if x is None else [x], row_masks=[mask], last_steps=[stamps],
                         max_grad_norm=0.5, **HYPER)
    assert abs(float(norm) - true) <= 2.0 ** -23 * true
    for t, old in zip((p, m, v) + ((x,) if x is not None else ()), (raw[0], raw[1], raw[2]) + tuple(raw[4:])):
        assert torch.equal(t[dead].view(torch.uint8 if t.dtype == torch.uint8 else torch.int32),
                           old[dead].view(torch.uint8 if t.dtype == torch.uint8 else torch.int32)), "a masked row was written"
    assert torch.equal(stamps, torch.where(dead, raw[3], torch.full_like(stamps, 20)))
    if not live.any():
        return
    rows = np.where(live)[0]
    cut = lambda a: a[rows]  # noqa: E731
    if bits == 32:
        _check_step(tuple(cut(b) for b in before[:4]) + (None,), (p[~dead], m[~dead], v[~dead], None), torch.float32, 20, 32,
                    scale=min(1.0, 0.5 / (true + 1e-6)), missed=(20 - 1 - raw[3].cpu().numpy())[rows])
    else:
        clean = [np.where(live[:, None], b, 0) for b in before]
        clean[4] = np.where(live[:, None], before[4], 100)
        p2, m2, v2, x2 = p.clone(), m.clone(), v.clone(), x.clone()
        p2[dead], m2[dead], v2[dead], x2[dead] = 0, 0, 0, 100
        _check_step(tuple(clean), (p2, m2, v2, x2), torch.float32, 20, 8, scale=min(1.0, 0.5 / (true + 1e-6)),
                    missed=19 - raw[3].cpu().numpy(), live=live)


def test_a_row_masked_for_a_while_continues_like_one_with_zero_gradients():
    """Lazy decay: moments of a row that missed d steps are those of d steps with gradient zero, to float32's rounding of d
    products (2 d 2^-24) and of the power (16 units)."""
    o = _optim()
    shape, d = (500, 56), 30
    p, g, m, v, _ = _inputs(shape, torch.float32, 32, 3)
    a, b = [t.clone() for t in (p, m, v)], [t.clone() for t in (p, m, v)]
    stamps = torch.full((500,), 10, dtype=torch.int32, device=DEV)
    mask = torch.ones(500, dtype=torch.int8, device=DEV)
    for t in range(11, 11 + d):
        o.adamw_step_([a[0]], [g], [a[1]], [a[2]], step=t, row_masks=[mask], last_steps=[stamps], **HYPER)
        o.adamw_step_([b[0]], [torch.zeros_like(g)], [b[1]], [b[2]], step=t, **HYPER)
    assert torch.equal(a[0], p) and int(stamps.max()) == 10
    b[0].copy_(p)
    mask.zero_()
    o.adamw_step_([a[0]], [g], [a[1]], [a[2]], step=11 + d, row_masks=[mask], last_steps=[stamps], **HYPER)
    o.adamw_step_([b[0]], [g], [b[1]], [b[2]], step=11 + d, **HYPER)
    bound = (2 * d + 16) * 2.0 ** -24
    for x, y, old in ((a[1], b[1], m), (a[2], b[2], v)):
        assert ((x - y).abs() <= bound * (old.abs() + y.abs()) + 1e-38).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e25])
def test_gradients_that_are_not_finite_stay_where_they_are(bits, bad):
    """32 bits: the element alone (1e25: its square is infinite, its update 0 / inf).  8 bits: its block, whose values become
    NaN where a moment has no finite value; every other block as if nothing had happened."""
    o = _optim()
    p, g, m, v, x = _inputs((640,), torch.float32, bits, 9)
    clean = [t.clone() for t in (p, g, m, v)] + ([x.clone()] if bits == 8 else [])
    g[130] = bad
    for q in ((p, g, m, v, x), clean + [None] * (5 - len(clean))):
        o.adamw_step_([q[0]], [q[1]], [q[2]], [q[3]], step=3, exponents=None if bits == 32 else [q[4]], **HYPER)
    other = torch.ones(640, dtype=torch.bool, device=DEV)
    other[128:192] = False
    alone = torch.ones(640, dtype=torch.bool, device=DEV)
    alone[130] = False
    assert torch.equal(p[alone], clean[0][alone])
    if bits == 32:
        assert torch.equal(m[alone], clean[2][alone]) and torch.equal(v[alone], clean[3][alone])
        assert not torch.isfinite(v[130])
        return
    assert torch.equal(m[other], clean[2][other]) and torch.equal(v[other], clean[3][other])
    (a,), (b,) = o.read_moments([m], [v], [x])
    assert torch.isnan(b[128:192]).all() and torch.isfinite(b[other]).all() and torch.isfinite(a[other]).all()
    assert torch.isnan(a[128:192]).all() == (not np.isfinite(bad))


def test_read_moments_gives_every_code_its_value():
    """All 256 x 256 pairs of codes under exponents from 0 to 255, in both types; the format's edges among them."""
    o = _optim()
    codes = torch.arange(256, dtype=torch.uint8)
    shapes = [(256, 64), (256 * 64,), (700, 3), (99, 7), (10, 16), (51, 65)]
    gen = torch.Generator().manual_seed(0)
    ms, vs, xs = [], [], []
    for s in shapes:
        n = int(np.prod(s))
        ms.append(codes.repeat(n // 256 + 1)[:n].view(s).contiguous().to(DEV))
        vs.append(codes.repeat(n // 256 + 1)[:n][torch.randperm(n, generator=gen)].view(s).contiguous().to(DEV))
        blocks = plain.blocks_of(s)[1]
        xs.append(torch.stack([torch.arange(blocks) % 256, (torch.arange(blocks) * 7 + 3) % 256], 1).to(torch.uint8).to(DEV))
    for dtype in (torch.float32, torch.bfloat16):
        a, b = o.read_moments(ms, vs, xs, dtype=dtype)
        for k, s in enumerate(shapes):
            m, v = plain.decode(_np(ms[k]), _np(vs[k]), _np(xs[k]), s)
            nan_code = (_np(ms[k]) & 127) == 127        # never written; it has a value of its own or NaN
            for got, want in ((a[k], np.where(nan_code, 0, m)), (b[k], v)):
                got = _np(got)
                got = np.where(nan_code, 0, got) if want is not v else got
                big = np.abs(want) > 3.4e38             # beyond float32: infinite
                got, want = np.where(big, 0, got), np.where(big, 0, want)
                tiny = np.abs(want) < 2.0 ** -126       # below the normal range nothing is promised but the size
                assert np.array_equal(np.isnan(got), np.isnan(want))
                assert (np.abs(got[tiny]) <= 2.0 ** -125).all()
                ok = ~tiny & ~np.isnan(want)
                assert np.array_equal(got[ok], want[ok])
    out = ([torch.full(s, 7.0, device=DEV) for s in shapes], [torch.full(s, 7.0, device=DEV) for s in shapes])
    got = o.read_moments(ms, vs, xs, out=out)
    f32 = o.read_moments(ms, vs, xs)
    for k in range(len(shapes)):
        assert got[0][k] is out[0][k] and torch.equal(out[0][k].nan_to_num(1.5), f32[0][k].nan_to_num(1.5))
        assert torch.equal(out[1][k].nan_to_num(1.5), f32[1][k].nan_to_num(1.5))


def test_second_moments_in_8_bits_reach_their_level_and_follow_it_down():
    """Constant gradient magnitudes with random signs: v goes to g^2, and from a hundred times as much back down to it.  With
    b2 = 0.99 a code step (1/16..1/8) is six times what a step moves: rounding to nearest would stay where it is.  Stationary
    spread: steps of s = 1/8 with the chance that keeps the mean add at most |change| s to the relative variance, 0.01 / 8
    each, remembered for 50: 0.0625, a deviation of 0.25 an element, of 0.25 / sqrt(65536 / 8) = 0.003 in the mean even if
    eight neighbours moved together; 5 deviations are 0.014."""
    o = _optim()
    n = 1 << 16
    gen = torch.Generator(device=DEV).manual_seed(1)
    size = 10.0 ** (torch.rand(n, device=DEV, generator=gen) * 2 - 3)
    for start in (0.0, 100.0):
        p = torch.zeros(n, device=DEV)
        m, v, x = o.new_moments(p, 8)
        t = 0
        def run(k, factor):
            nonlocal t
            for _ in range(k):
                t += 1
                g = size * factor * torch.where(torch.rand(n, device=DEV, generator=gen) < 0.5, -1.0, 1.0)
                o.adamw_step_([p], [g], [m], [v], step=t, exponents=[x], betas=(0.9, 0.99), lr=0.0, weight_decay=0.0)
        if start:
            run(600, start ** 0.5)
        run(1500, 1.0)
        b = o.read_moments([m], [v], [x])[1][0]
        ratio = (b / size ** 2)
        assert abs(float(ratio.mean()) - 1) < 0.014 + 0.01, float(ratio.mean())   # (0.99^1500 is nothing; 1 % for 16-bit chances)
        assert float((ratio - 1).square().mean().sqrt()) < 0.3


# ------------------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_grad_norm_of_mixed_types_and_sizes(offset):
    o = _optim()
    gen = torch.Generator().manual_seed(offset)
    sizes = [1, 5, 0, 64, 4095, 4096, 4097, 100_003, 2_500_001] + [7 + 13 * i for i in range(90)]
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    grads = [_place((torch.randn(n, generator=gen) * 10.0 ** (i % 5 - 2)).to(kinds[i % 3]), offset) for i, n in enumerate(sizes)]
    norm, each = o.grad_norm(grads, per_tensor=True)
    true = np.array([np.sqrt((_np(g) ** 2).sum()) for g in grads])
    # one rounding to float32 (2^-24) of sums that are right to 1e-12
    _assert_near(_np(each), true, true * 2.0 ** -24 * 1.001, "each")
    total = np.sqrt((true ** 2).sum())
    assert abs(float(norm) - total) <= total * 2.0 ** -24 * 1.001
    again, same = o.grad_norm(grads, per_tensor=True)
    assert torch.equal(norm, again) and torch.equal(each, same)
    assert torch.equal(o.grad_norm(grads), norm)


def test_grad_norm_shows_what_is_not_finite_and_skips_masked_rows():
    o = _optim()
    a, b = torch.randn(1000, 56, device=DEV), torch.randn(1000, 3, device=DEV)
    mask = (torch.arange(1000, device=DEV) % 3 == 0).to(torch.int8)
    for bad in (float("nan"), float("inf")):
        c = a.clone()
        c[300, 5] = bad                       # row 300 is masked
        norm = o.grad_norm([c, b], [mask, None])
        keep = a[mask == 0].double()
        true = float((keep.square().sum() + b.double().square().sum()).sqrt())
        assert abs(float(norm) - true) <= true * 2.0 ** -24 * 1.001
        c[301, 5] = bad
        norm, each = o.grad_norm([c, b], [mask, None], per_tensor=True)
        assert (np.isnan if np.isnan(bad) else np.isinf)(float(norm)) and not np.isfinite(float(each[0])) and np.isfinite(float(each[1]))
    assert float(o.grad_norm([a * 0])) == 0.0
    assert float(o.grad_norm([torch.zeros(0, device=DEV)])) == 0.0
    assert float(o.grad_norm([a], [torch.ones(1000, dtype=torch.int8, device=DEV)])) == 0.0
    # squares beyond float32 are added up in double precision
    assert abs(float(o.grad_norm([torch.full((4,), 1e30, device=DEV)])) - 2e30) < 1e24
    t = torch.randn(64, 64, device=DEV)
    assert torch.equal(o.grad_norm([t.t()]), o.grad_norm([t.t().contiguous()]))


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_equals_scaled_gradients(bits):
    """max_grad_norm against a step whose gradients were scaled by the coefficient before (one rounding of the product either
    way: the same bits), above and below the limit."""
    o = _optim()
    for limit in (0.01, 1e6):
        tensors = [_inputs(s, torch.float32, bits, i) for i, s in enumerate([(1000, 56), (1000, 3), (12_345,)])]
        twin = [[None if t is None else t.clone() for t in ts] for ts in tensors]
        args = dict(step=4, **HYPER)
        norm = o.adamw_step_(*[[t[k] for t in tensors] for k in range(4)], exponents=[t[4] for t in tensors] if bits == 8 else None,
                             max_grad_norm=limit, **args)
        true = float(torch.cat([t[1].flatten() for t in tensors]).double().norm())
        assert abs(float(norm) - true) <= true * 2.0 ** -24 * 1.001
        clip = torch.tensor(min(1.0, limit / (true + 1e-6)), device=DEV)
        o.adamw_step_([t[0] for t in twin], [t[1] * clip for t in twin], [t[2] for t in twin], [t[3] for t in twin],
                      exponents=[t[4] for t in twin] if bits == 8 else None, **args)
        for a, b in zip(tensors, twin):
            for k in (0, 2, 3, 4):
                assert a[k] is None or torch.equal(a[k], b[k])


# ------------------------------------------------------------------------------------------------ the optimiser
def _parameters(seed, kinds=(torch.float32,)):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    shapes = [(1001, 56), (333, 3), (7,), (65, 130)]
    return [torch.nn.Parameter(torch.randn(s, device=DEV, generator=gen).to(kinds[i % len(kinds)])) for i, s in enumerate(shapes)]


def _feed(params, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, device=DEV, generator=gen) * 10.0 ** (seed % 4 - 3)).to(p.dtype)


def test_class_follows_torch_adamw():
    """30 steps with two groups, a decaying rate and a parameter that now and then has no gradient.  A step's rounding is at
    most 16 units of 2^-24 of its size (adamw_plain.error_bounds), itself at most about 10 lr here, and the parameter's own
    2 units: 30 (160 lr + 3 |p|) 2^-24 for each of the two sides."""
    o = _optim()
    mine, ref = _parameters(1), _parameters(1)
    groups = lambda ps: [dict(params=ps[:2], lr=2e-3, weight_decay=0.1), dict(params=ps[2:], betas=(0.8, 0.99), eps=1e-6)]  # noqa: E731
    a = o.AdamW(groups(mine), lr=1e-3)
    b = torch.optim.AdamW(groups(ref), lr=1e-3, foreach=False, fused=False)
    sa, sb = (torch.optim.lr_scheduler.ExponentialLR(x, gamma=0.9) for x in (a, b))
    for it in range(30):
        _feed(mine, it)
        _feed(ref, it)
        if it % 7 == 3:
            mine[2].grad = ref[2].grad = None
        a.step()
        b.step()
        if it % 5 == 0:
            sa.step()
            sb.step()
    for p, q in zip(mine, ref):
        assert ((p - q).abs() <= 60 * 2.0 ** -24 * (160 * 2e-3 + 3 * q.abs())).all(), (p - q).abs().max()
    x, y = a.state_dict()["state"], b.state_dict()["state"]
    assert all(int(x[k]["step"]) == int(y[k]["step"]) for k in x)
    # torch's own state continues here
    c = o.AdamW(groups(ref), lr=1e-3)
    c.load_state_dict(b.state_dict())
    for k, p in enumerate(ref):
        m, v = c.moments(p)
        assert torch.equal(m, y[k]["exp_avg"]) and torch.equal(v, y[k]["exp_avg_sq"])
    _feed(mine, 99)
    _feed(ref, 99)
    a.step()
    c.step()
    for p, q in zip(mine, ref):
        assert ((p - q).abs() <= 62 * 2.0 ** -24 * (160 * 2e-3 + 3 * q.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_state_dict_round_trip_continues_bit_for_bit(bits, capturable, tmp_path):
    o = _optim()
    kinds = (torch.float32, torch.float32, torch.bfloat16, torch.float16)
    mask = (torch.arange(1001, device=DEV) % 4 == 0).to(torch.int8)

    def build():
        ps = _parameters(2, kinds)
        opt = o.AdamW(ps, lr=1e-3, state_bits=bits, max_grad_norm=1.0, seed=3, capturable=capturable)
        opt.set_row_mask(ps[0], mask)
        return ps, opt
    ps, opt = build()
    for it in range(4):
        _feed(ps, it)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "state.pt")
    qs, other = build()
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    other.load_state_dict(torch.load(tmp_path / "state.pt", weights_only=True))
    for it in range(4, 7):
        _feed(ps, it)
        _feed(qs, it)
        opt.step()
        other.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for name, value in opt.state[p].items():
            twin = other.state[q][name]
            assert type(value) is type(twin)
            if isinstance(value, torch.Tensor):
                assert value.dtype == twin.dtype and torch.equal(value, twin), name
            else:
                assert value == twin
    assert opt.state[ps[0]]["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
    assert "master" in opt.state[ps[2]] and "master" not in opt.state[ps[0]]


def test_load_state_dict_refuses_what_does_not_fit():
    o = _optim()
    ps = _parameters(2)
    opt = o.AdamW(ps, state_bits=8)
    _feed(ps, 0)
    opt.step()
    good = opt.state_dict()
    bad = {"state": {k: dict(s) for k, s in good["state"].items()}, "param_groups": good["param_groups"]}
    bad["state"][0]["exp_avg"] = bad["state"][0]["exp_avg"][:5]
    with pytest.raises(ValueError, match="shape"):
        o.AdamW(_parameters(2), state_bits=8).load_state_dict(bad)
    bad["state"][0]["exp_avg"] = good["state"][0]["exp_avg"].float()
    with pytest.raises(TypeError, match="uint8"):
        o.AdamW(_parameters(2), state_bits=8).load_state_dict(bad)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays_like_eager_steps(bits):
    """A step with clipping, masks, a 16-bit parameter with its copy, a step count and a learning rate on the device, captured
    once and replayed with new gradients and rates, eager work and waits in between: the same bits as an eager optimiser."""
    o = _optim()
    kinds = (torch.float32, torch.float32, torch.bfloat16, torch.float32)
    mask = (torch.arange(1001, device=DEV) % 5 == 0).to(torch.int8)
    sides = []
    for _ in range(2):
        ps = _parameters(5, kinds)
        lr = torch.tensor(1e-3, device=DEV)
        opt = o.AdamW(ps, lr=lr, state_bits=bits, max_grad_norm=0.7, capturable=True, seed=1)
        opt.set_row_mask(ps[0], mask)
        _feed(ps, 0)
        opt.step()
        sides.append((ps, lr, opt))
    (ps, lr, opt), (qs, lr2, eager) = sides
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    captured_norm = opt.last_grad_norm
    for it in range(1, 6):
        new = [torch.randn_like(p) * 10.0 ** (it % 3 - 2) for p in ps]
        for p, q, g in zip(ps, qs, new):
            p.grad.copy_(g)
            q.grad.copy_(g)
        lr.fill_(1e-3 / it)
        lr2.fill_(1e-3 / it)
        if it == 3:
            mask.copy_((torch.arange(1001, device=DEV) % 7 == 0).to(torch.int8))
        graph.replay()
        if it % 2:
            torch.cuda.synchronize()
        eager.step()
        assert torch.equal(captured_norm, eager.last_grad_norm)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q), it
            for name, value in opt.state[p].items():
                assert torch.equal(value, eager.state[q][name]), (it, name)
    assert int(opt.state[ps[0]]["step"]) == 6


def test_capture_is_refused_where_it_would_repeat_a_step():
    o = _optim()
    ps = _parameters(5)
    _feed(ps, 0)
    opt, fresh = o.AdamW(ps), o.AdamW(ps, capturable=True)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="same at every replay"):
            opt.step()
        with pytest.raises(RuntimeError, match="before capturing"):
            fresh.step()
        keep = ps[0] + 1        # (a graph holds something)
    graph.replay()
    torch.cuda.synchronize()
    assert keep.shape == ps[0].shape


def test_two_optimisers_on_two_streams_do_not_meet():
    """Interleaved steps with clipping on two streams, against the same steps one after the other."""
    o = _optim()
    def build(k):
        ps = _parameters(20 + k)
        return ps, o.AdamW(ps, state_bits=8, max_grad_norm=0.5, seed=k)
    serial = [build(k) for k in range(2)]
    for k, (ps, opt) in enumerate(serial):
        for it in range(10):
            _feed(ps, it + 100 * k)
            opt.step()
    torch.cuda.synchronize()
    both = [build(k) for k in range(2)]
    grads = []
    for k, (ps, _) in enumerate(both):
        rows = []
        for it in range(10):
            _feed(ps, it + 100 * k)
            rows.append([p.grad for p in ps])
        grads.append(rows)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for it in range(10):
        for k, (ps, opt) in enumerate(both):
            with torch.cuda.stream(streams[k]):
                for p, g in zip(ps, grads[k][it]):
                    p.grad = g
                opt.step()
    torch.cuda.synchronize()
    for (ps, a), (qs, b) in zip(serial, both):
        assert torch.equal(a.last_grad_norm, b.last_grad_norm)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


def test_device_refusals():
    o = _optim()
    p = torch.zeros(8, 8, device=DEV)
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    good = [[p], [z(8, 8)], [z(8, 8)], [z(8, 8)]]
    def step(lists=good, **more):
        return o.adamw_step_(*lists, **{"step": 1, **more})
    def swapped(k, t):
        return good[:k] + [[t]] + good[k + 1:]
    with pytest.raises(TypeError):
        step(swapped(0, z(8, 8, dtype=torch.float64)))
    with pytest.raises(TypeError):
        step(swapped(1, z(8, 8, dtype=torch.bfloat16)))
    with pytest.raises(ValueError, match="shape"):
        step(swapped(1, z(4, 16)))
    with pytest.raises(RuntimeError, match="device"):
        step(swapped(2, torch.zeros(8, 8)))
    with pytest.raises(ValueError, match="contiguous"):
        step(swapped(3, z(8, 8).t()[:, :]))
    with pytest.raises(TypeError):
        step(exponents=[z(8, 2, dtype=torch.uint8)])
    with pytest.raises(ValueError, match="master"):
        step(masters=[z(8, 8)])
    with pytest.raises(ValueError, match="counts from 1"):
        step(step=0)
    with pytest.raises(ValueError, match="step"):
        step(step=torch.zeros((), device=DEV))
    with pytest.raises(ValueError, match="lr"):
        step(lr=torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="lr"):
        step(lr=[1e-3, 1e-3])
    with pytest.raises(ValueError, match="hyper"):
        step(lr=-1e-3)
    with pytest.raises(ValueError, match="grad_scale"):
        step(grad_scale=torch.ones(()))
    with pytest.raises(RuntimeError, match="overlap"):
        step(swapped(2, good[0][0]))
    with pytest.raises(RuntimeError, match="overlap"):
        o.adamw_step_([p, p], [z(8, 8)] * 2, [z(8, 8), z(8, 8)], [z(8, 8), z(8, 8)], step=1)
    with pytest.raises(ValueError, match="rows"):
        o.adamw_step_([z(8, 65)], [z(8, 65)], [z(8, 65)], [z(8, 65)], step=1, row_masks=[z(8, dtype=torch.int8)],
                      last_steps=[z(8, dtype=torch.int32)])
    with pytest.raises(TypeError):
        step(row_masks=[z(8, dtype=torch.bool)], last_steps=[z(8, dtype=torch.int32)])
    with pytest.raises(ValueError):
        step(row_masks=[z(7, dtype=torch.int8)], last_steps=[z(8, dtype=torch.int32)])
    with pytest.raises(TypeError):
        half = [[t[0].bfloat16()] for t in good[:2]] + good[2:]
        step(half, row_masks=[z(8, dtype=torch.int8)], last_steps=[z(8, dtype=torch.int32)])
    with pytest.raises(TypeError):
        o.grad_norm([z(4, dtype=torch.int32)])
    with pytest.raises(TypeError):
        o.read_moments([z(4, dtype=torch.uint8)], [z(4, dtype=torch.uint8)], [z(1, 2, dtype=torch.uint8)], dtype=torch.float16)
    with pytest.raises(ValueError):
        o.read_moments([z(65, dtype=torch.uint8)], [z(65, dtype=torch.uint8)], [z(1, 2, dtype=torch.uint8)])
    assert not p.any()
    shared = z(8, 8) + 1       # two parameters may share a gradient
    o.adamw_step_([p, z(8, 8)], [shared, shared], [z(8, 8), z(8, 8)], [z(8, 8), z(8, 8)], step=1)


def test_offsets_beyond_32_bits():
    """A bfloat16 tensor of 2^31 + 77 elements, 8-bit moments (byte offsets up to 4 GiB, element offsets past 2^31): its head,
    the places around 2^31 and its tail."""
    o = _optim()
    n = (1 << 31) + 77
    p = torch.empty(n, dtype=torch.bfloat16, device=DEV).normal_()
    g = torch.empty(n, dtype=torch.bfloat16, device=DEV).normal_()
    m, v, x = o.new_moments(p, 8)
    spots = [slice(0, 4096), slice((1 << 31) - 2048, n)]
    before = [[_np(t[s]) for t in (p, g)] for s in spots]
    o.adamw_step_([p], [g], [m], [v], step=1, exponents=[x], seed=2, **HYPER)
    for s, (p0, g0) in zip(spots, before):
        q, mm, vv = plain.update(p0, g0, 0 * p0, 0 * p0, step=1, **HYPER)
        assert (np.abs(_np(p[s]) - q) <= 2.0 ** -8 * np.abs(q) * 1.001 + 1e-6).all()
        mc, vc, xs, _ = plain.encode(mm, vv, plain.noise_at(np.arange(s.start, s.stop, dtype=np.int64), 2, 0, 1), p0.shape)
        assert np.array_equal(x[s.start // 64:-(-s.stop // 64)].cpu().numpy(), xs)
        for got, want in ((m, mc), (v, vc)):
            assert (got[s].cpu().numpy() == want).mean() > 1 - 1e-3
    total = float(o.grad_norm([g]))
    assert abs(total / n ** 0.5 - 1) < 1e-3


def test_late_rows_of_long_gaps_against_64_bits():
    """Gaps from 1 to 20000 steps.  The power is that of beta rounded to float, so its relative error is d times that rounding's
    (known: e1, e2), with 2 units of 2^-24 for the power and one for the product; the step adds 8 of v' (sums of positive
    terms) and 4 of the parts of m'.  Below 2^-126 either may be zero."""
    o = _optim()
    shape = (4000, 56)
    p, g, m, v, _ = _inputs(shape, torch.float32, 32, 6)
    gaps = torch.cat([torch.arange(1, 2001), torch.randint(1, 20_000, (2000,), generator=torch.Generator().manual_seed(0))])
    stamps = (30_000 - 1 - gaps).to(torch.int32).to(DEV)
    before = [_np(t) for t in (p, g, m, v)]
    o.adamw_step_([p], [g], [m], [v], step=30_000, row_masks=[torch.zeros(4000, dtype=torch.int8, device=DEV)], last_steps=[stamps], **HYPER)
    _, wm, wv = plain.update(*before, step=30_000, missed=gaps.numpy(), **HYPER)
    d = gaps.numpy()[:, None].astype(np.float64)
    e1, e2 = (abs(float(np.float32(b)) / b - 1) for b in HYPER["betas"])
    u = 2.0 ** -24
    _assert_near(_np(v), wv, (11 * u + np.expm1(d * e2)) * wv + 2.0 ** -126, "exp_avg_sq")
    old = 0.9 ** d * np.abs(before[2])
    _assert_near(_np(m), wm, 4 * u * np.abs(before[1]) + (7 * u + np.expm1(d * e1)) * old + 2.0 ** -126, "exp_avg")


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_and_rates_for_each_tensor_as_numbers_and_device_tensors_mixed(bits):
    o = _optim()
    kinds = [torch.float32, torch.bfloat16, torch.float32]
    shapes = [(300, 3), (1000,), (77, 56)]
    counts, rates = [3, 900, 17], [1e-3, 2e-3, 5e-4]
    def run(as_tensor):
        tensors = [_inputs(s, d, bits, 40 + i) for i, (s, d) in enumerate(zip(shapes, kinds))]
        step = [torch.tensor(c, device=DEV) if as_tensor[0][i] else c for i, c in enumerate(counts)]
        lr = [torch.tensor(r, device=DEV) if as_tensor[1][i] else float(np.float32(r)) for i, r in enumerate(rates)]
        o.adamw_step_(*[[t[k] for t in tensors] for k in range(4)], step=step, lr=lr, weight_decay=[0.0, 0.1, 0.01],
                      exponents=[t[4] for t in tensors] if bits == 8 else None, tensor_ids=[5, 1, 9], seed=-3)
        return [x for t in tensors for x in t if x is not None]
    want = run([[0] * 3, [0] * 3])
    for as_tensor in ([[1, 0, 1], [0, 0, 0]], [[0, 0, 0], [0, 1, 1]], [[1, 1, 1], [1, 1, 1]]):
        got = run(as_tensor)
        # (the device's exponentials and logarithms in double precision may differ in their last bit: one unit of a float)
        for a, b in zip(got, want):
            if a.dtype == torch.uint8:
                assert (a != b).float().mean() <= 1e-3
            else:
                assert ((a.float() - b.float()).abs() <= (2.0 ** -7 if a.dtype == torch.bfloat16 else 2.0 ** -22) * b.float().abs() + 1e-9).all()


def test_gradients_that_are_not_contiguous_are_taken_as_they_are():
    o = _optim()
    def run(g):
        p, _, m, v, _ = _inputs((120, 56), torch.float32, 32, 1)
        norm = o.adamw_step_([p], [g], [m], [v], step=2, max_grad_norm=0.1, **HYPER)
        return p, m, v, norm
    base = torch.randn(56, 120, device=DEV)
    wide = torch.randn(120, 70, device=DEV)
    for g in (base.t(), wide[:, 7:63], torch.randn(1, 56, device=DEV).expand(120, 56), torch._neg_view(torch.randn(120, 56, device=DEV))):
        for a, b in zip(run(g), run(g.clone(memory_format=torch.contiguous_format))):
            assert torch.equal(a, b)


def test_copies_of_an_optimiser_keep_what_it_was_told():
    import copy
    import pickle
    o = _optim()
    ps = _parameters(3)
    mask = (torch.arange(1001, device=DEV) % 2).to(torch.int8)
    opt = o.AdamW(ps, state_bits=8, max_grad_norm=0.5, seed=4)
    opt.set_row_mask(ps[0], mask)
    _feed(ps, 1)
    opt.step()
    twins = [copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))]
    _feed(ps, 2)
    opt.step()
    for twin in twins:
        qs = [q for group in twin.param_groups for q in group["params"]]
        _feed(qs, 2)
        twin.step()
        assert torch.equal(twin.last_grad_norm, opt.last_grad_norm) and twin.seed == 4
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg_sq"], twin.state[q]["exp_avg_sq"])


def test_a_refused_state_dict_changes_nothing_and_moments_are_copies():
    o = _optim()
    ps = _parameters(2)
    opt = o.AdamW(ps, state_bits=8)
    _feed(ps, 0)
    opt.step()
    before = {k: t.clone() for k, t in opt.state[ps[1]].items() if isinstance(t, torch.Tensor)}
    saved = opt.state_dict()
    for change in (dict(amsgrad=True), dict(maximize=True)):
        bad = {"state": saved["state"], "param_groups": [{**g, **change} for g in saved["param_groups"]]}
        with pytest.raises(ValueError, match="amsgrad"):
            opt.load_state_dict(bad)
    broken = {"state": {k: dict(s) for k, s in saved["state"].items()}, "param_groups": saved["param_groups"]}
    broken["state"][3].pop("exp_avg_sq")
    with pytest.raises(ValueError, match="no AdamW state"):
        opt.load_state_dict(broken)
    with pytest.raises(ValueError):
        opt.load_state_dict({"state": {}, "param_groups": saved["param_groups"] * 2})
    for name, t in before.items():
        assert torch.equal(opt.state[ps[1]][name], t) and opt.state[ps[1]][name].dtype == t.dtype
    plain32 = o.AdamW(_parameters(2))
    qs = plain32.param_groups[0]["params"]
    _feed(qs, 0)
    plain32.step()
    m, _ = plain32.moments(qs[0])
    m.zero_()
    assert plain32.state[qs[0]]["exp_avg"].any()


def test_reading_moments_into_overlapping_buffers_is_refused():
    o = _optim()
    m, v, x = o.new_moments(torch.zeros(640, device=DEV), 8)
    out = torch.zeros(1000, device=DEV)
    with pytest.raises(RuntimeError, match="overlaps"):
        o.read_moments([m], [v], [x], out=([out[:640]], [out[300:940]]))
    with pytest.raises(RuntimeError, match="overlaps"):
        o.read_moments([m], [v], [x], out=([out[:640]], [out[:640]]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_graph_that_kept_a_parameter_notices_the_step(dtype):
    p = torch.nn.Parameter(torch.randn(100, device=DEV).to(dtype))
    opt = _optim().AdamW([p], lr=1e-2)
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    before = p._version
    opt.step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.backward()
    (p * p).sum().backward()


def test_a_refused_capturable_step_does_not_count():
    p = torch.nn.Parameter(torch.randn(6, 8, device=DEV))
    opt = _optim().AdamW([p], lr=1e-2, capturable=True)
    p.grad = torch.ones_like(p)
    opt.step()
    kept, version = p.detach().clone(), p._version
    p.grad = torch.sparse_coo_tensor([[1], [2]], [1.0], p.shape, device=DEV)
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    assert int(opt.state[p]["step"]) == 1 and torch.equal(p, kept) and p._version == version


def test_steps_from_two_threads_equal_steps_from_one():
    import threading
    optim = _optim()

    def run(seed, out):
        gen = torch.Generator().manual_seed(seed)
        params = [torch.randn(n, generator=gen).to(DEV) for n in (1, 100, 5000, 300000)]
        opt = optim.AdamW(params, lr=1e-2, state_bits=8, max_grad_norm=1.0, seed=seed)
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            for _ in range(20):
                for p in params:
                    p.grad = torch.randn(p.shape, generator=gen).to(DEV)
                opt.step()
            torch.cuda.current_stream().synchronize()
        out[seed] = params

    alone, together = {}, {}
    for seed in (1, 2):
        run(seed, alone)
    threads = [threading.Thread(target=run, args=(seed, together)) for seed in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for seed in (1, 2):
        assert all(torch.equal(a, b) for a, b in zip(alone[seed], together[seed])), seed


@pytest.mark.parametrize("dtype,with_master", TYPES)
@pytest.mark.parametrize("rows,offset", [(97, 1), (601, 0)])
def test_rows_of_every_length_with_8_bits(dtype, with_master, rows, offset):
    """Blocks of 1 to 64 elements, few of them (a quad a lane) and many; their moments read out."""
    o = _optim()
    tensors = [_inputs((rows + n % 3, n), dtype, 8, n, offset) for n in range(1, 65)]
    masters = [_place(t[0].float() * (1 + 2e-3), offset) for t in tensors] if with_master else None
    before = [((_np(masters[i]) if masters else _np(t[0])), *(_np(x) for x in t[1:])) for i, t in enumerate(tensors)]
    for out_dtype in (torch.float32, torch.bfloat16):
        for t, m, v in zip(tensors, *o.read_moments(*([t[k] for t in tensors] for k in (2, 3, 4)), dtype=out_dtype)):
            true_m, true_v = plain.decode(_np(t[2]), _np(t[3]), _np(t[4]), tuple(t[0].shape))
            normal = np.abs(true_m) >= 2.0 ** -126, true_v >= 2.0 ** -126
            assert np.array_equal(_np(m)[normal[0]], true_m[normal[0]]) and np.array_equal(_np(v)[normal[1]], true_v[normal[1]])
            assert (np.abs(_np(m)[~normal[0]]) <= 2.0 ** -125).all() and (_np(v)[~normal[1]] <= 2.0 ** -125).all()
    o.adamw_step_(*[[t[k] for t in tensors] for k in range(4)], step=17, exponents=[t[4] for t in tensors], masters=masters, seed=5, **HYPER)
    for i, t in enumerate(tensors):
        _check_step(before[i], (t[0], t[2], t[3], t[4]), dtype, 17, 8, seed=5, tensor=i, master=masters[i] if masters else None)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("columns", [2, 5, 8, 12, 15, 20, 24, 31, 32, 33, 36, 45, 60, 63])
def test_row_masks_of_more_lengths(bits, columns):
    test_row_masks_leave_rows_alone_and_late_rows_decay(bits, columns, 0.4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1])
def test_norms_of_masked_rows_of_every_length(dtype, offset):
    o = _optim()
    gen = torch.Generator().manual_seed(offset)
    grads = [_place((torch.randn(211 + n, n, generator=gen)).to(dtype), offset) for n in range(1, 65)]
    masks = [(torch.rand(len(g), generator=gen) < 0.3).to(torch.int8).to(DEV) for g in grads]
    true = np.array([np.sqrt((_np(g) ** 2)[_np(mask) == 0].sum()) for g, mask in zip(grads, masks)])
    for g, mask in zip(grads, masks):
        g[mask != 0] = float("nan")
    norm, each = o.grad_norm(grads, masks, per_tensor=True)
    _assert_near(_np(each), true, true * 2.0 ** -24 * 1.001, "each")
    total = np.sqrt((true ** 2).sum())
    assert abs(float(norm) - total) <= total * 2.0 ** -24 * 1.001
