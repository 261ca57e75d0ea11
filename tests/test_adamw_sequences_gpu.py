"""Sequences of calls of optim.AdamW and its operators on the device: masks that come and go, graphs, streams."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _optim():
    from taichi_3d_gaussian_splatting_amd import optim
    return optim


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_mask_that_goes_and_comes_back_owes_no_decay(bits, capturable):
    """Saved under a mask, continued without one and then under one again, against an optimiser that had a mask (of no row) all
    the time.  The moments go through the same operations; the parameters may differ by how p keep - rate change is contracted,
    two roundings a step: 12 steps of 2^-23 relative to the parameter and the change (of 10 lr at most)."""
    o = _optim()
    shapes = [(301, 56), (301, 3), (77, 17)]
    gen = torch.Generator().manual_seed(0)
    first = [torch.randn(s, generator=gen) for s in shapes]
    masks = [(torch.rand(s[0], generator=gen) < 0.4).to(torch.int8).to(DEV) for s in shapes]

    def build(start):
        ps = [torch.nn.Parameter(p.detach().clone().to(DEV)) for p in start]
        return ps, o.AdamW(ps, lr=1e-3, state_bits=bits, capturable=capturable, seed=2)
    ps, opt = build(first)
    for p, mask in zip(ps, masks):
        opt.set_row_mask(p, mask)
    for t in range(6):
        if t == 3:
            for mask in masks:
                mask[::2] = 0
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(DEV)
        opt.step()
    (qs, a), (rs, b) = build(ps), build(ps)
    a.load_state_dict(opt.state_dict())
    b.load_state_dict(opt.state_dict())
    none = [torch.zeros_like(mask) for mask in masks]
    for r, mask in zip(rs, none):
        b.set_row_mask(r, mask)
    if capturable:
        for q in qs:
            q.grad = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="before capturing"):
                a.step()
            keep = qs[0] + 1        # (a graph holds something)
        assert keep.shape == qs[0].shape
    for t in range(12):
        if t == 7:
            for q, mask in zip(qs, none):
                a.set_row_mask(q, mask)
        for q, r in zip(qs, rs):
            q.grad = torch.randn(q.shape, generator=gen).to(DEV)
            r.grad = q.grad.clone()
        a.step()
        b.step()
        assert all(("last_step" in a.state[q]) == (t >= 7) for q in qs)
    for q, r in zip(qs, rs):
        assert ((q - r).abs() <= 12 * 2.0 ** -23 * (r.abs() + 1e-2)).all()
        for name in ("step", "exp_avg", "exp_avg_sq", "exponents", "last_step"):
            x, y = a.state[q].get(name), b.state[r].get(name)
            assert torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y, name


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("columns", [1, 2, 3, 4, 5, 17, 56])
def test_masked_rows_may_be_written_while_the_others_are_stepped(bits, columns):
    """A writer of masked rows on one stream (new points that are laid out, say) and steps of the live rows on another: neither loses
    what it wrote.  Compared with the same work one after the other, bit for bit."""
    o = _optim()
    n, rounds = 1_200_000 // columns, 30
    gen = torch.Generator(device=DEV).manual_seed(columns)
    p, g = (torch.randn(n, columns, device=DEV, generator=gen) for _ in range(2))
    mask = (torch.rand(n, device=DEV, generator=gen) < 0.5).to(torch.int8)
    dead = mask.nonzero()[:, 0]

    def run(together):
        m, v, x = o.new_moments(p, bits)
        q, stamps = p.clone(), torch.zeros(n, dtype=torch.int32, device=DEV)
        written = [t for t in (q, m, v, stamps, x) if t is not None]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for t in range(1, rounds + 1):
            with torch.cuda.stream(streams[0]):
                o.adamw_step_([q], [g], [m], [v], step=t, exponents=None if x is None else [x], row_masks=[mask], last_steps=[stamps])
            if not together:
                torch.cuda.synchronize()
            with torch.cuda.stream(streams[1]):
                for w in written:
                    w[dead] = w[dead] + 1
            if not together:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return written
    for got, want in zip(run(True), run(False)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,masked", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, False)])
def test_finite_moments_at_the_end_of_float_stay_finite_in_8_bits(dtype, masked):
    """Blocks whose largest moment is finite but over the largest code's value under the last exponent: that value is held, as
    the format's tables say; infinite and NaN ones make 255.  With betas of zero the moments are the gradient and its square, which
    gradients of few bits make exact."""
    from tests import adamw_plain as plain
    o = _optim()
    shapes = [(40, 56), (40, 17), (40, 5), (41, 1), (41, 2), (41, 3), (41, 4), (40, 64)] + ([] if masked else [(1000,), (30, 65)])
    gen = torch.Generator().manual_seed(3)
    edge_v = [2.0 ** 63.5, 1.9 * 2.0 ** 63, 1.4 * 2.0 ** 63, 1.36 * 2.0 ** 63]      # squares about 2^127 (1 .. 2), the top code 1.875
    edge_m = [1.99 * 2.0 ** 127, 1.76 * 2.0 ** 127, 1.75 * 2.0 ** 127, -1.9 * 2.0 ** 127]
    over_v = [1.98 * 2.0 ** 63, 1.95 * 2.0 ** 63, 1.93 * 2.0 ** 63]                 # squares of 1.86 .. 1.97 times 2^127
    for edge in (over_v, edge_v[2:], edge_m, [float("inf")], [float("nan")], [edge_v[0], edge_v[3]]):
        grads = []
        for s in shapes:
            g = torch.randn(s, generator=gen)
            at = torch.rand(s, generator=gen) < 0.05
            g = g * abs(edge[0] if np.isfinite(edge[0]) else 1.0) * 0.3
            g[at] = torch.tensor(edge)[torch.randint(len(edge), (int(at.sum()),), generator=gen)]
            # (seven bits of mantissa: exact in bfloat16, squares exact in float32)
            grads.append(g.to(torch.bfloat16).to(dtype).to(DEV))
        params = [torch.zeros(s, dtype=dtype, device=DEV) for s in shapes]
        ms, vs, xs = zip(*[o.new_moments(p, 8) for p in params])
        more = {}
        if masked:
            masks = [torch.zeros(s[0], dtype=torch.int8, device=DEV) for s in shapes]
            for mask in masks:
                mask[1::5] = 1
            more = dict(row_masks=masks, last_steps=[torch.zeros(s[0], dtype=torch.int32, device=DEV) for s in shapes])
        o.adamw_step_(params, grads, ms, vs, step=1, exponents=xs, betas=(0.0, 0.0), lr=0.0, weight_decay=0.0, seed=6, **more)
        for i, s in enumerate(shapes):
            g = grads[i].double().cpu().numpy()
            with np.errstate(over="ignore", invalid="ignore"):
                mc, vc, x, _ = plain.encode(g, g * g, plain.noise(g.size, 6, i, 1), s)
            if masked:
                rows = (more["row_masks"][i] != 0).cpu().numpy()
                mc[rows], vc[rows], x[rows] = 0, 0, 0
            assert np.array_equal(xs[i].cpu().numpy(), x), (edge, s)
            assert np.array_equal(ms[i].cpu().numpy() % 128, mc % 128) and np.array_equal(vs[i].cpu().numpy(), vc), (edge, s)
            m, v = o.read_moments([ms[i]], [vs[i]], [xs[i]])
            assert np.array_equal(torch.isfinite(m[0]).cpu().numpy(), (x[:, 0] != 255)[plain.blocks_of(s)[0]].reshape(s))
            assert np.array_equal(torch.isfinite(v[0]).cpu().numpy(), (x[:, 1] != 255)[plain.blocks_of(s)[0]].reshape(s))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_moments_are_read_in_any_type_whatever_they_are_held_in(bits, dtype):
    o = _optim()
    p = torch.nn.Parameter(torch.zeros(100, 56, device=DEV))
    opt = o.AdamW([p], state_bits=bits)
    p.grad = torch.randn(100, 56, device=DEV)
    opt.step()
    want = [x.to(dtype) for x in opt.moments(p)]
    for got, value in zip(opt.moments(p, dtype), want):
        assert got.dtype == dtype and torch.equal(got, value)


def test_a_graph_that_kept_what_moments_are_read_into_notices():
    o = _optim()
    m, v, x = o.new_moments(torch.zeros(640, device=DEV), 8)
    out = [torch.randn(640, device=DEV) for _ in range(2)]
    w = torch.ones(640, device=DEV, requires_grad=True)
    y = [(w * t).sum() for t in out]
    before = [t._version for t in out + [m, v, x]]
    o.read_moments([m], [v], [x], out=([out[0]], [out[1]]))
    assert [t._version for t in out] == [b + 1 for b in before[:2]] and [t._version for t in (m, v, x)] == before[2:]
    for t in y:
        with pytest.raises(RuntimeError, match="inplace operation"):
            t.backward()
