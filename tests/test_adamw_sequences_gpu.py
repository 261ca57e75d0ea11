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
