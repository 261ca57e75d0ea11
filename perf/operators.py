"""Cases, plain forms and exact values of the optimiser's operators: the AdamW step over many tensors (moments in 32 or in
8 bits), the reading of 8-bit moments and the global norm of gradients.

Three layouts of tensors stand for what is trained:

* ``scene``: the two tensors of a point cloud, [points, 56] features and [points, 3] positions, every row stepped;
* ``capacity``: the same two tensors with a fixed capacity, of which a part of the rows holds a point (row mask, stamps);
* ``ragged``: many one-dimensional tensors of odd sizes, the layers of a network, in 16 bits.

8-bit moments: a block (a row of a two-dimensional tensor of at most 64 columns, else 64 consecutive elements) has two
exponent bytes; see ``decode`` and ``encode`` for what the codes stand for, ``noise`` for the bits that round them.
"""
import math

import torch

own = False

LEARNING_RATES = (1e-3, 1e-5)      # features and positions of the trainer
BETAS, EPS, WEIGHT_DECAY = (0.9, 0.999), 1e-8, 1e-2
BLOCK, FEATURES, POSITIONS = 64, 56, 3
M32 = 0xFFFFFFFF


def _case(name, op, layout, dtype, **more):
    case = dict(op=op, layout=layout, dtype=dtype, **more)
    return dict(name=name, **case) if name else case


def listed():
    f32, b16, f16 = "float32", "bfloat16", "float16"
    return [
        # a first scene of a small capture: the step is a few microseconds of memory traffic, its launches count
        _case("adamw32 scene 10k", "step", "scene", f32, points=10_000, bits=32, max_norm=0.0),
        # the size of the headline benchmark's scene
        _case("adamw32 scene 1M", "step", "scene", f32, points=1_000_000, bits=32, max_norm=0.0),
        # a training run with fixed capacity, early on: three tenths of the rows hold a point; clipped
        _case("adamw32 capacity 1.2M clip", "step", "capacity", f32, points=1_200_000, live=0.3, bits=32, max_norm=1.0),
        # a network's many tensors in bfloat16 with a float32 master copy, clipped
        _case("adamw32 ragged bf16 master clip", "step", "ragged", b16, tensors=180, smallest=5, largest=4_000_001,
              bits=32, master=True, max_norm=1.0),
        # the same four uses with the moments in 8 bits; the tensors of the last without a master copy
        _case("adamw8 scene 10k", "step", "scene", f32, points=10_000, bits=8, max_norm=0.0),
        _case("adamw8 scene 1M", "step", "scene", f32, points=1_000_000, bits=8, max_norm=0.0),
        _case("adamw8 capacity 1.2M clip", "step", "capacity", f32, points=1_200_000, live=0.3, bits=8, max_norm=1.0),
        _case("adamw8 ragged bf16 clip", "step", "ragged", b16, tensors=180, smallest=5, largest=4_000_001, bits=8,
              master=False, max_norm=1.0),
        # a large capture: what 8 bits are for
        _case("adamw8 scene 4M clip", "step", "scene", f32, points=4_000_000, bits=8, max_norm=1.0),
        # the norm by itself, as it is logged: two tensors, many tensors, a large scene
        _case("norm scene 10k", "norm", "scene", f32, points=10_000),
        _case("norm ragged f16", "norm", "ragged", f16, tensors=180, smallest=5, largest=4_000_001),
        _case("norm scene 4M", "norm", "scene", f32, points=4_000_000),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["step", "step", "step", "norm"])
    layout = rng.choice(["scene", "capacity", "ragged"] if op == "step" else ["scene", "ragged"])
    more = dict(bits=rng.choice([8, 32]), max_norm=rng.choice([0.0, 0.25, 1.0])) if op == "step" else {}
    if layout == "ragged":
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        if op == "step":
            more["master"] = dtype == "float16" or (dtype == "bfloat16" and rng.random() < 0.5)
        return _case("", op, layout, dtype, tensors=rng.randint(2, 200), smallest=rng.randint(1, 2000),
                     largest=_spread(rng, 4_000, 4_000_000), **more)
    points = _spread(rng, 5_000, 2_500_000)
    if layout == "capacity":
        more["live"] = round(rng.uniform(0.05, 1.0), 2)
    return _case("", op, layout, "float32", points=points, **more)


# ------------------------------------------------------------------------------------------------ layout
def _sizes(case):
    """Element counts of the ragged tensors: a geometric row from the smallest to the largest, odd where it falls so, in an
    order that mixes them."""
    k, low, high = case["tensors"], case["smallest"], case["largest"]
    row = [int(low * (high / low) ** (j / (k - 1))) for j in range(k)]
    return [row[(j * 67) % k] for j in range(k)] if k % 67 else row


def _shapes(case):
    if case["layout"] == "ragged":
        return [(n,) for n in _sizes(case)]
    return [(case["points"], FEATURES), (case["points"], POSITIONS)]


def work(case):
    sizes = [math.prod(s) for s in _shapes(case)]
    n, item = sum(sizes), 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        return {"bytes": n * item + 4 * len(sizes), "flops": 2 * n}
    per = 3 * item if not case.get("master") else 2 * item + 8      # parameter read and written (or master), gradient read
    per += 16 if case["bits"] == 32 else 4 + 4                      # moments read and written; 8 bits: and given out in bfloat16
    stepped = n * case.get("live", 1.0)
    extra = 0.0
    if case["bits"] == 8:
        rows = sum(s[0] if len(s) == 2 else -(-s[0] // BLOCK) for s in _shapes(case))
        extra += 4 * rows * case.get("live", 1.0)
        stepped_read = 2 * (n - stepped) + 4 * (n - stepped)        # the moments of rows without a point are given out too
        extra += stepped_read
    if case["layout"] == "capacity":
        extra += 2 * case["points"] * (1 + 8 * case["live"])        # mask and stamps
    return {"bytes": stepped * per + extra, "flops": 18 * stepped}


def _views(flat, shapes, starts):
    return [flat[a:a + math.prod(s)].view(s) for s, a in zip(shapes, starts)]


def prepare(case, seed):
    """Parameters, gradients and moments as views of flat buffers (every tensor starts at a multiple of 64 elements), with the
    distributions of training: gradients that differ by orders of magnitude between rows, many of them zero."""
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    total = at
    used = torch.zeros(total, dtype=torch.bool, device=dev)
    for a, n in zip(starts, sizes):
        used[a:a + n] = True

    def rand():
        return torch.randn(total, device=dev, generator=gen)

    # one magnitude for 16 elements each, spread over four orders; a fifth of them zero (points that no pixel saw)
    scale = 10.0 ** (torch.rand(total // 16, device=dev, generator=gen) * 4 - 6)
    scale = (scale * (torch.rand(total // 16, device=dev, generator=gen) > 0.2)).repeat_interleave(16)
    if case["dtype"] == "float16":
        scale = scale * 1024.0     # gradients under a loss scale
    grad = (rand() * scale * used).to(dtype)
    blocks = [-(-n // BLOCK) for n in sizes]
    # which tensor 64 elements belong to, and the index there of the first of them
    tensor_of = torch.repeat_interleave(torch.arange(len(sizes), device=dev), torch.tensor(blocks, device=dev))
    first = torch.tensor([a // BLOCK for a in starts], device=dev)
    index_of = (torch.arange(total // BLOCK, device=dev) - first[tensor_of]) * BLOCK
    s = dict(case=case, shapes=shapes, sizes=sizes, starts=starts, total=total, grad=grad,
             grads=_views(grad, shapes, starts), tensor_of=tensor_of, index_of=index_of)
    if case["op"] == "norm":
        return s
    master = rand() * used
    param = master.to(dtype)
    s.update(param=param, params=_views(param, shapes, starts), master=master if case.get("master") else None,
             masters=_views(master, shapes, starts) if case.get("master") else None)
    m = (grad.float() * 0.5 + 0.3 * rand() * scale) * used
    v = (grad.float() * 0.7).square() + 1.5 * m.square() + (scale * 0.2).square() * used
    s["step"] = 1000
    s["masks"] = s["stamps"] = None
    if case["layout"] == "capacity":
        mask = (torch.rand(case["points"], device=dev, generator=gen) >= case["live"]).to(torch.int8)
        # rows that came back to life within the last steps have old moments; the others were stepped last time
        back = torch.randint(0, 40, (case["points"],), device=dev, generator=gen)
        back = torch.where((back < 4) | (mask != 0), back * 3, torch.zeros_like(back))
        s["masks"] = [mask, mask]
        s["stamps"] = [(s["step"] - back).to(torch.int32), (s["step"] - back).to(torch.int32)]
        for g in s["grads"]:
            g[mask != 0] = 0
    # learning rates: one for each tensor
    s["lr"] = [LEARNING_RATES[0]] * len(shapes) if case["layout"] == "ragged" else list(LEARNING_RATES)
    if case["bits"] == 32:
        s.update(m=m, v=v, ms=_views(m, shapes, starts), vs=_views(v, shapes, starts), exponents=None)
        return s
    s["mcode"], s["vcode"] = (torch.zeros(total, dtype=torch.uint8, device=dev) for _ in range(2))
    s["ms"], s["vs"] = _views(s["mcode"], shapes, starts), _views(s["vcode"], shapes, starts)
    s["mvalue"], s["vvalue"] = (torch.zeros(total, dtype=torch.bfloat16, device=dev) for _ in range(2))
    s["mvalues"], s["vvalues"] = _views(s["mvalue"], shapes, starts), _views(s["vvalue"], shapes, starts)
    if case["layout"] == "ragged":
        s["exponent"] = torch.zeros(total // BLOCK, 2, dtype=torch.uint8, device=dev)
        s["exponents"] = list(s["exponent"].split(blocks))
    else:
        s["exponents"] = [torch.zeros(case["points"], 2, dtype=torch.uint8, device=dev) for _ in shapes]
    for mm, vv, mc, vc, x in _matrices(s, m, v, s["mcode"], s["vcode"], exponents=True):
        half = torch.full(mm.shape, 0x7FFF, dtype=torch.int64, device=dev)
        a, b, e = encode(mm, vv, half, half)
        mc.copy_(a)
        vc.copy_(b)
        x.copy_(e)
    return s


def _matrices(s, *flats, exponents=False):
    """Each flat buffer as matrices whose rows are the blocks: one matrix of 64 columns, or features and positions."""
    if s["case"]["layout"] == "ragged":
        rows = [tuple(f.view(-1, BLOCK) for f in flats) + ((s["exponent"],) if exponents else ())]
    else:
        rows = [tuple(f[a:a + math.prod(sh)].view(sh) for f in flats) + ((s["exponents"][k],) if exponents else ())
                for k, (sh, a) in enumerate(zip(s["shapes"], s["starts"]))]
    return rows


# ------------------------------------------------------------------------------------------------ 8-bit moments
def _power(biased):
    """2^(biased - 127) in float32, from the exponent bits (1..254)."""
    return (biased.to(torch.int32) << 23).view(torch.float32)


def _bits(x):
    return x.contiguous().view(torch.int32)


def decode(mcode, vcode, exponent):
    """Values of a matrix of codes [R, L] under its exponents [R, 2].  First moment: sign, 4 exponent bits, 3 of mantissa
    (gradual underflow), times 2^(X - 135).  Second: 0 for code 0, else 2^(c >> 3) (1 + (c & 7) / 8) 2^(X - 158).
    X = 255 stands for NaN."""
    xm, xv = exponent[:, :1].to(torch.int32), exponent[:, 1:].to(torch.int32)
    c = mcode.to(torch.int32)
    a = c & 127
    size = torch.where(a < 8, a.float() * 2.0 ** -9, ((a + 960) << 20).view(torch.float32))
    m = torch.where(c > 127, -size, size) * _power(xm.clamp(9, 254) - 8)
    c = vcode.to(torch.int32)
    v = torch.where(c == 0, torch.zeros_like(m), ((c << 20) + (127 << 23)).view(torch.float32)) * _power(xv.clamp(32, 254) - 31)
    nan = torch.full_like(m, float("nan"))
    return torch.where(xm == 255, nan, m), torch.where(xv == 255, nan, v)


def encode(m, v, rm, rv):
    """Codes and exponents of float32 moments [R, L]; rm, rv (16 bits each) round them."""
    def exponent(largest, carry, low):
        x = (_bits(largest) + carry) >> 23
        return torch.where(torch.isfinite(largest), x.clamp(low, 254), torch.full_like(x, 255))

    xm = exponent(m.abs().amax(1, keepdim=True), 0x1FFFFF, 9)
    xv = exponent(v.amax(1, keepdim=True), 0x0FFFFF, 32)
    t = m.abs() * _power((262 - xm).clamp(8, 254))
    tiny = t < 2.0 ** -6
    u = _bits(torch.where(tiny, t + 2.0 ** -6, t)) + (rm << 4).to(torch.int32) + 8
    a = ((u >> 20) - torch.where(tiny, 968, 960)).clamp(0, 126)
    a = torch.where(m < 0, a + 128, a)
    t = v * _power((285 - xv).clamp(31, 254))
    u = (_bits(t).long() - (127 << 23) + (rv << 4) + 8) >> 20
    b = torch.where(v > 0, u.clamp(1, 255), torch.zeros_like(u))
    a, b = torch.where(xm == 255, 0, a), torch.where(xv == 255, 0, b)
    return a.to(torch.uint8), b.to(torch.uint8), torch.cat([xm, xv], 1).to(torch.uint8)


def _mix(x):
    x = (x ^ (x >> 16)) * 0x6A09E667 & M32
    x = (x ^ (x >> 15)) * 0xBB67AE85 & M32
    return x ^ (x >> 16)


def noise(index, key):
    """The 32 bits that round element `index` (int64 tensor) under a tensor's key: the lower half for the first moment."""
    h = _mix((index >> 2) ^ key)
    turn = 8 * (index & 3)
    return ((h << turn) | (h >> (32 - turn))) & M32


def _key(tensor, step, seed=0):
    """A tensor's key at a step; `tensor` is its place in the list, as an int64 tensor."""
    return _mix((_mix((seed + 0x9E3779B1 * tensor) & M32) + step) & M32)


# ------------------------------------------------------------------------------------------------ plain forms
def _norms(s):
    """Norm of all tensors and of each, added up in 64 bits (zeros lie between the tensors): the sums of 64 elements each, laid
    out with one row for a tensor, then the rows' sums."""
    blocks = s["grad"].double().square().view(-1, BLOCK).sum(1)
    rows = blocks.new_zeros(len(s["sizes"]), -(-max(s["sizes"]) // BLOCK))
    rows[s["tensor_of"], s["index_of"] // BLOCK] = blocks
    each = rows.sum(1)
    return each.sum().sqrt(), each.sqrt()


def _scalars(lr, step):
    b1, b2 = BETAS
    return lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step), 1 - lr * WEIGHT_DECAY


def _update(p, g, m, v, lr, step):
    """One AdamW update in 32 bits."""
    rate, root, keep = _scalars(lr, step)
    m = m + (1 - BETAS[0]) * (g - m)
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    return p * keep - rate * (m / (v.sqrt() * root + EPS)), m, v


def _plain_step(s):
    case, step = s["case"], s["step"]
    out, clip = {}, 1.0
    if case["max_norm"]:
        norm = s["grad"].double().square().sum().sqrt()      # rows without a point have gradients of zero here
        clip = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        out["norm"] = norm.float()
    ragged, eight = case["layout"] == "ragged", case["bits"] == 8
    moments = (s["mcode"], s["vcode"]) if eight else (s["m"], s["v"])
    flats = (s["param"], s["grad"]) + moments + ((s["master"],) if s["master"] is not None else (s["param"],))
    flats += (s["mvalue"], s["vvalue"]) if eight else moments
    parts = _matrices(s, *flats, exponents=eight)
    results = [_plain_part(s, k, part, clip, ragged, eight, step) for k, part in enumerate(parts)]
    out.update(param=s["param"], step=[r for r in results if r is not None])
    out.update(m=s["mvalue"], v=s["vvalue"]) if eight else out.update(m=s["m"], v=s["v"])
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


def _plain_part(s, k, part, clip, ragged, eight, step):
    """The step of one matrix (all the ragged tensors, or one of a scene's two), in place; its stamps."""
    param, grad, mstore, vstore, master, mvalue, vvalue = part[:7]
    p, g = master.float(), grad.float() * clip
    m, v = decode(mstore, vstore, part[7]) if eight else (mstore, vstore)
    old = None
    if s["masks"] is not None:
        live = (s["masks"][k] == 0)[:, None]
        gap = (step - 1 - s["stamps"][k]).clamp(min=0)[:, None].float()
        old, m, v = (p, m, v), m * BETAS[0] ** gap, v * BETAS[1] ** gap
    p, m, v = _update(p, g, m, v, s["lr"][k], step)
    if eight:
        columns = torch.arange(m.shape[1], device=m.device)
        if ragged:
            r = noise(s["index_of"][:, None] + columns, _key(s["tensor_of"], step)[:, None])
        else:
            rows = torch.arange(m.shape[0], device=m.device)
            r = noise(rows[:, None] * m.shape[1] + columns, _key(torch.full((1, 1), k, device=m.device), step))
        mc, vc, x = encode(m, v, r & 0xFFFF, r >> 16)
        if old is not None:
            mc, vc, x = torch.where(live, mc, mstore), torch.where(live, vc, vstore), torch.where(live, x, part[7])
        mstore.copy_(mc)
        vstore.copy_(vc)
        part[7].copy_(x)
        m, v = decode(mc, vc, x)
        mvalue.copy_(m)
        vvalue.copy_(v)
    else:
        if old is not None:
            m, v = torch.where(live, m, old[1]), torch.where(live, v, old[2])
        mstore.copy_(m)
        vstore.copy_(v)
    if old is not None:
        p = torch.where(live, p, old[0])
    master.copy_(p)
    if master is not param:
        param.copy_(p)
    if old is None:
        return None
    s["stamps"][k].copy_(torch.where(live[:, 0], torch.full_like(s["stamps"][k], step), s["stamps"][k]))
    return s["stamps"][k]


def run(s):
    case = s["case"]
    if case["op"] == "norm":
        if own:
            from taichi_3d_gaussian_splatting_amd import optim
            return optim.grad_norm(s["grads"], per_tensor=True)
        total, each = _norms(s)
        return total.float(), each.float()
    s["step"] += 1
    if not own:
        return _plain_step(s)
    from taichi_3d_gaussian_splatting_amd import optim
    norm = optim.adamw_step_(s["params"], s["grads"], s["ms"], s["vs"], step=s["step"], lr=s["lr"], betas=BETAS, eps=EPS,
                             weight_decay=WEIGHT_DECAY, exponents=s["exponents"], masters=s["masters"],
                             row_masks=s["masks"], last_steps=s["stamps"], max_grad_norm=case["max_norm"] or None)
    out = {"param": s["param"], "step": s["stamps"] or []}
    if norm is not None:
        out["norm"] = norm
    if case["bits"] == 8:
        optim.read_moments(s["ms"], s["vs"], s["exponents"], out=(s["mvalues"], s["vvalues"]))
        out.update(m=s["mvalue"], v=s["vvalue"])
    else:
        out.update(m=s["m"], v=s["v"])
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The same outputs from the definition in 64 bits, tensor by tensor, from tables of what the codes stand for."""
    s = prepare(case, seed)
    gs = [g.double() for g in s["grads"]]
    each = torch.stack([torch.linalg.vector_norm(g) for g in gs])
    total = torch.linalg.vector_norm(each)
    if case["op"] == "norm":
        return total, each
    t = s["step"] + 1
    b1, b2 = BETAS
    clip = min(1.0, case["max_norm"] / (float(total) + 1e-6)) if case["max_norm"] else 1.0
    eight = case["bits"] == 8
    dev = s["grad"].device
    mtable = torch.tensor([(c & 7) * 2.0 ** -9 if c < 8 else 2.0 ** ((c >> 3) - 7) * (1 + (c & 7) / 8) for c in range(127)],
                          dtype=torch.float64, device=dev)
    vtable = torch.tensor([0.0] + [2.0 ** (c >> 3) * (1 + (c & 7) / 8) for c in range(1, 256)], dtype=torch.float64, device=dev)
    flat = {n: torch.zeros(s["total"], dtype=torch.float64, device=dev) for n in ("p", "m", "v")}
    stamps = []
    for k, shape in enumerate(s["shapes"]):
        n = s["sizes"][k]
        p = (s["masters"] or s["params"])[k].double()
        if eight:
            rows, width = (shape[0], shape[1]) if len(shape) == 2 else (-(-n // BLOCK), BLOCK)
            where = torch.arange(n, device=dev) // width
            e = s["exponents"][k].double()
            mc, vc = s["ms"][k].reshape(-1).long(), s["vs"][k].reshape(-1).long()
            m = (mtable[(mc % 128).clamp(max=126)] * (1 - 2 * (mc // 128)) * torch.exp2(e[:, 0] - 135)[where]).view(shape)
            v = (vtable[vc] * torch.exp2(e[:, 1] - 158)[where]).view(shape)
        else:
            m, v = s["ms"][k].double(), s["vs"][k].double()
        start, mold, vold = p, m, v
        if s["masks"] is not None:
            late = (t - 1 - s["stamps"][k].double()).clamp(min=0)[:, None]
            m, v = m * torch.pow(torch.tensor(b1, device=dev).double(), late), v * torch.pow(torch.tensor(b2, device=dev).double(), late)
        g = gs[k] * clip
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        lr = s["lr"][k]
        p = p - lr * WEIGHT_DECAY * p - lr * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
        if eight:
            m, v = _exact_rounding(m.reshape(-1), v.reshape(-1), where, rows, k, t, mtable, vtable)
            m, v = m.view(shape), v.view(shape)
        if s["masks"] is not None:
            live = (s["masks"][k] == 0)[:, None]
            p, m, v = torch.where(live, p, start), torch.where(live, m, mold), torch.where(live, v, vold)
            stamps.append(torch.where(live[:, 0], torch.full_like(s["stamps"][k], t), s["stamps"][k]))
        a = s["starts"][k]
        for name, value in (("p", p), ("m", m), ("v", v)):
            flat[name][a:a + n] = value.reshape(-1)
    out = {"param": flat["p"], "step": stamps, "m": flat["m"], "v": flat["v"]}
    if case["max_norm"]:
        out["norm"] = total
    if s["master"] is not None:
        out["master"] = flat["p"]
    return out


def _exact_rounding(m, v, where, rows, tensor, t, mtable, vtable):
    """Moments (float64, one tensor) rounded to the codes' values: to the upper neighbour with the chance that keeps the mean,
    decided by 16 random bits; a second moment over zero stays over zero."""
    word = 1 << 32

    def mixed(x):
        x = ((x ^ (x // 65536)) * 1779033703) % word
        x = ((x ^ (x // 32768)) * 3144134277) % word
        return x ^ (x // 65536)

    i = torch.arange(m.numel(), device=m.device)
    scalar = torch.tensor([(2654435761 * tensor) % word], device=m.device)
    h = mixed((i // 4) ^ mixed((mixed(scalar) + t) % word))
    turned = h * (256 ** (i % 4))                       # a rotation: what leaves at the top comes back below
    left = torch.where(i % 4 == 0, torch.zeros_like(h), h // (256 ** (4 - i % 4)))
    r = (turned % word + left) % word
    chance_m, chance_v = ((r % 65536).double() + 0.5) / 65536, ((r // 65536).double() + 0.5) / 65536

    def power_over(x, top):
        """Of each block, the exponent of 2 under which its largest value is at most `top` times that power."""
        largest = torch.zeros(rows, dtype=torch.float64, device=x.device).scatter_reduce(0, where, x, "amax")
        mantissa, exponent = torch.frexp(largest)       # largest = mantissa * 2^exponent, mantissa in [0.5, 1)
        exponent = exponent - 1 + (2 * mantissa > top)
        return torch.where(largest > 0, exponent.double(), torch.full_like(largest, -1000.0))

    def rounded(x, unit, table, chance):
        y = x / unit
        low = (torch.searchsorted(table, y, right=True) - 1).clamp(0, len(table) - 2)
        share = (y - table[low]) / (table[low + 1] - table[low])
        return table[low + (share + chance >= 1).long()]

    unit = torch.exp2(power_over(m.abs(), 1.75).clamp(min=-118) - 8)[where]
    m = torch.sign(m) * rounded(m.abs(), unit, mtable, chance_m) * unit
    unit = torch.exp2(power_over(v, 1.875).clamp(min=-95) - 31)[where]
    code = rounded(v, unit, vtable, chance_v)
    return m, torch.where((v > 0) & (code < 1.125), torch.full_like(v, 1.125), code) * unit
