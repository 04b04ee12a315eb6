"""The optimizer operators over many tensors at once: what is timed, and their plain forms.

Four operators, all on the parameter set of a splat model or on a list of tensors of any sizes:

  adamw    AdamW with moments in 32 bits                    ops.adamw_step_multi
  adamw8   AdamW with moments in 8 bits                     ops.adamw8_step_multi
  norm     norm of all gradients, clip factor, finite check ops.grad_norm_multi
  select   rows of 8-bit moments gathered into a new model  ops.adamw8_select_rows

AdamW, t the step, every tensor with its own learning rate and decay, both moments starting at zero:

  m <- b1 m + (1 - b1) g      v <- b2 v + (1 - b2) g^2      p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

with g the gradient times the clip factor where there is one.  The SH tensor [N, K, 3] of a splat model is one dense tensor of two column groups (the
first coefficient and the others), each with its own rate and decay.

8-bit moments: m and r = sqrt(v) are kept as float8_e4m3fn numbers with one float32 scale for each run of 128 consecutive values of a tensor (the
last run may be shorter): scale = max(|x| of the run) / 448, at least 2^-120; stored is x / scale rounded to the format, to the nearest one (ties to
even) or, with a seed, to one of the two neighbours with the probability that makes the mean right.  An r that is not zero is never stored as zero.
"""
import math
import random

import torch

own = False

BLOCK, TOP, FLOOR = 128, 448.0, 2.0 ** -120
BETA1, BETA2, EPS = 0.9, 0.999, 1e-15
MASK = 0xFFFFFFFF
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- the cases ---------------------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the smallest model of the framework's test scenes (10 000 splats, SH degree 0): launch latency is all there is
        dict(name="adamw-10k", op="adamw", n=10_000, k=1, clip=False),
        # one optimizer step of the 1 M splat benchmark scene behind a global-norm clip, step counter and clip factor on the device
        dict(name="adamw-1m-clip", op="adamw", n=1_000_000, k=16, clip=True),
        # a small network's parameter list in 16 bits: 150 tensors of odd sizes cut from one flat buffer, most of them unaligned
        dict(name="adamw-list-bf16", op="adamw", tensors=150, total=1_500_001, param="bf16", grad="bf16", cut=3, clip=False),
        # the same list with parameters and gradients in 32 bits and the clip
        dict(name="adamw-list-f32-clip", op="adamw", tensors=150, total=1_500_001, param="f32", grad="f32", cut=3, clip=True),
        # 8-bit moments: the smallest model, rounding to nearest
        dict(name="adamw8-10k", op="adamw8", n=10_000, k=1, clip=False, stochastic=False),
        # the benchmark scene with 8-bit moments, clip and stochastic rounding: how a long run uses them
        dict(name="adamw8-1m-clip", op="adamw8", n=1_000_000, k=16, clip=True, stochastic=True),
        # the 5 M splat scene, where the moments are what does not fit beside everything else
        dict(name="adamw8-5m", op="adamw8", n=5_000_000, k=16, clip=False, stochastic=True),
        # 8-bit moments on the list of odd sizes: most runs of 128 are whole, every tensor ends in a short one
        dict(name="adamw8-list", op="adamw8", tensors=150, total=1_500_001, param="f32", grad="bf16", cut=3, clip=False, stochastic=True),
        # the clip's norm alone: the smallest model and the largest
        dict(name="norm-10k", op="norm", n=10_000, k=1),
        dict(name="norm-5m", op="norm", n=5_000_000, k=16),
        # 8-bit moments carried over a growth step of 5 % and the reordering behind it: the random initialisation's 100 000 splats, and 1 M
        dict(name="select-100k", op="select", n=100_000, k=16, grow=0.05),
        dict(name="select-1m", op="select", n=1_000_000, k=16, grow=0.05),
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw", "adamw8", "adamw8", "norm", "select"])
    c = dict(op=op)
    if op != "select" and rng.random() < 0.35:   # a list of tensors
        c.update(tensors=rng.randint(1, 200), total=int(math.exp(rng.uniform(math.log(2e3), math.log(4e7)))) | 1, cut=rng.randrange(1000),
                 param=rng.choice(["f32", "bf16", "f16"]), grad=rng.choice(["f32", "bf16"]))
    else:
        c.update(n=int(math.exp(rng.uniform(math.log(1e3), math.log(3e6)))), k=rng.choice([1, 4, 9, 16, 16, 25]))
        if c["k"] == 25:
            c["n"] = min(c["n"], 1_900_000)
    if op in ("adamw", "adamw8"):
        c["clip"] = rng.random() < 0.5
    if op == "adamw8":
        c["stochastic"] = rng.random() < 0.6
    if op == "select":
        c["grow"] = rng.choice([0.0, 0.05, -0.2])   # reordered only, grown, pruned
    return c


def _cut(case):
    """Sizes of the tensors of a list case, spread over three orders of magnitude; their sum is `total`."""
    r = random.Random(case["cut"])
    w = [math.exp(r.uniform(0.0, math.log(1000.0))) for _ in range(case["tensors"])]
    s = sum(w)
    sizes = [max(1, int(x / s * case["total"])) for x in w]
    sizes[-1] += max(0, case["total"] - sum(sizes))
    return sizes


def _shapes(case):
    n, k = case["n"], case["k"]
    return [(n, 3), (n, k, 3), (n, 3), (n, 4), (n, 1)]   # means, sh, scaling, rotation, opacity


def _elements(case):
    return sum(_cut(case)) if "tensors" in case else sum(math.prod(s) for s in _shapes(case))


def _size(case, which):
    return 4 if case.get(which, "f32") == "f32" else 2


def work(case):
    n = _elements(case)
    runs = sum(-(-s // BLOCK) for s in (_cut(case) if "tensors" in case else [math.prod(s) for s in _shapes(case)]))
    p, g = _size(case, "param"), _size(case, "grad")
    again = g if case.get("clip") else 0   # the norm has to be known before the first parameter changes: the gradients are read twice
    if case["op"] == "adamw":
        return {"bytes": n * (2 * p + g + 16 + again), "flops": 14 * n}
    if case["op"] == "adamw8":
        return {"bytes": n * (2 * p + g + 4 + again) + 16 * runs, "flops": 20 * n}
    if case["op"] == "norm":
        return {"bytes": n * g, "flops": 2 * n}
    rows = case["n"] + int(case["grow"] * case["n"])
    old = min(rows, case["n"])
    return {"bytes": 2 * (old + rows) * (11 + 3 * case["k"]) + 16 * runs + 8 * rows, "flops": 6 * n}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rand = lambda n: torch.randn(n, generator=gen, device=dev)  # noqa: E731
    pt, gt = DTYPES[case.get("param", "f32")], DTYPES[case.get("grad", "f32")]
    s = dict(case=case, step=1200 + seed % 100, seed=seed % 1000, control=torch.zeros(8, dtype=torch.float64, device=dev))
    s["control"][1] = 1.0
    s["control"][3] = float(s["step"])
    if "tensors" in case:
        sizes = _cut(case)
        n = sum(sizes)
        s["sizes"] = sizes
        s["lrs"] = [1e-3 * (1 + i % 3) for i in range(len(sizes))]
        s["wds"] = [0.01 if i % 2 else 0.0 for i in range(len(sizes))]   # matrices decay, biases and norms do not
        s["splits"] = []
        shapes = [(n,)]
    else:
        shapes = _shapes(case)
        s["lrs"] = [1.6e-4, 2.5e-3, 5e-3, 1e-3, 5e-2]
        s["wds"] = [0.0, 0.01, 0.0, 0.0, 0.01]
        # (first column of the second group, its rate, its decay, whether either group is held as it is)
        s["splits"] = [(0, 0.0, 0.0, False, False)] * 5
        if case["k"] > 1:
            s["splits"][1] = (3, 2.5e-3 / 20, 0.02, False, False)
    s["grads"], s["params"], m, r = [], [], [], []
    for shape in shapes:
        n, rows = math.prod(shape), shape[0]
        # gradients of a view: most splats get little, some get nothing, orders of magnitude between the rest
        size = torch.exp2(4.0 * rand(rows) - 18.0) * (torch.rand(rows, generator=gen, device=dev) > 0.2)
        size = size.repeat_interleave(n // rows)
        g = rand(n) * size
        if case["op"] in ("adamw", "adamw8", "norm"):
            s["grads"].append(g.to(gt).reshape(shape))
        if case["op"] in ("adamw", "adamw8"):
            s["params"].append(rand(n).to(pt).reshape(shape))
        if case["op"] != "norm":
            r.append((size + 1e-7) * (0.2 + torch.rand(n, generator=gen, device=dev)))
            m.append(r[-1] * rand(n) * 0.4)
    if case["op"] == "adamw":
        s["m"] = [x.reshape(sh) for x, sh in zip(m, shapes)]
        s["v"] = [(x * x).reshape(sh) for x, sh in zip(r, shapes)]
    elif case["op"] != "norm":
        for name, xs, positive in (("m", m, False), ("r", r, True)):
            cut = s.get("sizes") or [x.numel() for x in xs]
            packed = [_pack(x, cut if "sizes" in s else [x.numel()], positive, None) for x in xs]
            s[name] = [c.reshape(sh) for (c, _), sh in zip(packed, shapes)]
            s[name + "_scale"] = [sc for _, sc in packed]
    if case["op"] == "select":
        n = case["n"]
        rows = n + int(case["grow"] * n)
        order = torch.randperm(max(rows, n), generator=gen, device=dev)[:rows]
        s["index"] = torch.where(order < n, order, -1)   # rows that did not exist get zero moments
    if "sizes" in s:   # the tensors of the list: views of the flat buffers, which are what run() returns
        runs = [-(-k // BLOCK) for k in s["sizes"]]
        for name in ("params", "grads", "m", "v", "r"):
            if s.get(name):
                s[name + "_list"] = list(s[name][0].split(s["sizes"]))
        for name in ("m_scale", "r_scale"):
            if name in s:
                s[name + "_list"] = list(s[name][0].split(runs))
        s["sizes_gpu"] = torch.tensor(s["sizes"], device=dev)
        s["lrs_gpu"] = torch.tensor(s["lrs"], device=dev)
        s["wds_gpu"] = torch.tensor(s["wds"], device=dev)
    return s


MAX_NORM = 1.0


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------
def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E46A9E5) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xF4B0A2DB) & MASK
    return x ^ (x >> 16)


def _key(seed, step, ordinal):
    """Random words of tensor `ordinal` of a call: word(i) = mix(i + key), bits 16..31 for m and 0..15 for r."""
    return _mix((_mix((seed + step * 0x9E3779B9) & MASK) + ordinal * 0xC2A6F0B5) & MASK)


def _round(y, positive, u):
    """y in -448..448 to float8_e4m3fn; u in [0, 1): to the neighbour away from zero where the fraction of the step that is left plus u reaches one."""
    if u is None:
        q = y.to(torch.float8_e4m3fn).float()
    else:
        a = y.abs()
        step = torch.ldexp(torch.ones_like(a), torch.frexp(a).exponent.clamp_min(-5) - 4)
        q = torch.copysign((torch.floor(a / step + u) * step).clamp_max(TOP), y)
    if positive:
        q = torch.where(y > 0, q.clamp_min(2.0 ** -9), q)
    return q.to(torch.float8_e4m3fn)


def _runs(sizes, device):
    """The run of 128 that each value of tensors of these sizes, one behind the other, belongs to."""
    if not torch.is_tensor(sizes):
        sizes = torch.tensor(sizes, device=device)
    runs = (sizes + BLOCK - 1) // BLOCK
    n = int(sizes.sum())
    at = torch.arange(n, device=device)
    which = torch.repeat_interleave(torch.arange(sizes.numel(), device=device), sizes)
    return (runs.cumsum(0) - runs)[which] + (at - (sizes.cumsum(0) - sizes)[which]) // BLOCK, int(runs.sum())


def _scales(x, sizes):
    if len(sizes) == 1:
        top = torch.nn.functional.pad(x.abs(), (0, -x.numel() % BLOCK)).reshape(-1, BLOCK).amax(1)
        return (top / TOP).clamp_min(FLOOR), None
    run, count = _runs(sizes, x.device)
    top = torch.zeros(count, device=x.device, dtype=x.dtype).scatter_reduce(0, run, x.abs(), "amax")
    return (top / TOP).clamp_min(FLOOR), run


def _spread(scale, run, n):
    return scale[run] if run is not None else scale.repeat_interleave(BLOCK)[:n]


def _pack(x, sizes, positive, u):
    scale, run = _scales(x, sizes)
    y = (x / _spread(scale, run, x.numel())).clamp(-TOP, TOP)
    return _round(y, positive, u), scale


def _plain_step(s, p, g, m, v, lr, wd, scale, step):
    """One AdamW update of flat tensors in 32 bits: new p, m, v."""
    g = g.float() * scale
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    denom = v.sqrt() / math.sqrt(1 - BETA2 ** step) + EPS
    p = p.float()
    return p - lr * wd * p - lr / (1 - BETA1 ** step) * m / denom, m, v


def _rates(s, i, device):
    """Learning rate and decay of the values of tensor i (a number, or one of each column of the SH tensor), or of the whole list."""
    if "sizes" in s:
        return s["lrs_gpu"].repeat_interleave(s["sizes_gpu"]), s["wds_gpu"].repeat_interleave(s["sizes_gpu"])
    split, lr_b, wd_b, _, _ = s["splits"][i]
    if not split:
        return s["lrs"][i], s["wds"][i]
    cols = torch.arange(s["case"]["k"] * 3, device=device)
    n = s["case"]["n"]
    return torch.where(cols < split, s["lrs"][i], lr_b).repeat(n), torch.where(cols < split, s["wds"][i], wd_b).repeat(n)


def _plain_norm(s):
    control = s["control"]
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    fine = torch.isfinite(total)
    control[0] = total.sqrt()
    control[1] = (MAX_NORM / (control[0] + 1e-6)).clamp_max(1.0)
    control[2] = (~fine).double()
    control[3] += fine.double()


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "norm":
        _plain_norm(s)
        return s["control"][:4]
    if op == "select":
        return _plain_select(s)
    scale = 1.0
    s["step"] += 1
    if case["clip"]:
        _plain_norm(s)
        scale = s["control"][1].float()
    step = s["step"]
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        lr, wd = _rates(s, i, p.device)
        n = p.numel()
        if op == "adamw":
            q, m, v = _plain_step(s, p.reshape(-1), g.reshape(-1), s["m"][i].reshape(-1), s["v"][i].reshape(-1), lr, wd, scale, step)
            s["m"][i].reshape(-1).copy_(m)
            s["v"][i].reshape(-1).copy_(v)
        else:
            sizes = s.get("sizes") or [n]
            run = _runs(s["sizes_gpu"], p.device)[0] if "sizes" in s else None
            m = s["m"][i].reshape(-1).float() * _spread(s["m_scale"][i], run, n)
            r = s["r"][i].reshape(-1).float() * _spread(s["r_scale"][i], run, n)
            q, m, v = _plain_step(s, p.reshape(-1), g.reshape(-1), m, r * r, lr, wd, scale, step)
            um = ur = None
            if case["stochastic"]:
                if "sizes" in s:
                    keys = torch.tensor([_key(s["seed"], step, k) for k in range(len(sizes))], device=p.device)
                    first = s["sizes_gpu"].cumsum(0) - s["sizes_gpu"]
                    base = (keys - first).repeat_interleave(s["sizes_gpu"])
                else:
                    base = _key(s["seed"], step, i)
                word = _mix((torch.arange(n, device=p.device) + base) & MASK)
                um, ur = (word >> 16).float() / 65536, (word & 0xFFFF).float() / 65536
            for name, x, positive, u in (("m", m, False, um), ("r", v.sqrt(), True, ur)):
                code, sc = _pack(x, sizes, positive, u)
                s[name][i].reshape(-1).copy_(code)
                s[name + "_scale"][i].copy_(sc)
        p.reshape(-1).copy_(q)
    return _outputs(s)


def _plain_select(s):
    out = dict(m=[], r=[], m_scale=[], r_scale=[])
    index = s["index"]
    for name in ("m", "r"):
        for code, scale in zip(s[name], s[name + "_scale"]):
            n = code.numel()
            x = (code.reshape(-1).float() * _spread(scale, None, n)).reshape(code.shape[0], -1)
            x = torch.where((index >= 0)[:, None], x[index.clamp_min(0)], 0.0).reshape(-1)
            c, sc = _pack(x, [x.numel()], name == "r", None)
            out[name].append(c.reshape((index.numel(),) + tuple(code.shape[1:])))
            out[name + "_scale"].append(sc)
    return out


def _outputs(s):
    out = {k: s[k] for k in ("params", "m", "v", "r", "m_scale", "r_scale") if k in s}
    if s["case"]["clip"]:
        out["control"] = s["control"][:4]
    return out


# ---- the framework's calls ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    import gsx  # noqa: F401
    from gsx import ops
    case, op = s["case"], s["case"]["op"]
    a = "_list" if "sizes" in s else ""
    if op == "norm":
        ops.grad_norm_multi(s["grads" + a], s["control"], MAX_NORM)
        return s["control"][:4]
    if op == "select":
        m, r, ms, rs = ops.adamw8_select_rows(s["m"], s["r"], s["m_scale"], s["r_scale"], s["index"])
        return dict(m=m, r=r, m_scale=ms, r_scale=rs)
    s["step"] += 1
    steps, control = [s["step"]] * len(s["lrs"]), None
    if case["clip"]:   # the norm advances the step that the update reads, on the device
        ops.grad_norm_multi(s["grads" + a], s["control"], MAX_NORM)
        steps, control = [], s["control"]
    if op == "adamw":
        ops.adamw_step_multi(s["params" + a], s["m" + a], s["v" + a], s["grads" + a], s["lrs"], s["wds"], BETA1, BETA2, EPS, steps,
                             control=control, splits=s["splits"])
    else:
        ops.adamw8_step_multi(s["params" + a], s["m" + a], s["r" + a], s["m_scale" + a], s["r_scale" + a], s["grads" + a], s["lrs"], s["wds"], BETA1,
                              BETA2, EPS, steps, control=control, splits=s["splits"], seed=s["seed"] if case["stochastic"] else None)
    return _outputs(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------------------------------
def _grid(device):
    """The 127 numbers of the format that are not negative, in order."""
    e = torch.arange(16, dtype=torch.float64, device=device)[:, None]
    f = torch.arange(8, dtype=torch.float64, device=device)[None]
    return torch.where(e > 0, (8 + f) * torch.exp2(e - 10), f * 2.0 ** -9).reshape(-1)[:127]


def _exact_pack(x, sizes, positive, draws):
    """Codes and scales of one flat tensor, or of several of these sizes one behind the other, by search in the table of the format's numbers."""
    grid = _grid(x.device)
    codes, scales, at = [], [], 0
    for size in sizes:
        part = x[at:at + size]
        full = torch.zeros(-(-size // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
        full[:size] = part.abs()
        scale = (full.view(-1, BLOCK).max(1).values / TOP).clamp(min=FLOOR)
        y = (full.view(-1, BLOCK) / scale[:, None]).view(-1)[:size].clamp(max=TOP)
        low = (torch.searchsorted(grid, y, right=True) - 1).clamp(max=125)
        a, b = grid[low], grid[low + 1]
        if draws is None:
            up = (y - a > b - y) | ((y - a == b - y) & (low % 2 == 1))
        else:
            up = (y - a) / (b - a) + draws[at:at + size] >= 1.0
        c = torch.where(up, b, a)
        if positive:
            c = torch.where(y > 0, c.clamp(min=2.0 ** -9), c)
        codes.append(torch.where(part < 0, -c, c))
        scales.append(scale)
        at += size
    return torch.cat(codes), torch.cat(scales)


def _exact_norm(s):
    total = sum(float(g.double().pow(2).sum()) for g in s["grads"])
    norm = math.sqrt(total)
    return norm, min(1.0, MAX_NORM / (norm + 1e-6)), 0.0, float(s["control"][3]) + 1.0


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return torch.tensor(_exact_norm(s), dtype=torch.float64)
    if case["op"] == "select":
        out = dict(m=[], r=[], m_scale=[], r_scale=[])
        for name in ("m", "r"):
            for code, scale in zip(s[name], s[name + "_scale"]):
                cols = code[0].numel()
                at = s["index"][:, None] * cols + torch.arange(cols, device=code.device)
                old = code.reshape(-1).double()[at.clamp(min=0)] * scale.double()[at.clamp(min=0) // BLOCK]
                c, sc = _exact_pack(torch.where(at < 0, 0.0, old).reshape(-1), [at.numel()], name == "r", None)
                out[name].append(c)
                out[name + "_scale"].append(sc)
        return out
    t = s["step"] + 1
    control = _exact_norm(s)
    factor = float(torch.tensor(control[1]).float()) if case["clip"] else 1.0
    out = {k: [] for k in (("params", "m", "v") if case["op"] == "adamw" else ("params", "m", "r", "m_scale", "r_scale"))}
    for i in range(len(s["params"])):
        p, g = s["params"][i].double().reshape(-1), s["grads"][i].double().reshape(-1) * factor
        n, dev = p.numel(), p.device
        sizes = s.get("sizes") or [n]
        lr, wd, split = s["lrs"][i], s["wds"][i], (s["splits"] or [(0,)])[i if s["splits"] else 0]
        if "sizes" in s:
            lr = torch.cat([torch.full((k,), x, dtype=torch.float64, device=dev) for k, x in zip(sizes, s["lrs"])])
            wd = torch.cat([torch.full((k,), x, dtype=torch.float64, device=dev) for k, x in zip(sizes, s["wds"])])
        elif split[0]:
            second = (torch.arange(n, device=dev) % (3 * case["k"])) >= split[0]
            lr, wd = torch.where(second, float(split[1]), lr).double(), torch.where(second, float(split[2]), wd).double()
        if case["op"] == "adamw":
            m, v = s["m"][i].double().reshape(-1), s["v"][i].double().reshape(-1)
        else:
            of = torch.cat([torch.div(torch.arange(k, device=dev), BLOCK, rounding_mode="floor") + b
                            for k, b in zip(sizes, [sum(-(-q // BLOCK) for q in sizes[:j]) for j in range(len(sizes))])])
            m = s["m"][i].double().reshape(-1) * s["m_scale"][i].double()[of]
            v = (s["r"][i].double().reshape(-1) * s["r_scale"][i].double()[of]) ** 2
        m = m * BETA1 + g * (1.0 - BETA1)
        v = v * BETA2 + g * g * (1.0 - BETA2)
        out["params"].append(p * (1.0 - lr * wd) - lr * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)).sqrt() + EPS))
        out["m"].append(m)
        if case["op"] == "adamw":
            out["v"].append(v)
            continue
        um = ur = None
        if case["stochastic"]:
            words = torch.cat([_mix((torch.arange(k, device=dev) + _key(s["seed"], t, j if "sizes" in s else i)) % 2 ** 32) for j, k in enumerate(sizes)])
            um, ur = torch.div(words, 65536, rounding_mode="floor").double() / 65536, (words % 65536).double() / 65536
        out["m"][-1], sc = _exact_pack(m, sizes, False, um)
        out["m_scale"].append(sc)
        c, sc = _exact_pack(v.sqrt(), sizes, True, ur)
        out["r"].append(c)
        out["r_scale"].append(sc)
    if case["clip"]:
        out["control"] = torch.tensor(control, dtype=torch.float64)
    return out
