"""The optimizer operators over many tensors (include/gsx_optim.h): AdamW with 32-bit and 8-bit moments, the norm of all gradients, the row selection of
8-bit moments — against their plain forms in 64 bits (adamw_reference.py), at the sizes, views and values where they can go wrong, and their refusals."""
import ctypes
import math
import os

import pytest
import torch

from tests import adamw_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# empty, one value, around the four of a lane, the 128 of a run, the 1024 of a pass and the 2048 of a chunk, and past the 32 tensors of a launch
SIZES = [0, 1, 2, 3, 4, 5, 7, 63, 127, 128, 129, 255, 257, 1000, 1023, 1024, 1025, 2047, 2048, 2049, 4097, 10007] + [11 + 3 * i for i in range(30)]
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def lib():
    l = ctypes.CDLL(os.path.join(ROOT, "gaussian-splatting-cuda_amd", "libgsx.so"))
    l.gsx_last_error.restype = ctypes.c_char_p
    l.gsx_grad_norm_multi_workspace_bytes.restype = ctypes.c_size_t
    return l


class Grad(ctypes.Structure):
    _fields_ = [("grad", ctypes.c_void_p), ("rows", ctypes.c_uint64), ("cols", ctypes.c_uint64), ("ld", ctypes.c_uint64), ("dtype", ctypes.c_uint32)]


class Tensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "exp_avg", "exp_avg_sq", "avg_scale", "rms_scale")] + \
        [(n, ctypes.c_uint64) for n in ("rows", "cols", "ld_param", "ld_grad", "step")] + [(n, ctypes.c_uint32) for n in ("split", "param_dtype", "grad_dtype")] + \
        [(n, ctypes.c_int32) for n in ("hold", "hold_b")] + [(n, ctypes.c_float) for n in ("lr", "lr_b", "weight_decay", "weight_decay_b")]


class Moments(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("avg_in", "rms_in", "avg_scale_in", "rms_scale_in", "avg_out", "rms_out", "avg_scale_out", "rms_scale_out")] + \
        [("cols", ctypes.c_uint64)]


# ---- refusals, without a GPU: everything below is turned down before any launch -----------------------------------------------------------------------
def good(**kw):
    x = Tensor(param=64, grad=64, exp_avg=64, exp_avg_sq=64, avg_scale=64, rms_scale=64, rows=4, cols=8, ld_param=8, ld_grad=8, step=1, lr=1e-3)
    for k, v in kw.items():
        setattr(x, k, v)
    return x


BAD = [dict(param=None), dict(grad=None), dict(exp_avg=None), dict(exp_avg_sq=None), dict(ld_param=7), dict(ld_grad=0), dict(split=9), dict(param_dtype=3),
       dict(grad_dtype=77), dict(step=0), dict(step=2 ** 32), dict(rows=2 ** 40, cols=2 ** 40), dict(cols=2 ** 31 + 1, ld_param=2 ** 32, ld_grad=2 ** 32),
       dict(rows=2 ** 33, cols=2 ** 10, ld_param=2 ** 10, ld_grad=2 ** 10)]


@pytest.mark.parametrize("bad", BAD, ids=[",".join(b) + str(i) for i, b in enumerate(BAD)])
def test_adamw_entry_points_refuse_bad_tensors(bad):
    l, d = lib(), ctypes.c_double
    for f, more in ((l.gsx_adamw_step_multi, ()), (l.gsx_adamw8_step_multi, (ctypes.c_int(1), ctypes.c_uint32(3)))):
        xs = (Tensor * 2)(Tensor(), good(**bad))   # (the first one is empty)
        assert f(ctypes.c_uint32(2), xs, d(0.9), d(0.999), d(1e-8), *more, None, None) == -1, bad
        assert b"adamw_step_multi" in l.gsx_last_error()


def test_adamw_entry_points_refuse_bad_scalars_and_take_empty_lists():
    l, d = lib(), ctypes.c_double
    assert l.gsx_optim_abi_version() == 1   # include/gsx_optim.h GSX_OPTIM_ABI_VERSION
    for f, more in ((l.gsx_adamw_step_multi, ()), (l.gsx_adamw8_step_multi, (ctypes.c_int(0), ctypes.c_uint32(0)))):
        for b1, b2, eps in ((1.0, 0.9, 0.0), (-0.1, 0.9, 0.0), (0.9, 1.0, 0.0), (float("nan"), 0.9, 0.0), (0.9, 0.99, -1e-8), (0.9, 0.99, float("nan"))):
            assert f(ctypes.c_uint32(1), (Tensor * 1)(good()), d(b1), d(b2), d(eps), *more, None, None) == -1
        assert f(ctypes.c_uint32(1), None, d(0.9), d(0.999), d(0.0), *more, None, None) == -1
        assert f(ctypes.c_uint32(0), None, d(0.9), d(0.999), d(0.0), *more, None, None) == 0
        assert f(ctypes.c_uint32(3), (Tensor * 3)(), d(0.9), d(0.999), d(0.0), *more, None, None) == 0   # empty tensors: nothing to launch
    for k in ("avg_scale", "rms_scale"):
        assert l.gsx_adamw8_step_multi(ctypes.c_uint32(1), (Tensor * 1)(good(**{k: None})), d(0.9), d(0.999), d(0.0), 0, ctypes.c_uint32(0), None, None) == -1


def test_norm_and_select_entry_points_refuse_bad_arguments():
    l, d, n32 = lib(), ctypes.c_double, ctypes.c_uint32
    ok = Grad(grad=64, rows=4, cols=1000, ld=1000)
    need = l.gsx_grad_norm_multi_workspace_bytes(n32(1), (Grad * 1)(ok))
    assert need >= 8
    ws = ctypes.c_void_p(64)
    call = lambda xs, norm, control, w, size: l.gsx_grad_norm_multi(n32(len(xs)), xs, d(norm), control, w, ctypes.c_size_t(size), None)  # noqa: E731
    for bad in (dict(grad=None), dict(ld=999), dict(dtype=3), dict(rows=2 ** 40, cols=2 ** 40), dict(cols=2 ** 31 + 1, ld=2 ** 33)):
        x = Grad(grad=64, rows=4, cols=1000, ld=1000)
        for k, v in bad.items():
            setattr(x, k, v)
        assert call((Grad * 1)(x), 1.0, ws, ws, 1 << 20) == -1, bad
        assert l.gsx_grad_norm_multi_workspace_bytes(n32(1), (Grad * 1)(x)) == 0
    for norm in (0.0, -1.0, float("nan")):
        assert call((Grad * 1)(ok), norm, ws, ws, 1 << 20) == -1
    assert call((Grad * 1)(ok), 1.0, None, ws, 1 << 20) == -1 and call((Grad * 1)(ok), 1.0, ws, None, 1 << 20) == -1
    assert call((Grad * 1)(ok), 1.0, ws, ws, need - 8) == -3
    good = dict(avg_in=64, rms_in=64, avg_scale_in=64, rms_scale_in=64, avg_out=64, rms_out=64, avg_scale_out=64, rms_scale_out=64, cols=3)
    sel = lambda x, rin, rout, index: l.gsx_adamw8_select_rows(n32(1), (Moments * 1)(x), ctypes.c_uint64(rin), ctypes.c_uint64(rout), index, None)  # noqa: E731
    for k in good:
        if k != "cols":
            assert sel(Moments(**dict(good, **{k: None})), 5, 5, ws) == -1, k
    assert sel(Moments(**dict(good, cols=2 ** 40)), 2 ** 30, 5, ws) == -1 and sel(Moments(**good), 5, 5, None) == -1
    assert sel(Moments(**good), 5, 0, None) == 0 and sel(Moments(cols=0), 5, 5, ws) == 0


def test_the_operators_refuse_cpu_tensors():
    import gsx  # noqa: F401
    from gsx import ops
    t = torch.zeros(8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adamw_step_multi([t], [t], [t], [t], [0.1], [0.0], 0.9, 0.999, 1e-8, [1])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.grad_norm_multi([t], ops.step_control("cpu"))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adamw8_select_rows([], [], [], [], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="one entry for each"):
        ops.adamw_step_multi([t], [t], [t], [t], [], [0.0], 0.9, 0.999, 1e-8, [1])


# ---- 32-bit moments -----------------------------------------------------------------------------------------------------------------------------------
def inputs(sizes, pt, gt, seed, spread=6.0):
    gen = torch.Generator().manual_seed(seed)
    mag = lambda n: torch.exp2(spread * torch.randn(n, generator=gen, dtype=torch.float64) - 10)  # noqa: E731
    out = []
    for n in sizes:
        r = mag(n)
        m = r * torch.randn(n, generator=gen, dtype=torch.float64)
        g = r * torch.randn(n, generator=gen, dtype=torch.float64) * (torch.rand(n, generator=gen) > 0.2)
        out.append((torch.randn(n, generator=gen).to(pt), g.clamp(-3e4, 3e4).to(gt), m.float(), (r * r).float(), r.float()))
    return out


def check32(p, m, v, x, lr, wd, step, factor=1.0, what="", **kw):
    """Device results (on the CPU, flat) against the plain form of the inputs x = (p, g, m, v, ...)."""
    p0, g, m0, v0 = (t.double() for t in x[:4])
    q, m1, v1, _, pp, mm = ref.adamw(p0, g, m0, v0, lr, wd, step, factor=factor, **kw)
    assert bool(((m.double() - m1).abs() <= 6 * ref.U * mm + 2.0 ** -148).all()), what + " m"
    assert bool(((v.double() - v1).abs() <= 8 * ref.U * v1 + 2.0 ** -147).all()), what + " v"
    half = ref.HALF[p.dtype] * q.abs() + ref.TINY[p.dtype] if p.dtype != torch.float32 else 0.0
    err = (p.double() - q).abs()
    assert bool((err <= pp * (1 + ref.HALF[p.dtype]) + half + 2.0 ** -148).all()), "%s p: %g" % (what, float((err - pp - half).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("pt,gt", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"),
                                   ("bf16", "f16"), ("f16", "bf16")])
def test_adamw_lists_of_odd_sizes(pt, gt):
    from gsx import ops
    x = inputs(SIZES, DT[pt], DT[gt], 1)
    lrs, wds = [1e-3 * (1 + i % 5) for i in range(len(x))], [0.1 * (i % 3) for i in range(len(x))]
    steps = [1 + 37 * i for i in range(len(x))]
    p, g, m, v = ([t[k].cuda() for t in x] for k in range(4))
    ops.adamw_step_multi(p, m, v, g, lrs, wds, 0.9, 0.999, 1e-15, steps)
    for i in range(len(x)):
        check32(p[i].cpu(), m[i].cpu(), v[i].cpu(), x[i], lrs[i], wds[i], steps[i], what="%d values" % SIZES[i])
        assert torch.equal(g[i].cpu(), x[i][1])


@pytest.mark.gpu
def test_adamw_mixed_types_in_one_call_and_betas():
    from gsx import ops
    kinds = [(a, b) for a in DT.values() for b in DT.values()] * 2
    x = [inputs([333 + 7 * i], a, b, i)[0] for i, (a, b) in enumerate(kinds)]
    for b1, b2, eps, step in ((0.0, 0.0, 1e-8, 1), (0.9, 0.95, 1e-6, 2), (0.5, 0.9999, 0.0, 100000), (0.95, 0.999, 1e-15, 2 ** 31)):
        p, g, m, v = ([t[k].clone().cuda() for t in x] for k in range(4))
        ops.adamw_step_multi(p, m, v, g, [2e-3] * len(x), [0.01] * len(x), b1, b2, eps, [step] * len(x))
        for i in range(len(x)):
            nz = (x[i][1] != 0) | (torch.tensor(b2 > 0.0))   # (beta2 = 0, a zero gradient: the formula divides zero by eps)
            got = [t[i].cpu()[nz] for t in (p, m, v)]
            check32(*got, [t[nz] for t in x[i]], 2e-3, 0.01, step, what=str((b1, b2, i)), b1=b1, b2=b2, eps=eps)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("K", [4, 9, 16, 25])
def test_adamw_views_and_column_groups_agree(bits, K):
    """The SH tensor as two row-strided views and as one tensor with two column groups: the plain form's values, and nothing outside the views touched."""
    from gsx import ops
    n = 301
    x = inputs([n * K * 3], torch.float32, torch.float32, K)[0]
    shape = lambda t: t.reshape(n, K, 3)  # noqa: E731
    lr, wd, step = (2.5e-3, 1.25e-4), (0.01, 0.1), 1001
    # one tensor, each group held in turn
    for hold in ((False, False), (False, True), (True, False), (True, True)):
        p, g = shape(x[0].clone()).cuda(), shape(x[1].clone()).cuda()
        split = [(3, lr[1], wd[1]) + hold]
        if bits == 32:
            m, v = shape(x[2].clone()).cuda(), shape(x[3].clone()).cuda()
            ops.adamw_step_multi([p], [m], [v], [g], [lr[0]], [wd[0]], 0.9, 0.999, 1e-15, [step], splits=split)
        else:
            (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
            m, v, sm, sv = shape(mc).cuda(), shape(rc).cuda(), ms.cuda(), rs.cuda()
            ops.adamw8_step_multi([p], [m], [v], [sm], [sv], [g], [lr[0]], [wd[0]], 0.9, 0.999, 1e-15, [step], splits=split, seed=5)
        held = torch.zeros(n, K, 3, dtype=torch.bool)
        held[:, :1], held[:, 1:] = hold
        held = held.flatten()
        rate = torch.full((n, K, 3), lr[1], dtype=torch.float64)
        decay = torch.full((n, K, 3), wd[1], dtype=torch.float64)
        rate[:, :1], decay[:, :1] = lr[0], wd[0]
        rate, decay = rate.flatten(), decay.flatten()
        assert torch.equal(p.cpu().flatten()[held], x[0][held])
        live = ~held
        if bits == 32:
            assert torch.equal(m.cpu().flatten()[held], x[2][held]) and torch.equal(v.cpu().flatten()[held], x[3][held])
            check32(p.cpu().flatten()[live], m.cpu().flatten()[live], v.cpu().flatten()[live], [t[live] for t in x], rate[live], decay[live], step)
        else:
            check8(p.cpu(), m.cpu(), v.cpu(), sm.cpu(), sv.cpu(), x, rate, decay, step, seed=5, ordinal=0, held=held)
    if bits == 8:
        return
    # two views of parameter and gradient; of the gradient or of the parameter alone
    for pv, gv in ((True, True), (True, False), (False, True)):
        big_p, big_g = shape(x[0].clone()).cuda(), shape(x[1].clone()).cuda()
        ps, gs, ms, vs = [], [], [], []
        for part in (slice(0, 1), slice(1, K)):
            ps.append(big_p[:, part] if pv else big_p[:, part].contiguous())
            gs.append(big_g[:, part] if gv else big_g[:, part].contiguous())
            ms.append(shape(x[2])[:, part].contiguous().cuda())
            vs.append(shape(x[3])[:, part].contiguous().cuda())
        ops.adamw_step_multi(ps[:1], ms[:1], vs[:1], gs[:1], lr[:1], wd[:1], 0.9, 0.999, 1e-15, [step])
        if pv:
            assert torch.equal(big_p[:, 1:].cpu(), shape(x[0])[:, 1:])
        ops.adamw_step_multi(ps[1:], ms[1:], vs[1:], gs[1:], lr[1:], wd[1:], 0.9, 0.999, 1e-15, [step])
        for j, part in enumerate((slice(0, 1), slice(1, K))):
            y = [shape(t)[:, part].reshape(-1) for t in x]
            check32(ps[j].cpu().reshape(-1), ms[j].cpu().reshape(-1), vs[j].cpu().reshape(-1), y, lr[j], wd[j], step)
        assert torch.equal(big_g.cpu(), shape(x[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_writes_nothing_outside_its_tensors(bits):
    """Tensors cut from flat buffers at odd places, with a gap of marked values between them."""
    from gsx import ops
    sizes, gap = [1, 5, 127, 130, 1027, 2049, 0, 4099], 3
    x = inputs(sizes, torch.float32, torch.float32, 9)
    total = sum(sizes) + gap * (len(sizes) + 1)
    flat = {k: torch.full((total,), 7.0, device="cuda") for k in ("p", "g", "m", "v")}
    codes = {k: torch.full((total,), 0x55, dtype=torch.uint8, device="cuda") for k in ("m", "v")}
    nr = sum(ref.runs(n) for n in sizes) + gap * (len(sizes) + 1)
    sc = {k: torch.full((nr,), 7.0, device="cuda") for k in ("m", "v")}
    views, at, ar = [], gap, gap
    for n, t in zip(sizes, x):
        view = {k: flat[k][at:at + n] for k in flat}
        view["p"].copy_(t[0]), view["g"].copy_(t[1])
        if bits == 32:
            view["m"].copy_(t[2]), view["v"].copy_(t[3])
        else:
            for k, val, pos in (("m", t[2], False), ("v", t[4], True)):
                c, s = ref.pack(val, pos)
                view[k] = codes[k][at:at + n].view(torch.float8_e4m3fn)
                view[k].copy_(c)
                view["s" + k] = sc[k][ar:ar + ref.runs(n)]
                view["s" + k].copy_(s)
        views.append(view)
        at, ar = at + n + gap, ar + ref.runs(n) + gap
    col = lambda k: [w[k] for w in views]  # noqa: E731
    k = len(sizes)
    if bits == 32:
        ops.adamw_step_multi(col("p"), col("m"), col("v"), col("g"), [1e-2] * k, [0.0] * k, 0.9, 0.999, 1e-15, [3] * k)
        for w, t in zip(views, x):
            check32(w["p"].cpu(), w["m"].cpu(), w["v"].cpu(), t, 1e-2, 0.0, 3)
    else:
        ops.adamw8_step_multi(col("p"), col("m"), col("v"), col("sm"), col("sv"), col("g"), [1e-2] * k, [0.0] * k, 0.9, 0.999, 1e-15, [3] * k, seed=1)
        for i, (w, t) in enumerate(zip(views, x)):
            check8(w["p"].cpu(), w["m"].cpu(), w["v"].cpu(), w["sm"].cpu(), w["sv"].cpu(), t, 1e-2, 0.0, 3, seed=1, ordinal=i)
    mark = torch.ones(total, dtype=torch.bool)
    at = gap
    for n in sizes:
        mark[at:at + n] = False
        at += n + gap
    for name, t in list(flat.items()) if bits == 32 else [("p", flat["p"]), ("g", flat["g"])]:
        assert bool((t.cpu()[mark] == 7.0).all()), name
    if bits == 8:
        mr, ar = torch.ones(nr, dtype=torch.bool), gap
        for n in sizes:
            mr[ar:ar + ref.runs(n)] = False
            ar += ref.runs(n) + gap
        for k in ("m", "v"):
            assert bool((codes[k].cpu()[mark] == 0x55).all()) and bool((sc[k].cpu()[mr] == 7.0).all())


# ---- 8-bit moments ------------------------------------------------------------------------------------------------------------------------------------
def check8(p, m, v, sm, sv, x, lr, wd, step, seed=None, ordinal=0, factor=1.0, held=None, what="", first=0, **kw):
    p0, g = x[0].double().flatten(), x[1].double().flatten()
    n = p0.numel()
    if n == 0:
        return
    (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
    m0, r0 = mc.double().flatten() * ref.spread(ms, n).double(), rc.double().flatten() * ref.spread(rs, n).double()
    q, m1, v1, r1, pp, mm = ref.adamw(p0, g, m0, r0 * r0, lr, wd, step, factor=factor, **kw)
    mtol, rtol = 7 * ref.U * mm + 2.0 ** -148, 6 * ref.U * r1 + 2.0 ** -75   # (one rounding more than in 32 bits: the decoded product; squares of less than 2^-149 are zero)
    if held is not None:
        m1, r1, q = torch.where(held, m0, m1), torch.where(held, r0, r1), torch.where(held, p0, q)
    half = ref.HALF[p.dtype] * q.abs() + ref.TINY[p.dtype] if p.dtype != torch.float32 else 0.0
    fine = torch.isfinite(q)
    err = (p.double().flatten() - q).abs()
    assert torch.equal(torch.isnan(p.flatten()), torch.isnan(q)), what + " p: NaN"
    assert bool((err[fine] <= (pp * (1 + ref.HALF[p.dtype]) + half + 2.0 ** -148)[fine]).all()), "%s p: %g" % (what, float((err - pp)[fine].max()))
    um, ur = ref.draws(seed, step, ordinal, first, n) if seed is not None else (None, None)
    ref.check_codes(m.flatten(), sm, m1, mtol, False, um, what + " m")
    ref.check_codes(v.flatten(), sv, r1, rtol, True, ur, what + " r")


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [None, 0, 2 ** 32 - 1])
@pytest.mark.parametrize("pt,gt", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16"), ("f16", "f16"), ("f32", "f16"),
                                   ("bf16", "f32"), ("f16", "bf16")])
def test_adamw8_lists_of_odd_sizes(pt, gt, seed):
    from gsx import ops
    x = inputs(SIZES, DT[pt], DT[gt], 2)
    k = len(x)
    lrs, wds, steps = [1e-3 * (1 + i % 5) for i in range(k)], [0.1 * (i % 3) for i in range(k)], [1 + 37 * i for i in range(k)]
    p, g = [t[0].clone().cuda() for t in x], [t[1].cuda() for t in x]
    mp, rp = [ref.pack(t[2], False) for t in x], [ref.pack(t[4], True) for t in x]
    m, sm, r, sr = [a.cuda() for a, _ in mp], [b.cuda() for _, b in mp], [a.cuda() for a, _ in rp], [b.cuda() for _, b in rp]
    ops.adamw8_step_multi(p, m, r, sm, sr, g, lrs, wds, 0.9, 0.999, 1e-15, steps, seed=seed)
    for i in range(k):
        check8(p[i].cpu(), m[i].cpu(), r[i].cpu(), sm[i].cpu(), sr[i].cpu(), x[i], lrs[i], wds[i], steps[i], seed=seed, ordinal=i, what="%d values" % SIZES[i])


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [None, 3])
def test_adamw8_infinities_nan_zeros_and_tiny_values(seed):
    """A gradient that is infinite or NaN spoils its own moments alone; runs of zeros stay zeros; values down to the last float32 bit."""
    from gsx import ops
    n = 128 * 9 + 17
    x = list(inputs([n], torch.float32, torch.float32, 4)[0])
    x[1][[5, 130, 131, 400]] = torch.tensor([float("inf"), float("nan"), float("-inf"), float("nan")])
    for t in (1, 2, 3, 4):
        x[t][256:384] = 0.0              # a run of zeros: gradient and moments
    x[2][512:640] = 0.0                  # moments zero, gradients of all sizes
    x[4][512:640] = 0.0
    x[1][512:640] = torch.exp2(torch.linspace(-140, 10, 128))
    x[1][640:768] *= 1e-30               # a run whose scale is at its floor or near it
    x[2][640:768] *= 1e-30
    x[4][640:768] *= 1e-30
    x[1][768] = 1.5e19                   # a square just below the largest number
    p, g = x[0].clone().cuda(), x[1].cuda()
    (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
    m, sm, r, sr = mc.cuda(), ms.cuda(), rc.cuda(), rs.cuda()
    sel = torch.ones(n, dtype=torch.bool)
    ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [g], [1e-3], [0.0], 0.9, 0.999, 1e-8, [7], seed=seed)
    check8(p.cpu(), m.cpu(), r.cpu(), sm.cpu(), sr.cpu(), x, 1e-3, 0.0, 7, seed=seed, eps=1e-8)
    assert bool((m.cpu().float()[256:384] == 0).all()) and bool((r.cpu().float()[256:384] == 0).all()) and torch.equal(p.cpu()[256:384], x[0][256:384])
    assert int((~sel).sum()) == 0
    # a second step without gradients: what was spoilt stays NaN, the neighbours go on
    ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [torch.zeros_like(g)], [1e-3], [0.0], 0.9, 0.999, 1e-8, [8], seed=seed)
    nan = torch.isnan(p.cpu())
    assert nan.nonzero().flatten().tolist() == [5, 130, 131, 400]
    # zero codes are zero moments: what a reset of rows writes
    m.view(torch.uint8)[[5, 130, 131, 400]] = 0
    r.view(torch.uint8)[[5, 130, 131, 400]] = 0
    p[[5, 130, 131, 400]] = 1.0
    ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [torch.zeros_like(g)], [1e-3], [0.0], 0.9, 0.999, 1e-8, [9], seed=seed)
    assert bool(torch.isfinite(p).all()) and p[5] == 1.0


@pytest.mark.gpu
def test_adamw8_stochastic_rounding_keeps_the_mean():
    """A constant gradient for 3 000 steps: the second moment's 8-bit average approaches 1 - beta2^t like the exact one; with rounding to nearest it comes to
    rest far below.  The mean of n values whose spread the rounding's random walk gives: step 1/8 of the value at most, a walk of
    variance below (1/8) / 2 relative to the square over the averaging time -> 0.25 / sqrt(n) a standard error; 5 of them."""
    from gsx import ops
    n = 128 * 64
    ratio = {}
    for seed in (11, None):
        p = torch.zeros(n, device="cuda")
        g = torch.full((n,), 1e-3, device="cuda")
        g[::128] = 8e-3                 # one larger value holds each run's scale
        c = [torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
        s = [torch.zeros(n // 128, device="cuda") for _ in range(2)]
        for t in range(1, 3001):
            ops.adamw8_step_multi([p], [c[0]], [c[1]], [s[0]], [s[1]], [g], [0.0], [0.0], 0.9, 0.999, 1e-8, [t], seed=seed)
        r = c[1].float() * s[1].repeat_interleave(128)
        keep = torch.arange(n, device="cuda") % 128 != 0
        ratio[seed] = float((r[keep] ** 2).mean()) / (1e-6 * (1 - 0.999 ** 3000))
    assert abs(ratio[11] - 1) < 0.03 + 5 * 0.25 / math.sqrt(n), ratio


@pytest.mark.gpu
def test_adamw8_draws_differ_by_step_seed_and_tensor_and_repeat():
    from gsx import ops
    x = inputs([4096], torch.float32, torch.float32, 6)[0]

    def run(seed, step, copies=1):
        p = [x[0].clone().cuda() for _ in range(copies)]
        (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
        m, sm, r, sr = ([t.cuda().clone() for _ in range(copies)] for t in (mc, ms, rc, rs))
        ops.adamw8_step_multi(p, m, r, sm, sr, [x[1].cuda()] * copies, [1e-3] * copies, [0.0] * copies, 0.9, 0.999, 1e-8, [step] * copies, seed=seed)
        return [t.view(torch.uint8).cpu() for t in m]
    a = run(1, 5)[0]
    assert torch.equal(a, run(1, 5)[0])
    assert not torch.equal(a, run(2, 5)[0]) and not torch.equal(a, run(1, 6)[0])
    both = run(1, 5, 2)
    assert torch.equal(a, both[0]) and not torch.equal(both[0], both[1])


# ---- the norm and the control block -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("gt", ["f32", "bf16", "f16", "mixed"])
def test_grad_norm_of_lists(gt):
    from gsx import ops
    kinds = list(DT.values())
    gs = [x[1] for i, n in enumerate(SIZES) for x in inputs([n], torch.float32, DT[gt] if gt != "mixed" else kinds[i % 3], 30 + i)]
    want = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
    c = ops.step_control("cuda", 41)
    dev = [g.cuda() for g in gs]
    ops.grad_norm_multi(dev, c, want / 3)
    a = c.cpu()
    # 64-bit sums of at most 2^17 squares (each exact or rounded once) in any order: 2^17 * 2^-53 of the sum at most, half of it on the root
    assert abs(float(a[0]) - want) <= 2.0 ** -36 * want and abs(float(a[1]) - want / 3 / (want + 1e-6)) < 1e-10
    assert a[2] == 0 and a[3] == 42 and a[4] == 0
    for _ in range(3):   # the same bits every time, and the block is ready for the next call
        ops.grad_norm_multi(dev, c)
    b = c.cpu()
    assert b[0] == a[0] and b[1] == 1.0 and b[3] == 45 and b[4] == 0


@pytest.mark.gpu
def test_grad_norm_special_values_views_and_nothing():
    from gsx import ops
    c = ops.step_control("cuda")
    ops.grad_norm_multi([], c, 1.0)
    assert c.cpu()[:4].tolist() == [0.0, 1.0, 0.0, 1.0]
    ops.grad_norm_multi([torch.zeros(0, device="cuda"), torch.zeros(0, 5, device="cuda")], c, 1.0)
    assert c.cpu()[:4].tolist() == [0.0, 1.0, 0.0, 2.0]
    g = torch.full((5000,), 3e38, device="cuda")
    ops.grad_norm_multi([g], c, 1.0)        # squares beyond 32 bits are none beyond 64
    top = float(torch.tensor(3e38).double()) * math.sqrt(5000)
    assert abs(float(c[0]) / top - 1) < 1e-12 and c[2] == 0 and c[3] == 3
    for bad in (float("inf"), float("-inf"), float("nan")):
        for dt in DT.values():
            h = torch.ones(5000, device="cuda", dtype=dt)
            h[4321] = bad
            ops.grad_norm_multi([torch.ones(7, device="cuda"), h], c, 1.0)
            assert c[2] == 1 and c[3] == 3 and not math.isfinite(float(c[0]))
    sh = torch.randn(300, 16, 3, device="cuda")
    ops.grad_norm_multi([sh[:, 1:], sh[:, :1]], c)
    assert abs(float(c[0]) / float(sh.double().norm()) - 1) < 1e-12 and c[2] == 0 and c[3] == 4
    ops.grad_norm_multi([sh[:, 1:]], c)
    assert abs(float(c[0]) / float(sh[:, 1:].double().norm()) - 1) < 1e-12
    one = torch.tensor(-2.0, device="cuda")   # no dimension at all
    ops.grad_norm_multi([one, one], c)
    assert abs(float(c[0]) - math.sqrt(8)) < 1e-14


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_steps_follow_the_control_block(bits):
    """Norm, then update, as a training step has them: clipped, with the step on the device; an infinite gradient leaves everything as it is."""
    from gsx import ops
    sizes = [1000, 77, 4096, 130]
    x = inputs(sizes, torch.float32, torch.float32, 12)
    k = len(sizes)
    p, g = [t[0].clone().cuda() for t in x], [t[1].clone().cuda() for t in x]
    if bits == 32:
        m, v = [t[2].clone().cuda() for t in x], [t[3].clone().cuda() for t in x]
    else:
        mp, rp = [ref.pack(t[2], False) for t in x], [ref.pack(t[4], True) for t in x]
        m, sm, v, sv = [a.cuda() for a, _ in mp], [b.cuda() for _, b in mp], [a.cuda() for a, _ in rp], [b.cuda() for _, b in rp]
    c = ops.step_control("cuda", 99)

    def step():
        ops.grad_norm_multi(g, c, 0.5)
        if bits == 32:
            ops.adamw_step_multi(p, m, v, g, [1e-3] * k, [0.1] * k, 0.9, 0.999, 1e-15, [], control=c)
        else:
            ops.adamw8_step_multi(p, m, v, sm, sv, g, [1e-3] * k, [0.1] * k, 0.9, 0.999, 1e-15, [], control=c, seed=8)
    bad = g[2][17].clone()
    g[2][17] = float("nan")
    before = [t.clone() for t in p + m + v]
    step()
    for a, b in zip(before, p + m + v):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert c[2] == 1 and c[3] == 99
    g[2][17] = bad
    step()
    norm = math.sqrt(sum(float((t[1].double() ** 2).sum()) for t in x))
    factor = float(torch.tensor(min(1.0, 0.5 / (norm + 1e-6)), dtype=torch.float32))
    assert norm > 0.5 and c[3] == 100
    for i in range(k):
        if bits == 32:
            check32(p[i].cpu(), m[i].cpu(), v[i].cpu(), x[i], 1e-3, 0.1, 100, factor=factor)
        else:
            check8(p[i].cpu(), m[i].cpu(), v[i].cpu(), sm[i].cpu(), sv[i].cpu(), x[i], 1e-3, 0.1, 100, seed=8, ordinal=i, factor=factor)


@pytest.mark.gpu
def test_control_block_with_steps_of_the_call_and_without_a_norm():
    """Explicit steps win over the block's, its factor and skip flag hold all the same; a block that no norm has advanced counts as the first step."""
    from gsx import ops
    x = inputs([3000], torch.float32, torch.float32, 14)[0]
    for c0, steps, step, factor in (([0.0, 0.25, 0.0, 77.0], [5], 5, 0.25), ([0.0, 1.0, 0.0, 0.0], [], 1, 1.0), ([0.0, 0.5, 0.0, 12.0], [], 12, 0.5)):
        c = ops.step_control("cuda")
        c[:4] = torch.tensor(c0, dtype=torch.float64)
        p, m, v = x[0].clone().cuda(), x[2].clone().cuda(), x[3].clone().cuda()
        ops.adamw_step_multi([p], [m], [v], [x[1].cuda()], [1e-2], [0.1], 0.9, 0.999, 1e-15, steps, control=c)
        check32(p.cpu(), m.cpu(), v.cpu(), x, 1e-2, 0.1, step, factor=factor)
    # the device's bias corrections, over the steps where they change most
    for t in (1, 2, 3, 5, 7, 50, 499, 500, 501, 700, 1000, 5000, 30000):
        c = ops.step_control("cuda", t)
        p, m, v = x[0].clone().cuda(), x[2].clone().cuda(), x[3].clone().cuda()
        ops.adamw_step_multi([p], [m], [v], [x[1].cuda()], [1e-2], [0.0], 0.9, 0.999, 1e-15, [], control=c)
        check32(p.cpu(), m.cpu(), v.cpu(), x, 1e-2, 0.0, t, what=str(t))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_replay_like_eager_ones(bits):
    """Norm and update captured on a side stream and replayed, the step advancing on the device, with eager work between the replays."""
    from gsx import ops
    sizes = [2049, 300, 128]
    x = inputs(sizes, torch.float32, torch.float32, 21)
    k = len(sizes)

    def fresh():
        s = dict(p=[t[0].clone().cuda() for t in x], g=[t[1].clone().cuda() for t in x], c=ops.step_control("cuda", 4))
        if bits == 32:
            s.update(m=[t[2].clone().cuda() for t in x], v=[t[3].clone().cuda() for t in x], sm=[], sv=[])
        else:
            mp, rp = [ref.pack(t[2], False) for t in x], [ref.pack(t[4], True) for t in x]
            s.update(m=[a.cuda() for a, _ in mp], sm=[b.cuda() for _, b in mp], v=[a.cuda() for a, _ in rp], sv=[b.cuda() for _, b in rp])
        return s

    def step(s):
        ops.grad_norm_multi(s["g"], s["c"], 0.7)
        if bits == 32:
            ops.adamw_step_multi(s["p"], s["m"], s["v"], s["g"], [1e-2] * k, [0.0] * k, 0.9, 0.999, 1e-15, [], control=s["c"])
        else:
            ops.adamw8_step_multi(s["p"], s["m"], s["v"], s["sm"], s["sv"], s["g"], [1e-2] * k, [0.0] * k, 0.9, 0.999, 1e-15, [], control=s["c"], seed=77)
    def bits_of(s):
        return [t.view(torch.uint8).cpu() for t in s["p"] + s["m"] + s["v"] + s["sm"] + s["sv"]] + [s["c"].cpu()]
    eager, other, captured = fresh(), fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        step(captured)
    for it in range(5):
        for a, b in zip(captured["g"], eager["g"]):   # new gradients in the captured buffers
            new = torch.randn(a.shape, generator=torch.Generator().manual_seed(it)).cuda() * 1e-2
            a.copy_(new), b.copy_(new)
        graph.replay()
        step(eager)
        step(other)
        torch.cuda.synchronize()
        for a, b in zip(bits_of(captured), bits_of(eager)):
            assert torch.equal(a, b), it


@pytest.mark.gpu
def test_operators_on_a_side_stream():
    """The calls run on the current stream: behind a long job there, with the default stream idle."""
    from gsx import ops
    x = inputs([100_003], torch.float32, torch.float32, 33)[0]
    p, m, v = x[0].clone().cuda(), x[2].cuda(), x[3].cuda()
    g, c = torch.empty_like(p), ops.step_control("cuda", 2)
    src = x[1].cuda()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-3
        g.copy_(src)
        ops.grad_norm_multi([g], c, 1e9)
        ops.adamw_step_multi([p], [m], [v], [g], [1e-3], [0.0], 0.9, 0.999, 1e-15, [], control=c)
    st.synchronize()
    check32(p.cpu(), m.cpu(), v.cpu(), x, 1e-3, 0.0, 3)


# ---- rows of 8-bit moments ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows_in,kind", [(500, "permute"), (500, "grow"), (500, "prune"), (500, "repeat"), (1, "permute"), (1, "grow"), (333, "none"), (0, "new"),
                                          (4099, "permute"), (500, "outside")])
def test_select_rows(rows_in, kind):
    from gsx import ops
    gen = torch.Generator().manual_seed(rows_in)
    order = torch.randperm(rows_in, generator=gen)
    index = {"permute": order, "grow": torch.cat([order, torch.full((rows_in // 20 + 1,), -1)]), "prune": order[:rows_in // 3], "none": order[:0],
             "repeat": torch.randint(0, max(rows_in, 1), (2 * rows_in,), generator=gen), "new": torch.full((77,), -1),
             "outside": torch.cat([order, torch.tensor([rows_in, rows_in + 1, 2 ** 62, -2 ** 62, -1])])}[kind]
    shapes = [(3,), (16, 3), (4,), (1,), (15, 3), (25, 3), (7,), (128,), (1500,)]
    state = []
    for i, sh in enumerate(shapes):
        n = rows_in * math.prod(sh)
        x = inputs([n], torch.float32, torch.float32, 50 + i, spread=9.0)[0]
        state.append([t if j >= 2 else t.reshape((rows_in,) + sh) for j, t in enumerate([ref.pack(x[2], False)[0], ref.pack(x[4], True)[0],
                                                                                        ref.pack(x[2], False)[1], ref.pack(x[4], True)[1]])])
    dev = [[s[j].cuda() for s in state] for j in range(4)]
    got = ops.adamw8_select_rows(*dev, index.cuda())
    for i, sh in enumerate(shapes):
        cols = math.prod(sh)
        for j in range(2):
            n = rows_in * cols
            old = (state[i][j].double().reshape(-1) * ref.spread(state[i][j + 2], n).double()).reshape(rows_in, cols)
            inside = (index >= 0) & (index < rows_in)
            want = torch.zeros(index.numel(), cols, dtype=torch.float64)
            want[inside] = old[index[inside]]
            want = want.reshape(-1)
            code, scale = got[j][i].cpu(), got[j + 2][i].cpu()
            assert code.shape == (index.numel(),) + sh and code.dtype == torch.float8_e4m3fn and scale.numel() == ref.runs(want.numel())
            if want.numel():
                ref.check_codes(code.reshape(-1), scale, want, 2 * ref.U * want.abs(), j == 1, None, "%s %s" % (kind, sh))
        assert torch.equal(dev[0][i].view(torch.uint8).cpu(), state[i][0].view(torch.uint8))


@pytest.mark.gpu
def test_select_rows_keeps_nan_and_identity():
    """The rows as they were: the same codes and scales (the largest code of a run that the operators wrote is 448, so the scale is the same number)."""
    from gsx import ops
    x = inputs([700 * 48], torch.float32, torch.float32, 3)[0]
    (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
    mc.view(torch.uint8)[1000] = 0x7F
    rc.view(torch.uint8)[1000] = 0x7F
    m, r = mc.reshape(700, 48).cuda(), rc.reshape(700, 48).cuda()
    a, b, sa, sb = ops.adamw8_select_rows([m], [r], [ms.cuda()], [rs.cuda()], torch.arange(700, device="cuda"))
    for got, want in ((a, mc), (b, rc)):   # (a NaN has no sign that means anything: 0x7F or 0xFF)
        got, nan = got[0].cpu().reshape(-1), torch.isnan(want.float())
        assert torch.equal(torch.isnan(got.float()), nan) and torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])
    # scale * 448 / 448: two roundings
    assert bool(((sa[0].cpu() - ms).abs() <= 2 * ref.U * ms).all()) and bool(((sb[0].cpu() - rs).abs() <= 2 * ref.U * rs).all())


# ---- refusals of the Python entry points ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_python_entry_points_refuse():
    from gsx import ops
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    f8 = torch.float8_e4m3fn
    call = lambda p, m, v, g, lr=1e-3, steps=(1,), **kw: ops.adamw_step_multi([p], [m], [v], [g], [lr], [0.0], 0.9, 0.999, 1e-8, list(steps), **kw)  # noqa: E731
    call(z(4), z(4), z(4), z(4))
    for bad, match in (((z(4).double(), z(4), z(4), z(4)), "float32, bfloat16"), ((z(4), z(4), z(4), z(5)), "its gradient"), ((z(4), z(3), z(4), z(4)), "moments"),
                       ((z(4), z(4, dt=torch.bfloat16), z(4), z(4)), "moments"), ((z(4), z(4), z(4), torch.zeros(4)), "is on cpu"),
                       ((z(4, 2), z(4, 2), z(4, 2), z(4, 1).expand(4, 2)), "neither dense"), ((z(4, 2), z(4, 2), z(4, 2), z(2).expand(4, 2)), "overlap"),
                       ((z(2, 4).t(), z(4, 2), z(4, 2), z(4, 2)), "neither dense")):
        with pytest.raises(RuntimeError, match=match):
            call(*bad)
    p = z(4)
    with pytest.raises(RuntimeError, match="twice"):
        ops.adamw_step_multi([p, p], [z(4)] * 2, [z(4)] * 2, [z(4)] * 2, [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])
    m = z(4)
    for two in (dict(exp_avgs=[m, m], exp_avg_sqs=[z(4), z(4)]), dict(exp_avgs=[m, z(4)], exp_avg_sqs=[z(4), m]), dict(exp_avgs=[z(4), z(4)], exp_avg_sqs=[m, m])):
        with pytest.raises(RuntimeError, match="twice"):
            ops.adamw_step_multi([z(4), z(4)], two["exp_avgs"], two["exp_avg_sqs"], [z(4)] * 2, [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])
    with pytest.raises(RuntimeError, match="count from 1"):
        call(z(4), z(4), z(4), z(4), steps=(0,))
    with pytest.raises(RuntimeError, match="control block"):
        call(z(4), z(4), z(4), z(4), steps=())
    for c in (z(8), z(7, dt=torch.float64), torch.zeros(8, dtype=torch.float64)):
        with pytest.raises(RuntimeError, match="control block"):
            call(z(4), z(4), z(4), z(4), control=c)
    with pytest.raises(RuntimeError, match="split"):
        call(z(4, 3), z(4, 3), z(4, 3), z(4, 3), splits=[(4, 0.1, 0.0, False, False)])
    call8 = lambda m, v, a, b, seed=None: ops.adamw8_step_multi([z(200)], [m], [v], [a], [b], [z(200)], [0.1], [0.0], 0.9, 0.999, 1e-8, [1], seed=seed)  # noqa: E731
    c = z(200, dt=f8)
    call8(c, c.clone(), z(2), z(2))
    for bad in ((z(200), c, z(2), z(2)), (c, z(200, dt=torch.uint8), z(2), z(2)), (c, c, z(1), z(2)), (c, c, z(2), z(2, dt=torch.float64)), (c, c, z(4)[::2], z(2))):
        with pytest.raises(RuntimeError):
            call8(*bad)
    for seed in (-1, 2 ** 32):
        with pytest.raises(RuntimeError, match="seed"):
            call8(c, c.clone(), z(2), z(2), seed=seed)
    with pytest.raises(RuntimeError, match="max_norm"):
        ops.grad_norm_multi([z(4)], ops.step_control("cuda"), 0.0)
    with pytest.raises(RuntimeError, match="gradient 1"):
        ops.grad_norm_multi([z(4), z(4, dt=torch.int32)], ops.step_control("cuda"))
    m = z(5, 3, dt=f8)
    ops.adamw8_select_rows([m], [m], [z(1)], [z(1)], torch.zeros(4, dtype=torch.int64, device="cuda"))
    for bad in (torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int64, device="cuda"), torch.zeros(8, dtype=torch.int64, device="cuda")[::2]):
        with pytest.raises(RuntimeError, match="index"):
            ops.adamw8_select_rows([m], [m], [z(1)], [z(1)], bad)
    with pytest.raises(RuntimeError):
        ops.adamw8_select_rows([m, z(6, 3, dt=f8)], [m, z(6, 3, dt=f8)], [z(1)] * 2, [z(1)] * 2, torch.zeros(4, dtype=torch.int64, device="cuda"))


# ---- past 32 bits ----------------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_past_32_bit_offsets(bits):
    """One tensor of more than 2^32 values with work at its start and its end alone, read back there (58 to 69 GB of the card)."""
    from gsx import ops
    n = 2 ** 32 + 128 * 3 + 21 if bits == 8 else 2 ** 32 + 517
    first = 2 ** 32 - 128 * 4
    pt = torch.bfloat16
    p, g = torch.zeros(n, dtype=pt, device="cuda"), torch.zeros(n, dtype=pt, device="cuda")
    x = inputs([n - first], pt, pt, 2)[0]
    p[first:], g[first:] = x[0].cuda(), x[1].cuda()
    c = ops.step_control("cuda", 9)
    ops.grad_norm_multi([g], c)
    want = float(x[1].double().norm())
    assert abs(float(c[0]) - want) < 1e-10 * want
    if bits == 32:
        m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        m[first:], v[first:] = x[2].cuda(), x[3].cuda()
        ops.adamw_step_multi([p], [m], [v], [g], [1e-2], [0.1], 0.9, 0.999, 1e-15, [10])
        check32(p[first:].cpu(), m[first:].cpu(), v[first:].cpu(), x, 1e-2, 0.1, 10)
        # p = 0 and no moments: zero over eps
        assert float(p[:4096].abs().max()) == 0 and float(m[:4096].abs().max()) == 0
        return
    m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    sm, sr = torch.zeros(ref.runs(n), device="cuda"), torch.zeros(ref.runs(n), device="cuda")
    (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
    m[first:], r[first:], sm[first // 128:], sr[first // 128:] = mc.cuda(), rc.cuda(), ms.cuda(), rs.cuda()
    ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [g], [1e-2], [0.1], 0.9, 0.999, 1e-15, [10], seed=6)
    check8(p[first:].cpu(), m[first:].cpu(), r[first:].cpu(), sm[first // 128:].cpu(), sr[first // 128:].cpu(), x, 1e-2, 0.1, 10, seed=6, first=first)
    # the last rows of it as a model of 21-value rows: offsets past 32 bits in the gather
    rows = n // 21
    whole = rows * 21
    idx = torch.tensor([rows - 1, rows - 2, 0, rows - 3], device="cuda")
    a, _, sa, _ = ops.adamw8_select_rows([m[:whole].view(rows, 21)], [r[:whole].view(rows, 21)], [sm[:ref.runs(whole)]], [sr[:ref.runs(whole)]], idx)
    at = torch.cat([torch.arange(int(i) * 21, int(i) * 21 + 21) for i in idx.cpu()])
    old = m.view(torch.uint8)[at.cuda()].view(torch.float8_e4m3fn).cpu().double() * sm[at.cuda() // 128].cpu().double()
    ref.check_codes(a[0].cpu().reshape(-1), sa[0].cpu(), old, 2 * ref.U * old.abs(), False, None)


# ---- the optimizer of a model --------------------------------------------------------------------------------------------------------------------------------------
def splat_model(n, K, dev, seed=0):
    import gsx  # noqa: F401
    from gsx import rasterizer
    g = torch.Generator().manual_seed(seed)
    m = rasterizer.SplatData(means=torch.randn(n, 3, generator=g).to(dev), sh=torch.randn(n, K, 3, generator=g).to(dev), scaling_raw=torch.randn(n, 3, generator=g).to(dev),
                             rotation_raw=torch.randn(n, 4, generator=g).to(dev), opacity_raw=torch.randn(n, 1, generator=g).to(dev), active_sh_degree=0)
    for p in m.params():
        p.requires_grad_(True)
    return m


def test_fused_adamw_refuses_and_keeps_its_books_without_a_gpu():
    import gsx  # noqa: F401
    from gsx import optim, parameters, rasterizer, trainer
    m = splat_model(50, 16, "cpu")
    mk = lambda **kw: optim.FusedAdamW.for_splat_data(m, **kw)  # noqa: E731
    for bad in (dict(moments=16), dict(weight_decay={"colour": 0.1}), dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            mk(**bad)
    assert [g["lr"] for g in mk().groups] == [g["lr"] for g in optim.FusedAdam.for_splat_data(m).groups]
    opt = mk(moments=8)
    assert opt.begin_fused_sh_step(5) is None
    opt.step(1)                                                     # no gradients: nothing to do
    assert opt.steps == 0
    with pytest.raises(RuntimeError, match="skip_sh"):
        opt.step(1, skip_sh=True)
    for o in (opt, mk(max_grad_norm=1.0)):
        with pytest.raises(RuntimeError, match="row sharding"):
            o.step(1, rows=(0, 10))
    for name in ("means", "sh0", "opacity"):
        opt._moments(name)
    st = opt.state["sh"]
    assert st["exp_avg"].shape == (50, 16, 3) and st["exp_rms"].dtype == torch.float8_e4m3fn and st["avg_scale"].numel() == -(-50 * 48 // 128)
    st["exp_avg"].view(torch.uint8).fill_(0x38)                     # ones
    st["avg_scale"].fill_(2.0)
    opt.reset_state(torch.tensor([3, 7]))
    v = opt.moment_values("shN")[0]
    assert bool((v[[3, 7]] == 0).all()) and bool((v[4:7] == 2).all())
    opt.extend_state(13)
    v = opt.moment_values("sh0")[0]
    assert v.shape == (63, 16, 3) and bool((v[50:] == 0).all()) and bool((v[10:50] == 2).all()) and st["avg_scale"].numel() == -(-63 * 48 // 128)
    assert opt.state["opacity_raw"]["rms_scale"].numel() == 1 and opt.state["means"]["exp_avg"].shape == (63, 3)
    cam = rasterizer.Camera(viewmat=torch.eye(4), K=torch.eye(3), width=16, height=16)
    tr = lambda **kw: trainer.Trainer(m, [cam], [torch.zeros(3, 16, 16)], parameters.OptimizationParameters(), **kw)  # noqa: E731
    for bad in (dict(optimizer="sgd"), dict(optimizer_options={"seed": 3}), dict(optimizer="adamw8", sharded_adam=True),
                dict(optimizer="adamw", optimizer_options={"max_grad_norm": 1.0}, sharded_adam=True)):
        with pytest.raises(ValueError, match="Trainer"):
            tr(**bad)
    assert isinstance(tr(optimizer="adamw8", optimizer_options={"seed": 3}).strategy.optimizer, optim.FusedAdamW)
    assert tr(optimizer="adamw").strategy.optimizer.moments == 32 and type(tr().strategy.optimizer) is optim.FusedAdam


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 9, 16])
@pytest.mark.parametrize("clip", [None, 0.5, float("inf")])
def test_fused_adamw_follows_the_plain_form_over_steps(K, clip):
    """Five steps of a model with 32-bit moments, shN held for the first of them, against the plain form in 64 bits: the parameters' bounds of the steps add up."""
    import gsx  # noqa: F401
    from gsx import optim
    m = splat_model(333, K, "cuda")
    decay = {"shN": 0.3, "opacity": 0.1}
    opt = optim.FusedAdamW.for_splat_data(m, weight_decay=decay, max_grad_norm=clip)
    lr = {g["name"]: g["lr"] for g in opt.groups}
    names = [("means", "means"), ("sh", "sh0"), ("scaling_raw", "scaling"), ("rotation_raw", "rotation"), ("opacity_raw", "opacity")]
    want = {a: [getattr(m, a).detach().cpu().double(), 0.0, 0.0, 0.0] for a, _ in names}
    for t, it in enumerate((1000, 1001, 1002, 1003, 1004), start=1):
        g = {a: torch.randn(getattr(m, a).shape, generator=torch.Generator().manual_seed(100 * t + i)) * 10.0 ** (i - 2) for i, (a, _) in enumerate(names)}
        for a, _ in names:
            getattr(m, a).grad = g[a].cuda()
        norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in g.values()))
        factor = 1.0 if clip is None else float(torch.tensor(min(1.0, clip / (norm + 1e-6)), dtype=torch.float32))
        opt.step(it)
        if clip is not None:
            assert abs(opt.last_norm() - norm) < 1e-10 * norm and not opt.skipped_last()
        for a, n in names:
            p, mm, vv, tol = want[a]
            rate, wd = torch.full(p.shape, lr[n], dtype=torch.float64), torch.full(p.shape, decay.get(n, 0.0), dtype=torch.float64)
            zero = torch.zeros_like(p)
            mm, vv, tol = (zero.clone() if isinstance(x, float) else x for x in (mm, vv, tol))
            live = torch.ones(p.shape, dtype=torch.bool)
            if a == "sh" and K > 1:
                rate[:, 1:], wd[:, 1:] = lr["shN"], 0.3
                live[:, 1:] = it > 1000
            q, m1, v1, _, pp, _ = ref.adamw(p, g[a].double(), mm, vv, rate, wd, t, factor=factor)
            # the moments that a step starts from carry up to 8 roundings each for every step before it: t times the bound of one step covers them
            want[a] = [torch.where(live, q, p), torch.where(live, m1, mm), torch.where(live, v1, vv), torch.where(live, tol + t * pp, tol)]
    for a, _ in names:
        err = (getattr(m, a).detach().cpu().double() - want[a][0]).abs()
        assert bool((err <= want[a][3] + 1e-40).all()), (a, float((err - want[a][3]).max()))
    assert opt.step_count("means") == 5 and (clip is None or float(opt.control[3]) == 5)


@pytest.mark.gpu
def test_fused_adamw8_through_growth_reordering_pruning_and_relocation():
    """The 8-bit moments of a model follow its rows: the values move with them, up to one rounding to nearest for every regrouping."""
    import gsx  # noqa: F401
    from gsx import optim
    n = 777
    m = splat_model(n, 16, "cuda")
    opt = optim.FusedAdamW.for_splat_data(m, moments=8, max_grad_norm=1.0, seed=3)
    for t in range(3):
        for i, p in enumerate(m.params()):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).cuda()
        opt.step(2000 + t)
    before = {k: [x.cpu() for x in opt.moment_values(k)] for k in ("means", "sh0", "opacity")}
    dead = torch.tensor([5, 17, 700], device="cuda")
    opt.reset_state(dead)
    opt.extend_state(39)
    order = torch.randperm(n + 39, generator=torch.Generator().manual_seed(4))
    opt.select_state(order.cuda())
    assert opt.reindex_generation == 1
    for k, (a0, v0) in before.items():
        a, v = (x.cpu() for x in opt.moment_values(k))
        for old, new, root in ((a0, a, False), (v0.sqrt(), v.sqrt(), True)):
            full = torch.zeros((n + 39,) + old.shape[1:])
            full[:n] = old
            full[dead.cpu()] = 0
            full = full[order]
            # a code is off by 2^-4 of the value, or half of the smallest step (2^-10, roots up to 2^-9) of the largest of its run / 448
            top = torch.nn.functional.pad(full.abs().flatten(), (0, -full.numel() % 128)).view(-1, 128).amax(1).repeat_interleave(128)[:full.numel()].view(full.shape)
            assert bool(((new - full).abs() <= (2.0 ** -4 + 1e-6) * full.abs() + 2.0 ** -9 / 448 * top * (1 + 1e-6)).all())
            assert bool((new[full == 0] == 0).all()) and (not root or bool((new[full > 0] > 0).all()))
    p0 = m.means.detach().clone()
    m2 = splat_model(n + 39, 16, "cuda", seed=9)
    opt.model = m2
    for p in m2.params():
        p.grad = torch.zeros_like(p)
    opt.step(2010)
    assert all(bool(torch.isfinite(p).all()) for p in m2.params()) and p0.shape[0] == n
    # a NaN gradient: skipped, on the device
    m2.means.grad[3, 1] = float("nan")
    kept = [p.detach().clone() for p in m2.params()]
    codes = opt.state["sh"]["exp_avg"].view(torch.uint8).clone()
    opt.step(2011)
    assert opt.skipped_last() and float(opt.control[3]) == 4 and all(torch.equal(a, b) for a, b in zip(kept, m2.params())) and torch.equal(codes, opt.state["sh"]["exp_avg"].view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer,options", [("adamw", None), ("adamw", {"max_grad_norm": 0.05, "weight_decay": {"shN": 0.01}}), ("adamw8", {"max_grad_norm": 0.05}), ("adamw8", {"seed": None})])
def test_training_steps_with_adamw(optimizer, options):
    """Training through the trainer, with growth, relocation and reordering on the way: finite parameters, moments of the model's size, and the same run twice gives
    the same moments' sizes and steps."""
    from tests.test_gpu_training import _scene
    import gsx  # noqa: F401
    from gsx import rasterizer, strategy, trainer
    sc, model, cams = _scene("cuda:0")
    bg = sc["background"].to("cuda:0")
    with torch.no_grad():
        images = [rasterizer.rasterize_fused(c, model, bg).image.clone() for c in cams]
    model.means = (model.means + 0.01 * torch.randn(model.means.shape, generator=torch.Generator().manual_seed(1)).cuda()).contiguous()
    n0 = model.means.shape[0]
    params = strategy.OptimizationParameters(iterations=60, start_refine=10, refine_every=20, stop_refine=50, max_cap=3200)
    tr = trainer.Trainer(model, cams, images, params, bg, seed=1, optimizer=optimizer, optimizer_options=options)
    tr.train(60)
    n = model.means.shape[0]
    assert n > n0 and all(bool(torch.isfinite(p).all()) for p in model.params())
    opt = tr.strategy.optimizer
    for name in ("means", "sh0", "scaling", "rotation", "opacity"):
        a, v = opt.moment_values(name)
        assert a.shape[0] == n and bool(torch.isfinite(a).all()) and bool((v >= 0).all()) and float(a.abs().max()) > 0
    if options and "max_grad_norm" in options:
        assert float(opt.control[3]) == opt.steps and opt.last_norm() > 0


# ---- long lists -----------------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("count", [16, 17, 64, 65, 256, 257, 600])
def test_lists_around_the_argument_blocks_sizes(count):
    """One tensor more or less than an argument block holds, and several launches; the draws go by the place in the list, wherever the launch begins."""
    from gsx import ops
    sizes = [(37 * i) % 301 for i in range(count)]
    sizes[0], sizes[-1] = 2500, 1029
    x = inputs(sizes, torch.float32, torch.bfloat16, count)
    lrs, wds = [1e-3 * (1 + i % 7) for i in range(count)], [0.01 * (i % 3) for i in range(count)]
    g, c = [t[1].cuda() for t in x], ops.step_control("cuda", 11)
    ops.grad_norm_multi(g, c)
    want = math.sqrt(sum(float((t[1].double() ** 2).sum()) for t in x))
    assert abs(float(c[0]) - want) <= 2.0 ** -36 * want and c[3] == 12 and c[4] == 0
    p, m, v = [t[0].clone().cuda() for t in x], [t[2].clone().cuda() for t in x], [t[3].clone().cuda() for t in x]
    ops.adamw_step_multi(p, m, v, g, lrs, wds, 0.9, 0.999, 1e-15, [12] * count)
    for i in range(count):
        check32(p[i].cpu(), m[i].cpu(), v[i].cpu(), x[i], lrs[i], wds[i], 12, what=str(i))
    p = [t[0].clone().cuda() for t in x]
    mp, rp = [ref.pack(t[2], False) for t in x], [ref.pack(t[4], True) for t in x]
    m, sm, r, sr = [a.cuda() for a, _ in mp], [b.cuda() for _, b in mp], [a.cuda() for a, _ in rp], [b.cuda() for _, b in rp]
    ops.adamw8_step_multi(p, m, r, sm, sr, g, lrs, wds, 0.9, 0.999, 1e-15, [], control=c, seed=9)
    for i in range(count):
        check8(p[i].cpu(), m[i].cpu(), r[i].cpu(), sm[i].cpu(), sr[i].cpu(), x[i], lrs[i], wds[i], 12, seed=9, ordinal=i, what=str(i))
    rows = 23
    y = [inputs([rows * (1 + i % 50)], torch.float32, torch.float32, i)[0] for i in range(count)]
    mp, rp = [ref.pack(t[2], False) for t in y], [ref.pack(t[4], True) for t in y]
    index = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:17]
    got = ops.adamw8_select_rows([a.cuda().view(rows, -1) for a, _ in mp], [a.cuda().view(rows, -1) for a, _ in rp], [b.cuda() for _, b in mp], [b.cuda() for _, b in rp],
                                 index.cuda())
    for i in range(count):
        old = (mp[i][0].double() * ref.spread(mp[i][1], y[i][2].numel()).double()).view(rows, -1)[index].reshape(-1)
        ref.check_codes(got[0][i].cpu().reshape(-1), got[2][i].cpu(), old, 2 * ref.U * old.abs(), False, None, str(i))


@pytest.mark.gpu
def test_captured_steps_of_a_long_list():
    """A captured launch keeps its whole list (30 KB of arguments): replays on the list's buffers equal eager steps."""
    from gsx import ops
    x = inputs([100 + i for i in range(100)], torch.float32, torch.float32, 5)
    k = len(x)

    def fresh():
        return dict(p=[t[0].clone().cuda() for t in x], g=[t[1].clone().cuda() for t in x], m=[t[2].clone().cuda() for t in x], v=[t[3].clone().cuda() for t in x],
                    c=ops.step_control("cuda", 4))

    def step(s):
        ops.grad_norm_multi(s["g"], s["c"], 0.7)
        ops.adamw_step_multi(s["p"], s["m"], s["v"], s["g"], [1e-2] * k, [0.0] * k, 0.9, 0.999, 1e-15, [], control=s["c"])
    eager, captured = fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for it in range(4):
        graph.replay()
        step(eager)
        torch.cuda.synchronize()
        for name in ("p", "m", "v"):
            assert all(torch.equal(a, b) for a, b in zip(eager[name], captured[name])), (it, name)
        assert torch.equal(eager["c"], captured["c"])


@pytest.mark.gpu
def test_fused_adamw_by_rows_equals_the_whole_step():
    """step(rows=...) on two copies, each with its block of rows: together the bits of one step over all rows (distributed.ShardedAdam's use)."""
    import gsx  # noqa: F401
    from gsx import optim
    n, cut = 401, 170
    models = [splat_model(n, 16, "cuda") for _ in range(3)]
    opts = [optim.FusedAdamW.for_splat_data(m, weight_decay={"shN": 0.2, "rotation": 0.1}) for m in models]
    for t in range(3):
        g = [torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).cuda() for i, p in enumerate(models[0].params())]
        for m in models:
            for p, x in zip(m.params(), g):
                p.grad = x.clone()
        it = 999 + t   # shN held, held, stepped
        opts[0].step(it)
        opts[1].step(it, rows=(0, cut))
        opts[2].step(it, rows=(cut, n))
        for whole, lo, hi in zip(*(m.params() for m in models)):
            assert torch.equal(whole[:cut], lo[:cut]) and torch.equal(whole[cut:], hi[cut:])
    for k, st in opts[0].state.items():
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(st[name][:cut], opts[1].state[k][name][:cut]) and bool((opts[1].state[k][name][cut:] == 0).all())
            assert torch.equal(st[name][cut:], opts[2].state[k][name][cut:])


def test_fused_adamw_has_no_norm_before_a_clipped_step():
    import gsx  # noqa: F401
    from gsx import optim
    for options in ({}, {"max_grad_norm": 1.0}):
        opt = optim.FusedAdamW.for_splat_data(splat_model(5, 1, "cpu"), **options)
        for read in (opt.last_norm, opt.skipped_last):
            with pytest.raises(RuntimeError, match="max_grad_norm"):
                read()
