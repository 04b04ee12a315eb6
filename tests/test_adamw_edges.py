"""The optimizer operators over many tensors (include/gsx_optim.h) at their edges: quotients next to the middle between two numbers, runs of chunks that cross from tensor
to tensor, views with 8-bit moments, what is refused, what autograd is told — against the plain forms in 64 bits (adamw_reference.py)."""
import argparse
import importlib.util
import os
import socket
import sys
import types

import pytest
import torch

from tests import adamw_reference as ref
from tests.test_adamw import DT, check8, check32, inputs

f8 = torch.float8_e4m3fn


def quotients_next_to_the_middle(count, seed):
    """float32 pairs (x, s), 1 <= x / s < 2, whose quotient is (Q + 1/2 +- 1 / (2 S)) 2^-23, S the significand of s: no quotient of two such numbers lies nearer to the
    middle between its neighbours Q and Q + 1.  (X 2^24 = (2 Q + 1) S +- 1, so 2 Q + 1 is -+ the inverse of S modulo 2^24.)  Q + 1 is a multiple of 16: one of
    the two neighbours lies on a border of the stochastic rounding."""
    gen = torch.Generator().manual_seed(seed)
    S = (torch.randint(2 ** 22, 2 ** 23, (64 * count,), generator=gen) * 2 + 1).unique()
    inverse = S.clone()
    for _ in range(5):
        inverse = inverse * ((2 - S * inverse) % 2 ** 24) % 2 ** 24
    X, D = [], []
    for r in (1, -1):
        q = (-r * inverse) % 2 ** 24 + 2 ** 24
        num = q * S + r
        x = num >> 24
        ok = (num % 2 ** 24 == 0) & (x >= S) & (x < 2 ** 24) & ((q + 1) % 32 == 0)
        X.append(x[ok])
        D.append(S[ok])
    X, D = torch.cat(X), torch.cat(D)
    pick = torch.randperm(X.numel(), generator=gen)[:count]
    assert pick.numel() == count
    return X[pick].float() * 2.0 ** -40, D[pick].float() * 2.0 ** -40   # (24 bits each: exact)


def largest_of_scale(s):
    """float32 values t with t * (1 / 448) = s in 32 bits, NaN where there is none."""
    c, out = torch.tensor(1.0 / 448.0, dtype=torch.float32), torch.full_like(s, float("nan"))
    near = (s.double() * 448).float().view(torch.int32)
    for d in range(-2, 3):
        t = (near + d).view(torch.float32)
        out = torch.where(t * c == s, t, out)
    return out


@pytest.mark.gpu
def test_codes_of_quotients_next_to_the_middle():
    """x / scale is rounded to the nearest float32 before it becomes a code: 20 000 of the hardest quotients, each at a place whose draw decides by the last bit of the
    quotient.  beta1 = 0 makes the first moment the gradient itself."""
    import gsx  # noqa: F401
    from gsx import ops
    runs, seed, step = 65536, 5, 9
    n = runs * 128
    x, s = quotients_next_to_the_middle(26000, 1)
    t = largest_of_scale(s)
    x, s, t = x[~t.isnan()][:20000], s[~t.isnan()][:20000], t[~t.isnan()][:20000]
    assert x.numel() == 20000
    y = (x.double() / s.double()).float()        # (a double is never as near to a middle as these are far from it: 2^-25 of a place)
    u = ref.draws(seed, step, 0, 0, n)[0]
    word = (u * 65536).long()
    word[127::128] = -1                          # the last place of a run holds its largest value
    border = (x.double() / s.double() * 2 ** 23).round().long()
    border = torch.where(border % 16 == 0, border, border + 1)     # Q + 1
    need = (-(border % 2 ** 20) % 2 ** 20) // 16                   # the draw that carries from there, and not from Q
    order = word.argsort()
    at = torch.searchsorted(word[order], need).tolist()
    places, used, kept = [], set(), []
    order, need = order.tolist(), need.tolist()
    for k in range(len(need)):
        i = at[k]
        while i < n and int(word[order[i]]) == need[k] and order[i] // 128 in used:
            i += 1
        if i < n and int(word[order[i]]) == need[k]:
            used.add(order[i] // 128)
            places.append(order[i])
            kept.append(k)
    assert len(kept) > 19000
    places, kept = torch.tensor(places), torch.tensor(kept)
    x, s, t, y = x[kept], s[kept], t[kept], y[kept]
    sign = torch.where(torch.arange(len(kept)) % 2 == 0, 1.0, -1.0)
    g = torch.zeros(n)
    g[places] = x * sign
    g[places // 128 * 128 + 127] = t
    m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(f8) for _ in range(2))
    sm, sr = torch.zeros(runs, device="cuda"), torch.zeros(runs, device="cuda")
    ops.adamw8_step_multi([torch.zeros(n, device="cuda")], [m], [r], [sm], [sr], [g.cuda()], [0.0], [0.0], 0.0, 0.999, 1e-8, [step], seed=seed)
    assert torch.equal(sm.cpu()[places // 128], s)
    want = ref.rounded(y.double(), False, u[places]) * sign
    got = m.cpu()[places].double()
    assert torch.equal(got, want.double()), "%d of %d codes" % (int((got != want).sum()), len(kept))


# ---- many chunks, groups, views --------------------------------------------------------------------------------------------------------------------------
def packed(x):
    """The 8-bit state of inputs() on the device: codes and scales of both moments."""
    (mc, ms), (rc, rs) = ref.pack(x[2], False), ref.pack(x[4], True)
    return mc.cuda(), rc.cuda(), ms.cuda(), rs.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("K,seed,hold", [(16, 3, (False, True)), (16, None, (True, False)), (25, 8, (False, False)), (9, 1, (False, True))])
def test_adamw8_of_more_than_4096_chunks(K, seed, hold):
    """From 4 096 chunks on a workgroup takes two: column groups followed from the first to the second, pairs that cross from one tensor into the next (odd counts of
    chunks on every side), ends of tensors in either place of a pair."""
    import gsx  # noqa: F401
    from gsx import ops
    rows = 4_300_001 // (3 * K)
    shapes = [(1500,), (700,), (rows, K, 3), (1024,), (7, K, 3), (3 * 1024 + 5,), (2047,), (999, 4)]
    sizes = [torch.Size(sh).numel() for sh in shapes]
    assert sum(-(-n // 1024) for n in sizes) > 4096
    x = inputs(sizes, torch.float32, torch.float32, K)
    lr, wd, step = [1e-3 * (1 + i) for i in range(len(sizes))], [0.1 * (i % 3) for i in range(len(sizes))], 700
    none = (0, 0.0, 0.0, False, False)
    splits = [(3, 5e-4, 0.3) + hold if len(sh) == 3 else none for sh in shapes]
    p, g = [t[0].clone().reshape(sh).cuda() for t, sh in zip(x, shapes)], [t[1].reshape(sh).cuda() for t, sh in zip(x, shapes)]
    m, r, sm, sr = (list(c) for c in zip(*[packed(t) for t in x]))
    ops.adamw8_step_multi(p, m, r, sm, sr, g, lr, wd, 0.9, 0.999, 1e-15, [step] * len(p), splits=splits, seed=seed)
    for i, sh in enumerate(shapes):
        rate, decay, held = lr[i], wd[i], None
        if splits[i][0]:
            second = torch.arange(sizes[i]) % (3 * K) >= 3
            rate, decay = torch.where(second, 5e-4, lr[i]).double(), torch.where(second, 0.3, wd[i]).double()
            held = torch.where(second, hold[1], hold[0])
            assert torch.equal(p[i].cpu().flatten()[held], x[i][0][held])
        check8(p[i].cpu(), m[i].cpu(), r[i].cpu(), sm[i].cpu(), sr[i].cpu(), x[i], rate, decay, step, seed=seed, ordinal=i, held=held, what=str(sh))


def view_of(t, rows, cols, room, at):
    """t as [rows, cols] between marked columns of a wider tensor on the device: the view, the wider tensor."""
    wide = torch.full((rows, room), 7.0, dtype=t.dtype, device="cuda")
    wide[:, at:at + cols] = t.reshape(rows, cols).cuda()
    return wide[:, at:at + cols], wide


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,split,pt,gt,seed",
                         [shape + kind for shape in [(301, 45, 0), (301, 3, 0), (67, 45, 3), (1, 300, 7), (5, 3001, 2000)]
                          for kind in [("f32", "f32", 4), ("f32", "f32", None), ("bf16", "bf16", 4), ("f16", "f32", 9), ("f32", "f16", 2)]] + [(95003, 45, 9, "f32", "f32", 4)])
@pytest.mark.parametrize("bits", [32, 8])
def test_views_of_rows(bits, rows, cols, split, pt, gt, seed):
    """Row-strided parameters and gradients, each alone and both (the moments are dense), with column groups, one held, and of more than 4 096 chunks: the plain form's values, and
    the columns beside the view as they were."""
    import gsx  # noqa: F401
    from gsx import ops
    n, step = rows * cols, 33
    x = inputs([n], DT[pt], DT[gt], rows + cols)[0]
    splits = [(split, 5e-4, 0.3, False, True)] if split else ()
    second = torch.arange(n) % cols >= split if split else torch.zeros(n, dtype=torch.bool)
    rate, decay = torch.where(second, 5e-4, 2e-3).double(), torch.where(second, 0.3, 0.1).double()
    for pv, gv in ((True, True), (True, False), (False, True)):
        p, pw = view_of(x[0], rows, cols, cols + 3, 1) if pv else (x[0].clone().reshape(rows, cols).cuda(), None)
        g, gw = view_of(x[1], rows, cols, cols + 5, 2) if gv else (x[1].reshape(rows, cols).cuda(), None)
        if bits == 32:
            m, v = x[2].clone().reshape(rows, cols).cuda(), x[3].clone().reshape(rows, cols).cuda()
            ops.adamw_step_multi([p], [m], [v], [g], [2e-3], [0.1], 0.9, 0.999, 1e-15, [step], splits=splits)
            live = ~second
            check32(p.cpu().flatten()[live], m.cpu().flatten()[live], v.cpu().flatten()[live], [t[live] for t in x], rate[live], decay[live], step)
            assert torch.equal(m.cpu().flatten()[second], x[2][second]) and torch.equal(v.cpu().flatten()[second], x[3][second])
        else:
            m, r, sm, sr = packed(x)
            ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [g], [2e-3], [0.1], 0.9, 0.999, 1e-15, [step], splits=splits, seed=seed)
            check8(p.cpu(), m.cpu(), r.cpu(), sm.cpu(), sr.cpu(), x, rate, decay, step, seed=seed, held=second)
        assert torch.equal(p.cpu().flatten()[second], x[0][second]) and torch.equal(g.cpu().flatten(), x[1])
        for w, at in ((pw, 1), (gw, 2)):
            assert w is None or (bool((w[:, :at] == 7).all()) and bool((w[:, at + cols:] == 7).all()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,split", [(3, 70001, 65537), (2, 65536, 65535), (40, 70001, 1), (2, 1 << 21, 1 << 20)])
@pytest.mark.parametrize("bits", [32, 8])
def test_column_groups_of_long_rows(bits, rows, cols, split):
    """Rows of more than 65 535 values, whose columns are found by another quotient."""
    import gsx  # noqa: F401
    from gsx import ops
    n = rows * cols
    x = inputs([n], torch.float32, torch.float32, cols % 1000)[0]
    second = torch.arange(n) % cols >= split
    rate, decay = torch.where(second, 5e-4, 2e-3).double(), torch.where(second, 0.3, 0.1).double()
    p, g = x[0].clone().reshape(rows, cols).cuda(), x[1].reshape(rows, cols).cuda()
    splits = [(split, 5e-4, 0.3, False, False)]
    if bits == 32:
        m, v = x[2].clone().cuda(), x[3].clone().cuda()
        ops.adamw_step_multi([p], [m], [v], [g], [2e-3], [0.1], 0.9, 0.999, 1e-15, [50], splits=splits)
        check32(p.cpu().flatten(), m.cpu(), v.cpu(), x, rate, decay, 50)
    else:
        m, r, sm, sr = packed(x)
        ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [g], [2e-3], [0.1], 0.9, 0.999, 1e-15, [50], splits=splits, seed=2)
        check8(p.cpu(), m.cpu(), r.cpu(), sm.cpu(), sr.cpu(), x, rate, decay, 50, seed=2)


@pytest.mark.gpu
def test_adamw_of_more_than_two_to_the_23_chunks():
    """Beyond 2^23 chunks (2^33 values, 103 GB here) a workgroup of the 32-bit update takes two of them as well; two column groups in rows of 48."""
    import gsx  # noqa: F401
    from gsx import ops
    rows = 2 ** 33 // 48 + 1000
    assert -(-rows * 48 // 1024) > 2 ** 23
    p, g = (torch.zeros(rows, 48, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(rows, 48, device="cuda") for _ in range(2))
    spots = [0, rows // 3, 2 ** 32 // 48 - 30, rows - 60]
    x = inputs([60 * 48 * len(spots)], torch.bfloat16, torch.bfloat16, 3)[0]
    parts = [[t[60 * 48 * i:60 * 48 * (i + 1)] for t in x] for i in range(len(spots))]
    for at, part in zip(spots, parts):
        for dst, src in ((p, part[0]), (g, part[1]), (m, part[2]), (v, part[3])):
            dst[at:at + 60] = src.reshape(60, 48).cuda()
    ops.adamw_step_multi([p], [m], [v], [g], [2e-3], [0.1], 0.9, 0.999, 1e-8, [50], splits=[(3, 5e-4, 0.3, False, False)])
    second = torch.arange(60 * 48) % 48 >= 3
    rate, decay = torch.where(second, 5e-4, 2e-3).double(), torch.where(second, 0.3, 0.1).double()
    for at, part in zip(spots, parts):
        check32(*[t[at:at + 60].cpu().flatten() for t in (p, m, v)], part, rate, decay, 50, eps=1e-8)
    for a, b in zip(spots, spots[1:]):      # between the places: zeros stay zeros
        at = (a + b) // 2
        assert float(p[at:at + 100].abs().max()) == 0 and float(m[at:at + 100].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("gt", ["f32", "bf16", "mixed"])
def test_norm_of_more_than_2048_chunks(gt):
    """Chunks of 4 096 values; beyond 2 048 of them a workgroup takes several, here of one tensor, across ends of tensors, and of views."""
    import gsx  # noqa: F401
    from gsx import ops
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    sizes = [9_000_003, 5, 4097, 8191, 1, 0, 12_289, 4096, 7_000_001]
    gs = [inputs([n], torch.float32, DT[gt] if gt != "mixed" else kinds[i % 3], 60 + i)[0][1] for i, n in enumerate(sizes)]
    want = sum(float((g.double() ** 2).sum()) for g in gs)
    dev = [g.cuda() for g in gs]
    rows = 4_400_000 // 45
    sh = torch.randn(rows, 16, 3, generator=torch.Generator().manual_seed(1)).to(gs[0].dtype)
    dev.append(sh.cuda()[:, 1:])
    want = (want + float((sh[:, 1:].double() ** 2).sum())) ** 0.5
    c = ops.step_control("cuda")
    bits = []
    for _ in range(3):
        ops.grad_norm_multi(dev, c)
        bits.append(c.cpu()[0])
    # 64-bit sums of at most 2^25 squares in any order: 2^25 * 2^-53 of the sum at most, half of it on the root, the same again for the sums here
    assert abs(float(bits[0]) - want) <= 2.0 ** -27 * want and bits[0] == bits[1] == bits[2] and c[3] == 3 and c[4] == 0
    views = [sh.cuda()[:, :1], sh.cuda()[:, 1:]]
    ops.grad_norm_multi(views, c)
    assert abs(float(c[0]) / float(sh.double().norm()) - 1) < 2.0 ** -27


# ---- what is refused -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_scale_twice_in_the_lists_is_refused():
    """One scale tensor for both moments, for two parameters, or in the place of another tensor: the runs would overwrite each other's."""
    import gsx  # noqa: F401
    from gsx import ops
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    p, m, r = [z(200), z(200)], [z(200, dt=f8), z(200, dt=f8)], [z(200, dt=f8), z(200, dt=f8)]
    call = lambda sm, sr, p=p: ops.adamw8_step_multi(p, m, r, sm, sr, [z(200)] * 2, [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])  # noqa: E731
    a, b, c, d = (z(2) for _ in range(4))
    call([a, b], [c, d])
    for sm, sr in (([a, b], [a, d]), ([a, a], [c, d]), ([a, b], [c, c]), ([a, b], [c, a])):
        with pytest.raises(RuntimeError, match="twice"):
            call(sm, sr)
    with pytest.raises(RuntimeError, match="twice"):
        call([p[1][:2], b], [c, d])
    e = z(0)                                     # (empty tensors have no memory to share)
    ops.adamw8_step_multi([e, e], [z(0, dt=f8)] * 2, [z(0, dt=f8)] * 2, [e, e], [e, e], [e, e], [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 2, 40])
def test_a_tensor_twice_is_found_wherever_it_is(count):
    """Lists cut one behind the other from flat buffers (seen to be apart by their order) and in any other order (by a table): taken as they are, refused with any
    tensor of theirs in the place of another."""
    import gsx  # noqa: F401
    from gsx import ops
    gen = torch.Generator().manual_seed(count)

    def lists(ascending):
        flat = [torch.zeros(200 * count, device="cuda"), torch.zeros(200 * count, dtype=f8, device="cuda"), torch.zeros(200 * count, dtype=f8, device="cuda"),
                torch.zeros(2 * count, device="cuda"), torch.zeros(2 * count, device="cuda")]
        cut = [list(t.split(t.numel() // count)) for t in flat]
        if not ascending:
            cut = [[c[i] for i in torch.randperm(count, generator=gen).tolist()] for c in cut]
        return cut
    def call(x):
        ops.adamw8_step_multi(*x[:3], x[3], x[4], [torch.zeros(200, device="cuda")] * count, [0.1] * count, [0.0] * count, 0.9, 0.999, 1e-8, [1] * count)
    for ascending in (True, False):
        call(lists(ascending))
        for a in range(5):
            for b in range(5):
                i, j = (int(k) for k in torch.randint(0, count, (2,), generator=gen))
                if (a in (1, 2)) != (b in (1, 2)) or (a == 0) != (b == 0) or (a == b and i == j):
                    continue   # (of another type or size: refused for that)
                x = lists(ascending)
                x[a][i] = x[b][j]
                with pytest.raises(RuntimeError, match="twice"):
                    call(x)


@pytest.mark.gpu
def test_a_split_beyond_32_bits_is_refused():
    """A row of 2^32 values (26 GB with its moments) has no second group at column 2^32: not one group in its place."""
    import gsx  # noqa: F401
    from gsx import ops
    n = 2 ** 32 + 128
    p = torch.empty(1, n, dtype=torch.bfloat16, device="cuda")
    m, r = (torch.empty(1, n, dtype=torch.uint8, device="cuda").view(f8) for _ in range(2))
    sm, sr = torch.empty(ref.runs(n), device="cuda"), torch.empty(ref.runs(n), device="cuda")
    for split in (2 ** 32, 2 ** 32 + 64, 2 ** 31 + 1, -1, 2 ** 33):
        with pytest.raises(RuntimeError, match="split"):
            ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [p], [0.1], [0.0], 0.9, 0.999, 1e-8, [1], splits=[(split, 0.1, 0.0, False, False)])
    with pytest.raises(RuntimeError, match="2.31"):   # (a split within 32 bits, of rows that are too long for one)
        ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [p], [0.1], [0.0], 0.9, 0.999, 1e-8, [1], splits=[(3, 0.1, 0.0, False, False)])


# ---- the norm --------------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.25, float("inf")])
def test_the_factor_of_gradients_that_are_not_finite_is_zero(max_norm):
    import gsx  # noqa: F401
    from gsx import ops
    c = ops.step_control("cuda", 3)
    for bad in (float("inf"), float("-inf"), float("nan")):
        g = torch.ones(1000, device="cuda")
        g[77] = bad
        ops.grad_norm_multi([g], c, max_norm)
        a = c.cpu()
        assert not bool(torch.isfinite(a[0])) and a[1:4].tolist() == [0.0, 1.0, 3.0]
    ops.grad_norm_multi([torch.ones(16, device="cuda")], c, max_norm)   # (the block is whole again)
    assert c.cpu()[:4].tolist() == [4.0, min(1.0, max_norm / (4.0 + 1e-6)), 0.0, 4.0]


# ---- what autograd is told -------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_backward_over_a_step_is_refused(bits):
    """A graph kept over a step that needs a parameter's old values: an error, not gradients of the new ones.  Through the operators and through the optimizer."""
    import gsx  # noqa: F401
    from gsx import ops, optim
    from tests.test_adamw import splat_model
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    p = torch.nn.Parameter(torch.ones(200, device="cuda"))
    plain = torch.ones(200, device="cuda")
    loss = (p * p).sum() + (torch.ones(200, device="cuda", requires_grad=True) * plain).sum()
    loss.backward(retain_graph=True)
    versions = [p._version, plain._version]
    both, grads = [p, plain], [p.grad, torch.ones(200, device="cuda")]
    if bits == 32:
        ops.adamw_step_multi(both, [z(200), z(200)], [z(200), z(200)], grads, [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])
    else:
        ops.adamw8_step_multi(both, [z(200, dt=f8) for _ in both], [z(200, dt=f8) for _ in both], [z(2), z(2)], [z(2), z(2)], grads, [0.1] * 2, [0.0] * 2, 0.9, 0.999, 1e-8, [1, 1])
    assert [p._version, plain._version] == [v + 1 for v in versions]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                 # (such tensors have no counter)
        q = torch.ones(8, device="cuda")
        ops.adamw_step_multi([q], [z(8)], [z(8)], [torch.ones(8, device="cuda")], [0.1], [0.0], 0.9, 0.999, 1e-8, [1])
        assert float(q[0]) < 1
    m = splat_model(100, 16, "cuda")
    opt = optim.FusedAdamW.for_splat_data(m, moments=bits)
    loss = sum((t * t).sum() for t in m.params())
    loss.backward(retain_graph=True)
    opt.step(2000)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    if bits == 32:                               # rows of it count for the whole
        loss = sum((t * t).sum() for t in m.params())
        loss.backward(retain_graph=True)
        opt.step(2001, rows=(0, 40))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


# ---- what comes of many steps ----------------------------------------------------------------------------------------------------------------------------
def test_the_plain_form_rounded_to_nearest_comes_to_rest():
    """The walk that the next test's moments take, by the definition alone: 1.75, 2.5, 3, ... 6.5 codes, where 6.5 sqrt(0.999 + 0.001 (56 / 6.5)^2) = 6.73 rounds back."""
    code, walk = 0.0, []
    for _ in range(20):
        code = float(ref.rounded(torch.tensor([(0.999 * code ** 2 + 0.001 * 56.0 ** 2) ** 0.5], dtype=torch.float64), True, None))
        walk.append(code)
    assert walk[:10] == [1.75, 2.5, 3.0, 3.5, 4.0, 4.5, 5.0, 5.5, 6.0, 6.5] and set(walk[10:]) == {6.5}


@pytest.mark.gpu
def test_moments_rounded_to_nearest_come_to_rest():
    """A constant gradient, 1 / 8 of the one that holds the run's scale (whose moment is at its end from the start): to nearest, the second moment stops after ten steps at
    (6.5 / 56)^2 = 1.3 % of where it belongs and stays; stochastically it goes on."""
    import gsx  # noqa: F401
    from gsx import ops
    n = 128 * 16
    last = {}
    for seed in (None, 11):
        p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-3, device="cuda")
        g[::128] = 8e-3
        m, r = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(f8) for _ in range(2))
        sm, sr = torch.zeros(n // 128, device="cuda"), torch.full((n // 128,), 8e-3 / 448, device="cuda")
        r.view(torch.uint8)[::128] = 0x7E        # 448
        keep = torch.arange(n, device="cuda") % 128 != 0
        for t in range(1, 401):
            ops.adamw8_step_multi([p], [m], [r], [sm], [sr], [g], [0.0], [0.0], 0.9, 0.999, 1e-8, [t], seed=seed)
            if seed is None and t in (9, 10, 100, 400):
                assert bool((r.float()[keep] == (6.0 if t == 9 else 6.5)).all()), t
        last[seed] = float(((r.float() * sr.repeat_interleave(128))[keep] ** 2).mean()) / 1e-6
    # stochastically: 1 - 0.999^400 = 0.33 of it, the mean within the walk's 0.25 / sqrt(n) a standard error (five of them) and 3 %
    assert last[None] < 0.0136 and abs(last[11] / (1 - 0.999 ** 400) - 1) < 0.03 + 5 * 0.25 / n ** 0.5, last


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_the_same_training_twice(optimizer):
    """Growth, relocation and reordering on the way: the same rows, steps and moments' sizes both times."""
    import gsx  # noqa: F401
    from gsx import rasterizer, strategy, trainer
    from tests.test_gpu_training import _scene
    seen = []
    for _ in range(2):
        sc, model, cams = _scene("cuda:0")
        bg = sc["background"].to("cuda:0")
        with torch.no_grad():
            images = [rasterizer.rasterize_fused(c, model, bg).image.clone() for c in cams]
        model.means = (model.means + 0.01 * torch.randn(model.means.shape, generator=torch.Generator().manual_seed(1)).cuda()).contiguous()
        params = strategy.OptimizationParameters(iterations=45, start_refine=10, refine_every=15, stop_refine=40, max_cap=3200)
        tr = trainer.Trainer(model, cams, images, params, bg, seed=1, optimizer=optimizer, optimizer_options={"max_grad_norm": 0.05})
        tr.train(45)
        opt = tr.strategy.optimizer
        seen.append((model.means.shape[0], opt.steps, float(opt.control[3]), {k: {n: tuple(t.shape) for n, t in st.items()} for k, st in opt.state.items()}))
    assert seen[0] == seen[1]


@pytest.mark.gpu
def test_bias_corrections_of_the_device_and_of_the_call():
    """A step counted on the device forms its corrections in 32 bits, one of the call in 64: 1 / (1 - beta1^t) within 8 * 2^-24 (the series or the exponential 6, the
    reciprocal 2), 1 / sqrt(1 - beta2^t) within 5; from p = 0 the two updates differ by those, half a unit each of the other, and seven roundings on either side."""
    import gsx  # noqa: F401
    from gsx import ops
    x = inputs([1000], torch.float32, torch.float32, 14)[0]
    for betas in ((0.9, 0.999), (0.5, 0.9), (0.99, 0.99999), (0.0, 0.0)):
        for t in (1, 2, 3, 6, 7, 8, 50, 400, 499, 500, 501, 690, 700, 1000, 5000, 30000, 10 ** 6, 2 ** 32 - 1):
            out = []
            for steps, c in (([t], None), ([], ops.step_control("cuda", t))):
                p, m, v = torch.zeros(1000, device="cuda"), x[2].clone().cuda(), x[3].clone().cuda()
                ops.adamw_step_multi([p], [m], [v], [x[1].cuda()], [1e-2], [0.0], *betas, 1e-8, steps, control=c)
                out.append(p.cpu().double())
            a, b = out
            assert bool(((a - b).abs() <= 28 * ref.U * a.abs() + 2.0 ** -148).all()), (betas, t, float(((a - b).abs() / a.abs().clamp(min=1e-300)).max() / ref.U))


# ---- captured steps of a model ---------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("moments", [32, 8])
def test_captured_steps_of_a_model(moments):
    """FusedAdamW.step in a graph: replays equal eager steps, the step counted on the device, with eager work between them.  What would come out wrong in every replay is
    refused: the step that makes the moments, and a step number that is the call's."""
    import gsx  # noqa: F401
    from gsx import optim
    from tests.test_adamw import splat_model
    models = [splat_model(211, 16, "cuda") for _ in range(2)]
    opts = [optim.FusedAdamW.for_splat_data(m, moments=moments, max_grad_norm=0.5, weight_decay={"shN": 0.1}) for m in models]
    uncounted = optim.FusedAdamW.for_splat_data(splat_model(211, 16, "cuda"), moments=moments)
    fresh = optim.FusedAdamW.for_splat_data(splat_model(211, 16, "cuda"), moments=moments, max_grad_norm=float("inf"))

    def gradients(t):
        for m in models + [uncounted.model, fresh.model]:
            for i, p in enumerate(m.params()):
                g = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * t + i)).cuda()
                p.grad = g if p.grad is None else p.grad.copy_(g)
    gradients(0)
    for o in opts + [uncounted]:
        o.step(2000)
    torch.cuda.synchronize()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1)
        for o, match in ((uncounted, "max_grad_norm"), (fresh, "before the capture")):
            with pytest.raises(RuntimeError, match=match):
                o.step(2001)
        opts[1].step(2001)
    assert uncounted.steps == 1 and fresh.steps == 0 and not fresh.state and fresh.control is None
    for t in range(1, 5):
        gradients(t)
        opts[0].step(2001)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(models[0].params(), models[1].params()):
            assert torch.equal(a, b), t
        for k, st in opts[0].state.items():
            assert all(torch.equal(v.view(torch.uint8), opts[1].state[k][n].view(torch.uint8)) for n, v in st.items())
        assert torch.equal(opts[0].control, opts[1].control) and float(opts[1].control[3]) == t + 1
    fresh.step(2001)
    assert fresh.steps == 1 and float(x[0]) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("moments", [32, 8])
def test_rows_selected_by_32_bit_indices(moments):
    """select_state takes what FusedAdam's takes: indices of 32 bits, and strided ones."""
    import gsx  # noqa: F401
    from gsx import optim
    from tests.test_adamw import splat_model
    out = []
    index = torch.arange(210, -1, -1)
    for form in (index.cuda(), index.int().cuda(), torch.stack([index, index], 1).cuda()[:, 0]):
        opt = optim.FusedAdamW.for_splat_data(splat_model(211, 16, "cuda"), moments=moments)
        for i, p in enumerate(opt.model.params()):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(i)).cuda()
        opt.step(2000)
        opt.select_state(form)
        out.append([t.cpu() for n in ("means", "sh0", "opacity") for t in opt.moment_values(n)])
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


# ---- over ranks --------------------------------------------------------------------------------------------------------------------------------------------
def _plain_adamw(params, exp_avgs, exp_avg_sqs, grads, lrs, weight_decays, beta1, beta2, eps, steps, control=None, splits=()):
    """ops.adamw_step_multi in torch operations of float32 on the CPU, value by value (so that a block of rows has the bits of the whole)."""
    assert control is None and len(splits) == len(params)
    for p, m, v, g, lr, wd, t, (split, lr_b, wd_b, hold_a, hold_b) in zip(params, exp_avgs, exp_avg_sqs, grads, lrs, weight_decays, steps, splits):
        cols = p.numel() // max(1, p.shape[0])
        second = ((torch.arange(cols) >= split) if split else torch.zeros(cols, dtype=torch.bool)).reshape(p.shape[1:])
        rate, decay = torch.where(second, lr_b, lr), torch.where(second, wd_b, wd)
        live = ~torch.where(second, torch.tensor(bool(hold_b)), torch.tensor(bool(hold_a)))
        m1, v1 = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
        p1 = p - rate * decay * p - rate / (1 - beta1 ** t) * m1 / (v1.sqrt() / (1 - beta2 ** t) ** 0.5 + eps)
        for old, new in ((m, m1), (v, v1), (p, p1)):
            old.copy_(torch.where(live, new, old))


def _sharded_adamw_worker(rank, world, port, out):
    os.environ.update(RANK=str(rank), LOCAL_RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist

    import gsx  # noqa: F401
    from gsx import distributed as gdist
    from gsx import ops, optim
    from tests.test_adamw import splat_model
    ops.adamw_step_multi = _plain_adamw          # (the kernel needs a GPU)
    gdist.init_from_env(backend="gloo")
    models = {mode: splat_model(101, 16, "cpu", seed=4) for mode in ("whole", "rows")}
    opts = {mode: optim.FusedAdamW.for_splat_data(m, weight_decay={"shN": 0.2, "opacity": 0.1}) for mode, m in models.items()}
    sharded = gdist.ShardedAdam(opts["rows"])
    buckets = {mode: gdist.GradBucket(m.params()) for mode, m in models.items()}
    for t in range(8):
        if t in (3, 6):                          # growth by 5 rows, then (6) a permutation and a removal behind it
            for mode, m in models.items():
                for name in ("means", "sh", "scaling_raw", "rotation_raw", "opacity_raw"):
                    old = getattr(m, name).detach()
                    setattr(m, name, torch.cat([old, 0.5 * old[:5]]).requires_grad_(True))
                opts[mode].extend_state(5)
        if t == 6:
            sharded.merge_moments()
            order = torch.randperm(models["rows"].means.shape[0], generator=torch.Generator().manual_seed(3))[:-2]
            for mode, m in models.items():
                for name in ("means", "sh", "scaling_raw", "rotation_raw", "opacity_raw"):
                    setattr(m, name, getattr(m, name).detach()[order].clone().requires_grad_(True))
                opts[mode].select_state(order)
        if t in (3, 6):
            buckets = {mode: gdist.GradBucket(m.params()) for mode, m in models.items()}
        gen = torch.Generator().manual_seed(100 * t + rank)   # this rank's camera
        for a, b in zip(models["whole"].params(), models["rows"].params()):
            a.grad.copy_(torch.randn(a.shape, generator=gen))
            b.grad.copy_(a.grad)
        buckets["whole"].all_reduce_mean()
        opts["whole"].step(997 + t)              # shN held for the first four
        sharded.step(997 + t, buckets["rows"])
        for a, b in zip(models["whole"].params(), models["rows"].params()):
            assert torch.equal(a, b), (rank, t)
    sharded.merge_moments()
    for key, st in opts["whole"].state.items():
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(st[name], opts["rows"].state[key][name]), (rank, key, name)
    assert float(opts["rows"].state["sh"]["exp_avg"][:, 1:].abs().max()) > 0 and opts["rows"].steps == 8
    with pytest.raises(RuntimeError, match="row sharding"):
        gdist.ShardedAdam(optim.FusedAdamW.for_splat_data(models["rows"], moments=8), buckets["rows"]).step(2000)
    torch.save([p.detach() for p in models["rows"].params()], os.path.join(out, "rank%d.pt" % rank))
    dist.barrier()
    dist.destroy_process_group()


def test_sharded_adamw_over_two_ranks(tmp_path):
    """distributed.ShardedAdam with FusedAdamW on two ranks, through growth, reordering and removal: the bits of the whole step on every rank, parameters and moments."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_sharded_adamw_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    a, b = (torch.load(str(tmp_path / ("rank%d.pt" % r)), weights_only=True) for r in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a[0].shape == (109, 3)


# ---- the training examples -----------------------------------------------------------------------------------------------------------------------------------
def _example(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("name", ["train_colmap", "train_synthetic", "train_garden_standin"])
def test_examples_hand_their_decay_to_the_optimizer(name, monkeypatch):
    """The command's decay arrives as the Trainer's option, up to which a stand-in takes the place of what needs a GPU."""
    mod = _example(name)
    seen = {}
    argv = {"train_colmap": ["-d", "x", "--optimizer", "adamw8", "--weight-decay", "0.25", "--max-grad-norm", "2"], "train_synthetic": ["10", "adamw8", "0.25"],
            "train_garden_standin": ["10", "--optimizer=adamw8", "--weight-decay=0.25"]}[name]
    monkeypatch.setattr(sys, "argv", [name] + argv)

    class Reached(Exception):
        pass

    def stop(*args, **kw):
        seen.update(kw)
        raise Reached
    if name == "train_garden_standin":
        monkeypatch.setattr(mod, "setup", stop)
    elif name == "train_colmap":
        scene = types.SimpleNamespace(points=[0], colors=None, scene_center=None, cameras=[], load_images=lambda *a, **kw: [])
        monkeypatch.setattr(mod.io_colmap, "load_colmap", lambda *a, **kw: scene)
        monkeypatch.setattr(mod.io_colmap, "init_model_from_pointcloud", lambda *a, **kw: (None, 1.0))
        monkeypatch.setattr(mod.trainer, "Trainer", stop)
    else:
        monkeypatch.setattr(mod.trainer, "Trainer", stop)
        monkeypatch.setattr(mod.rasterizer, "rasterize_fused", lambda *a, **kw: types.SimpleNamespace(image=torch.zeros(3, 4, 4)))
    on_cpu = lambda f: lambda *a, **kw: f(*[("cpu" if isinstance(x, str) and x.startswith("cuda") else x) for x in a], **{k: "cpu" if k == "device" else v for k, v in kw.items()})  # noqa: E731
    monkeypatch.setattr(torch, "zeros", on_cpu(torch.zeros))
    monkeypatch.setattr(torch.Tensor, "to", on_cpu(torch.Tensor.to))
    with pytest.raises(Reached):
        mod.main()
    assert seen["optimizer"] == "adamw8" and seen["optimizer_options"]["weight_decay"] == {"shN": 0.25}
    assert seen["optimizer_options"].get("max_grad_norm", 2.0) == 2.0 and (name != "train_colmap" or "max_grad_norm" in seen["optimizer_options"])


@pytest.mark.gpu
def test_train_colmap_example_with_decay(tmp_path):
    """The command, for a few iterations, without and with a decay: it reaches its group and no other."""
    mod = _example("train_colmap")
    cap = mod.make_synthetic(str(tmp_path / "capture"))
    kept, make = [], mod.trainer.Trainer

    def keep(*a, **kw):
        kept.append(make(*a, **kw))
        return kept[-1]
    for decay in (0.0, 0.5):
        args = argparse.Namespace(data=cap, images="images", iter=25, config=None, eval=True, test_every=8, resize_factor=-1, max_width=3840, output=None, json=None, log_every=0,
                                  optimizer="adamw", weight_decay=decay, max_grad_norm=1.0)
        mod.trainer.Trainer = keep
        try:
            res = mod.run(args)
        finally:
            mod.trainer.Trainer = make
        assert res["iterations"] == 25
    a, b = (t.strategy.optimizer for t in kept)
    assert a.weight_decay["shN"] == 0.0 and b.weight_decay == dict(a.weight_decay, shN=0.5) and b.max_grad_norm == 1.0
    assert a.steps == b.steps == 24              # (the last iteration of a run takes no step: MCMC.step)
