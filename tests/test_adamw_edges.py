"""The optimizer operators over many tensors (include/gsx_optim.h) at their edges: quotients next to the middle between two numbers, runs of chunks that cross from tensor
to tensor, views with 8-bit moments, what is refused, what autograd is told — against the plain forms in 64 bits (adamw_reference.py)."""
import pytest
import torch

from tests import adamw_reference as ref

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
