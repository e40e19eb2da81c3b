"""Products of row groups on the GPU: `gemm_grouped_` (rows and their gradient) and `gemm_grouped_grad_` against 64-bit
products of each group.  f16 / bf16 products are exact in fp32; a sum of K of them in fp32, in whatever order and
rounded or cut, is off by at most K * 2^-23 of the sum of magnitudes, alpha and beta add 3 roundings, and the output
rounding eps / 2 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# borders, rows, N, K: one row, empty groups at both ends and between, rows before the first and behind the last group,
# groups larger than any tile, sizes that fill no tile, one element
CASES = [([0, 1], 1, 8, 8), ([0, 0, 5, 5, 5, 9, 9], 9, 136, 72), ([2, 3, 20, 37], 41, 1000, 200), ([0, 0, 0], 3, 64, 64),
         ([0, 129, 700], 700, 256, 136), ([0, 300, 301, 1100], 1111, 72, 1336), ([0] + list(range(16, 16 * 33, 16)), 512, 128, 512),
         ([0, 513], 513, 520, 64), ([0, 40, 100], 100, 2056, 8)]


def operands(rows, groups, n, k, dtype, dev, seed=1):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).to(dtype)
    return r(rows, k), r(groups, n, k), r(rows, n)


def within(got, want, mag, terms, out):
    tol = (terms + 3) * 2.0 ** -23 * mag
    if out != torch.float32:
        tol = tol + torch.finfo(out).eps / 2 * want.abs() + torch.finfo(out).tiny * torch.finfo(out).eps
    return bool(((got.double() - want).abs() <= tol).all())


def by_group(offsets, rows, f):
    """Concatenated f(g, slice) over groups into (rows, ...) float64; NaN outside the groups."""
    out = None
    for g in range(len(offsets) - 1):
        s = slice(offsets[g], offsets[g + 1])
        v = f(g, s)
        if out is None:
            out = torch.full((rows, v.shape[1]), float("nan"), dtype=torch.float64, device=v.device)
        out[s] = v
    return out


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_grouped_product_and_row_gradient(mb, dev, case, kind, out):
    offsets, rows, n, k = CASES[case]
    dt = DT[kind]
    ot = dt if out == "same" else torch.float32
    a, b, d = operands(rows, len(offsets) - 1, n, k, dt, dev)
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    inside = torch.zeros(rows, dtype=torch.bool, device=dev)
    inside[offsets[0]:offsets[-1]] = True
    # b is read along K for the product and along N for the gradient of the rows
    for x, w, width, terms in ((a, b, n, k), (d, b.transpose(1, 2), k, n)):
        got = torch.full((rows, width), float("nan"), dtype=ot, device=dev)
        assert mb.gemm_grouped_(got, x, w, edge) is got
        mb.synchronize_status(dev)
        want = by_group(offsets, rows, lambda g, s: x[s].double() @ w[g].double().T)
        mag = by_group(offsets, rows, lambda g, s: x[s].double().abs() @ w[g].double().abs().T)
        assert bool(got[~inside].isnan().all())
        assert within(got[inside], want[inside], mag[inside], terms, ot)


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_weight_gradient(mb, dev, case, kind, out):
    offsets, rows, n, k = CASES[case]
    dt = DT[kind]
    ot = dt if out == "same" else torch.float32
    a, b, d = operands(rows, len(offsets) - 1, n, k, dt, dev)
    for x in (a, d):  # what lies outside the groups must not reach any gradient
        x[:offsets[0]] = float("nan")
        x[offsets[-1]:] = float("inf")
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    got = torch.full(b.shape, float("nan"), dtype=ot, device=dev)
    assert mb.gemm_grouped_grad_(got, d, a, edge) is got
    mb.synchronize_status(dev)
    for g in range(len(offsets) - 1):
        s = slice(offsets[g], offsets[g + 1])
        want = d[s].double().T @ a[s].double()
        mag = d[s].double().abs().T @ a[s].double().abs()
        assert within(got[g], want, mag, offsets[g + 1] - offsets[g], ot)


def test_alpha_beta_and_pitched_views(mb, dev):
    offsets, rows, n, k = [0, 7, 7, 150], 160, 200, 96
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    dt = torch.bfloat16
    gen = torch.Generator(device=dev).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).to(dt)
    a, b, d = r(rows, 2 * k)[:, 8:8 + k], r(3, n + 5, k + 16)[:, 2:n + 2, 8:8 + k], r(rows, n + 24)[:, 16:16 + n]
    base = r(rows, n + 31)
    for alpha, beta in ((0.5, 1.0), (-2.0, 0.25)):
        big = base.clone()
        got = big[:, 3:3 + n]                                        # rows of D on no 16-byte boundary
        mb.gemm_grouped_(mb.MoYeArray(got), mb.MoYeArray(a), mb.MoYeArray(b), edge, alpha=alpha, beta=beta)
        old = base[:, 3:3 + n].double()
        for g in range(3):
            s = slice(offsets[g], offsets[g + 1])
            want = alpha * (a[s].double() @ b[g].double().T) + beta * old[s]
            mag = abs(alpha) * (a[s].double().abs() @ b[g].double().abs().T) + abs(beta) * old[s].abs()
            assert within(got[s], want, mag, k, dt)
        assert torch.equal(big[150:], base[150:]) and torch.equal(big[:, :3], base[:, :3]) and torch.equal(big[:, 3 + n:], base[:, 3 + n:])
        gbase = torch.randn(3, n + 2, k + 5, generator=gen, device=dev)
        gbig = gbase.clone()
        gw = gbig[:, 1:n + 1, 2:2 + k]
        mb.gemm_grouped_grad_(gw, d, a, edge, alpha=alpha, beta=beta)
        for g in range(3):
            s = slice(offsets[g], offsets[g + 1])
            want = alpha * (d[s].double().T @ a[s].double()) + beta * gbase[g, 1:n + 1, 2:2 + k].double()
            mag = abs(alpha) * (d[s].double().abs().T @ a[s].double().abs()) + abs(beta) * gbase[g, 1:n + 1, 2:2 + k].double().abs()
            assert within(gw[g], want, mag, offsets[g + 1] - offsets[g], torch.float32)
        gw.copy_(gbase[:, 1:n + 1, 2:2 + k])
        assert torch.equal(gbig, gbase)
    mb.synchronize_status(dev)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("alpha,beta", [(1.0, 1.0), (0.5, 1.0), (1.5, -0.75)])
def test_adding_to_aligned_outputs(mb, dev, kind, alpha, beta):
    """beta on rows that vectors and TMA may write: the memory adds, or the old values are read, also at group ends."""
    offsets, rows, n, k = [0, 40, 40, 300, 333], 340, 264, 200
    a, b, d = operands(rows, 4, n, k, torch.bfloat16, dev, seed=6)
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    gen = torch.Generator(device=dev).manual_seed(7)
    old, old_b = (torch.randn(*s, generator=gen, device=dev).to(DT[kind]) for s in ((rows, n), (4, n, k)))
    got = mb.gemm_grouped_(old.clone(), a, b, edge, alpha=alpha, beta=beta)
    got_b = mb.gemm_grouped_grad_(old_b.clone(), d, a, edge, alpha=alpha, beta=beta)
    mb.synchronize_status(dev)
    assert torch.equal(got[333:], old[333:])
    for g in range(4):
        s = slice(offsets[g], offsets[g + 1])
        want = alpha * (a[s].double() @ b[g].double().T) + beta * old[s].double()
        mag = abs(alpha) * (a[s].double().abs() @ b[g].double().abs().T) + abs(beta) * old[s].double().abs()
        assert within(got[s], want, mag, k, DT[kind])
        want = alpha * (d[s].double().T @ a[s].double()) + beta * old_b[g].double()
        mag = abs(alpha) * (d[s].double().abs().T @ a[s].double().abs()) + abs(beta) * old_b[g].double().abs()
        assert within(got_b[g], want, mag, offsets[g + 1] - offsets[g], DT[kind])


@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_odd_extents_between_padded_pitches(mb, dev, out):
    """Extents that are no multiple of anything; what lies in the padding (not numbers) is neither read nor written."""
    offsets, rows, n, k = [0, 5, 70, 333], 333, 131, 203
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    gen = torch.Generator(device=dev).manual_seed(8)

    def padded(*shape):
        x = torch.full((*shape[:-1], (shape[-1] + 15) // 8 * 8), float("nan"), dtype=torch.bfloat16, device=dev)
        x[..., :shape[-1]] = torch.randn(*shape, generator=gen, device=dev)
        return x[..., :shape[-1]]

    a, b, d, bt = padded(rows, k), padded(3, n, k), padded(rows, n), padded(3, k, n)
    for x, w, width in ((a, b, n), (a, bt.transpose(1, 2), n), (d, b.transpose(1, 2), k)):
        big = torch.full((rows, (width + 15) // 8 * 8), 9.0, dtype=DT[out], device=dev)
        got = mb.gemm_grouped_(big[:, :width], x, w, edge)
        for g in range(3):
            s = slice(offsets[g], offsets[g + 1])
            assert within(got[s], x[s].double() @ w[g].double().T, x[s].double().abs() @ w[g].double().abs().T, x.shape[1], DT[out])
        assert bool((big[:, width:] == 9).all())
    big = torch.full((3, n, (k + 15) // 8 * 8), 9.0, dtype=DT[out], device=dev)
    got = mb.gemm_grouped_grad_(big[:, :, :k], d, a, edge)
    for g in range(3):
        s = slice(offsets[g], offsets[g + 1])
        assert within(got[g], d[s].double().T @ a[s].double(), d[s].double().abs().T @ a[s].double().abs(), offsets[g + 1] - offsets[g], DT[out])
    assert bool((big[:, :, k:] == 9).all())
    mb.synchronize_status(dev)


@pytest.mark.parametrize("k", [1001, 1008])
def test_the_pitch_of_a_single_row_says_nothing(mb, dev, k):
    gen = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).to(torch.bfloat16)
    one = lambda t: t.as_strided(t.shape, (t.shape[1] + 3, 1))
    a, b, d = one(r(1, k)), r(2, 72, 1008)[:, :, :k], one(r(1, 72))
    edge = torch.tensor([0, 0, 1], dtype=torch.int32, device=dev)
    got = mb.gemm_grouped_(one(torch.zeros(1, 72, device=dev, dtype=torch.bfloat16)), a, b, edge)
    want, mag = a.double() @ b[1].double().T, a.double().abs() @ b[1].double().abs().T
    assert within(got, want, mag, k, torch.bfloat16)
    grad = mb.gemm_grouped_grad_(torch.ones(2, 72, k, device=dev, dtype=torch.bfloat16), d, a, edge)
    mb.synchronize_status(dev)
    assert bool((grad[0] == 0).all())
    want = d.double().T @ a.double()
    assert within(grad[1], want, want.abs(), 1, torch.bfloat16)


def test_a_group_longer_than_many_tiles(mb, dev):
    """9 row tiles (a full band of 8 and one more) and a sum over 2100 rows."""
    offsets, rows, n, k = [0, 2100, 2110], 2110, 520, 136
    a, b, d = operands(rows, 2, n, k, torch.bfloat16, dev, seed=9)
    edge = torch.tensor(offsets, dtype=torch.int32, device=dev)
    for ot in (torch.bfloat16, torch.float32):
        got = mb.gemm_grouped_(torch.empty(rows, n, dtype=ot, device=dev), a, b, edge)
        grad = mb.gemm_grouped_grad_(torch.empty(2, n, k, dtype=ot, device=dev), d, a, edge)
        for g in range(2):
            s = slice(offsets[g], offsets[g + 1])
            assert within(got[s], a[s].double() @ b[g].double().T, a[s].double().abs() @ b[g].double().abs().T, k, ot)
            assert within(grad[g], d[s].double().T @ a[s].double(), d[s].double().abs().T @ a[s].double().abs(), offsets[g + 1] - offsets[g], ot)
    mb.synchronize_status(dev)


def test_neighbours_do_not_leak(mb, dev):
    """A group of infinities beside an ordinary one: neither the rows' products nor the weights' gradients mix."""
    edge = torch.tensor([0, 5, 9, 100], dtype=torch.int32, device=dev)
    a, b, d = operands(100, 3, 64, 128, torch.bfloat16, dev)
    a[5:9], d[5:9] = float("inf"), float("nan")
    out = mb.gemm_grouped_(torch.empty(100, 64, device=dev), a, b, edge)
    assert bool(out[:5].isfinite().all()) and bool(out[9:].isfinite().all()) and not bool(out[5:9].isfinite().any())
    g = mb.gemm_grouped_grad_(torch.empty(3, 64, 128, device=dev), d, a, edge)
    assert bool(g[0].isfinite().all()) and bool(g[2].isfinite().all()) and not bool(g[1].isfinite().any())


def test_borders_out_of_range_are_clamped(mb, dev):
    """Borders that run backwards or out of the array give empty groups and whole groups, never a bad address."""
    a, b, d = operands(50, 4, 72, 64, torch.bfloat16, dev)
    for bad, good in (([-7, 20, 10, 40, 1000], [0, 20, 20, 40, 50]), ([60, 70, 3, -1, 50], [50, 50, 50, 50, 50])):
        bad, good = (torch.tensor(v, dtype=torch.int32, device=dev) for v in (bad, good))
        x, y = (mb.gemm_grouped_(torch.zeros(50, 72, device=dev), a, b, e) for e in (bad, good))
        assert torch.equal(x, y)
        x, y = (mb.gemm_grouped_grad_(torch.ones(4, 72, 64, device=dev), d, a, e) for e in (bad, good))
        assert torch.equal(x, y)
    mb.synchronize_status(dev)


def test_no_rows(mb, dev):
    edge = torch.zeros(4, dtype=torch.int32, device=dev)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    mb.gemm_grouped_(torch.empty(0, 32, dtype=torch.bfloat16, device=dev), e, torch.ones(3, 32, 64, dtype=torch.bfloat16, device=dev), edge)
    g = torch.full((3, 32, 64), 3.0, device=dev)
    mb.gemm_grouped_grad_(g, torch.empty(0, 32, dtype=torch.bfloat16, device=dev), e, edge, beta=0.5)
    assert bool((g == 1.5).all())
    mb.gemm_grouped_grad_(g.fill_(float("nan")), torch.empty(0, 32, dtype=torch.bfloat16, device=dev), e, edge)
    assert bool((g == 0).all())
    mb.synchronize_status(dev)


def test_same_bits_every_time_and_captured(mb, dev):
    edge = torch.tensor([0, 37, 37, 300, 640], dtype=torch.int32, device=dev)
    a, b, d = operands(640, 4, 512, 256, torch.bfloat16, dev)
    out, grad = torch.zeros(640, 512, dtype=torch.bfloat16, device=dev), torch.zeros(4, 512, 256, device=dev)
    mb.gemm_grouped_(out, a, b, edge)
    mb.gemm_grouped_grad_(grad, d, a, edge)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    o2, g2 = torch.zeros_like(out), torch.zeros_like(grad)
    with torch.cuda.graph(graph):
        mb.gemm_grouped_(o2, a, b, edge)
        mb.gemm_grouped_grad_(g2, d, a, edge)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, o2) and torch.equal(grad, g2)
    edge.copy_(torch.tensor([0, 1, 200, 201, 640], dtype=torch.int32))  # the captured launch follows new borders
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o2, mb.gemm_grouped_(torch.zeros_like(out), a, b, edge))
    assert torch.equal(g2, mb.gemm_grouped_grad_(torch.zeros_like(grad), d, a, edge))


def test_gradients_against_differences(mb, dev):
    """The product is linear in A and in B.  With whole numbers below 8, K = 16 and N = 24, every sum is exact in fp32:
    a difference of <gemm_grouped(A, B), dD> over a step of 1 IS the derivative."""
    edge = torch.tensor([0, 3, 3, 8], dtype=torch.int32, device=dev)
    gen = torch.Generator(device=dev).manual_seed(4)
    a, b, d = (torch.randint(-7, 8, s, generator=gen, device=dev).to(torch.float16) for s in ((8, 16), (3, 24, 16), (8, 24)))
    value = lambda a, b: float((mb.gemm_grouped_(torch.zeros(8, 24, device=dev), a, b, edge).double() * d.double()).sum())
    da = mb.gemm_grouped_(torch.zeros(8, 16, device=dev), d, b.transpose(1, 2), edge)
    db = mb.gemm_grouped_grad_(torch.zeros(3, 24, 16, device=dev), d, a, edge)
    base = value(a, b)
    for t, g in ((a, da), (b, db)):
        for i in range(0, t.numel(), 7):
            moved = t.clone()
            moved.view(-1)[i] += 1
            assert (value(moved, b) if t is a else value(a, moved)) - base == float(g.reshape(-1)[i])


def test_refusals(mb, dev):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    edge = torch.zeros(4, dtype=torch.int32, device=dev)

    def refused(code, fn, *args, **kw):
        with pytest.raises(mb.MoyeError) as e:
            fn(*args, **kw)
        assert e.value.code == code, str(e.value)

    ok = (z(16, 32), z(16, 64), z(3, 32, 64), edge)
    mb.gemm_grouped_(*ok)
    for code, i, bad in ((-4, 0, z(16, 40)), (-4, 0, z(15, 32)), (-4, 1, z(16, 72)), (-4, 2, z(32, 64)), (-2, 0, z(16, 32, dtype=torch.float16)),
                         (-2, 1, z(16, 64, dtype=torch.float16)), (-2, 2, z(3, 32, 64, dtype=torch.float32)), (-3, 0, z(32, 16).t()),
                         (-3, 1, z(64, 16).t()), (-5, 1, z(16, 68)[:, :64]), (-5, 1, z(16, 72)[:, 4:68]), (-5, 2, z(3, 32, 68)[:, :, :64]),
                         (-3, 2, z(64, 32, 3).permute(2, 1, 0)), (-3, 2, z(1, 32, 64).expand(3, 32, 64)),
                         (-4, 3, edge[:3]), (-1, 3, edge.long())):
        args = list(ok)
        args[i] = bad
        refused(code, mb.gemm_grouped_, *args)
    ok = (z(3, 32, 64), z(16, 32), z(16, 64), edge)
    mb.gemm_grouped_grad_(*ok)
    for code, i, bad in ((-4, 0, z(3, 40, 64)), (-4, 1, z(15, 32)), (-2, 0, z(3, 32, 64, dtype=torch.float16)), (-3, 0, z(3, 64, 32).transpose(1, 2)),
                         (-3, 1, z(32, 16).t()), (-5, 2, z(16, 68)[:, :64]), (-4, 3, edge[:3])):
        args = list(ok)
        args[i] = bad
        refused(code, mb.gemm_grouped_grad_, *args)
    many = torch.zeros(1026, dtype=torch.int32, device=dev)
    refused(-4, mb.gemm_grouped_, z(16, 8), z(16, 8), z(1025, 8, 8), many)
    with pytest.raises(RuntimeError):
        mb.gemm_grouped_(torch.zeros(16, 32, dtype=torch.bfloat16), z(16, 64), z(3, 32, 64), edge)
    torch.cuda.synchronize()


def test_a_layer_of_experts(mb, dev):
    """The operators together, as a mixture-of-experts layer uses them in training: route, sort, first product, relu,
    second product, weighted sum back, and the way back through all of it, against autograd in 64 bits.  Every stage
    rounds its result to bf16 (half a step 2^-9 of its scale); six such roundings on the longest way and sums of at most
    256 of them, whose errors add like independent ones, stay below 6 * 2^-9 of the result's rms, and the largest of
    10^5 values below 6 times that."""
    tokens, choices, groups, width, hidden = 500, 2, 6, 128, 256
    gen = torch.Generator(device=dev).manual_seed(8)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device=dev) * scale).to(torch.bfloat16)
    x, w1, w2 = r(tokens, width), r(groups, hidden, width, scale=width ** -0.5), r(groups, width, hidden, scale=hidden ** -0.5)
    logits = torch.randn(tokens, groups, generator=gen, device=dev)
    top, ids = logits.topk(choices, 1)
    weights = torch.softmax(top, 1)
    dy = r(tokens, width)
    n = tokens * choices
    z = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=dev)

    plan = mb.group_rows(ids, groups)
    xs = mb.gather_rows_(z(n, width), x, plan)
    h = mb.gemm_grouped_(z(n, hidden), xs, w1, plan)
    act = h.relu()
    ys = mb.gemm_grouped_(z(n, width), act, w2, plan)
    y = mb.combine_rows_(z(tokens, width), ys, plan, weights)
    dys, dw = mb.combine_rows_grad_(z(n, width), torch.empty_like(weights), dy, ys, plan, weights)
    dact = mb.gemm_grouped_(z(n, hidden), dys, w2.transpose(1, 2), plan)
    dw2 = mb.gemm_grouped_grad_(torch.empty(w2.shape, device=dev), dys, act, plan)
    dh = dact * (h > 0)
    dxs = mb.gemm_grouped_(z(n, width), dh, w1.transpose(1, 2), plan)
    dw1 = mb.gemm_grouped_grad_(torch.empty(w1.shape, device=dev), dh, xs, plan)
    dx = mb.combine_rows_(z(tokens, width), dxs, plan)
    mb.synchronize_status(dev)

    X, W1, W2, P = (t.double().requires_grad_() for t in (x, w1, w2, weights))
    Y = torch.zeros(tokens, width, dtype=torch.float64, device=dev)
    for g in range(groups):
        t, j = (ids == g).nonzero(as_tuple=True)
        Y = Y.index_add(0, t, P[t, j][:, None] * ((X[t] @ W1[g].T).relu() @ W2[g].T))
    Y.backward(dy.double())
    for got, want in ((y, Y), (dx, X.grad), (dw1, W1.grad), (dw2, W2.grad), (dw, P.grad)):
        want = want.detach()
        rms = want.square().mean().sqrt()
        err = (got.double() - want).abs()
        assert float(err.square().mean().sqrt() / rms) < 6 * 2.0 ** -9
        assert float(err.max() / rms) < 36 * 2.0 ** -9 + float(want.abs().max() / rms) * 2.0 ** -8


def test_two_streams_at_once(mb, dev):
    """The operators of two streams share no scratch: run beside one another they give what they give alone."""
    def make(seed):
        gen = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device=dev) * scale).to(torch.bfloat16)
        ids = torch.randint(0, 6, (700, 2), generator=gen, device=dev)
        return {"ids": ids, "x": r(700, 256), "w": r(6, 512, 256, scale=1 / 16), "a": r(3, 16, 512, scale=1 / 16), "b": r(3, 256, 16),
                "which": torch.arange(7, dtype=torch.int32, device=dev) % 4, "edge": (torch.arange(8, device=dev) * 200).int(), "weights": torch.rand(700, 2, generator=gen, device=dev)}

    def step(s):
        plan = mb.group_rows(s["ids"], 6)
        xs = mb.gather_rows_(torch.zeros(1400, 256, dtype=torch.bfloat16, device=dev), s["x"], plan)
        h = mb.gemm_grouped_(torch.zeros(1400, 512, dtype=torch.bfloat16, device=dev), xs, s["w"], plan)
        g = mb.gemm_grouped_grad_(torch.zeros(6, 512, 256, device=dev), h, xs, plan)
        y = mb.gemm_lora_(torch.zeros(1400, 256, dtype=torch.bfloat16, device=dev), h, s["a"], s["b"], s["which"], s["edge"])
        return plan.order, h, g, y, mb.combine_rows_(torch.zeros(700, 256, dtype=torch.bfloat16, device=dev), y, plan, s["weights"])

    states = [make(31), make(32)]
    alone = [step(s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(states[i]))
    torch.cuda.synchronize()
    mb.synchronize_status(dev)
    for i in (0, 1):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, alone[i]))


def test_under_the_debug_build(dev):
    """The debug library checks every tile against the arrays on the device: the small tests pass under it unchanged."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    res = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-k",
                          "(test_grouped_product and 5-bf16) or (test_weight_gradient and 5-f16) or (test_lora_tiles and 0-bf16) or clamped or no_rows",
                          os.path.join(here, "test_gpu_grouped.py"), os.path.join(here, "test_gpu_lora.py")], capture_output=True, text=True,
                         env=dict(os.environ, MOYE_B200_DEBUG="1"), timeout=600)
    assert res.returncode == 0 and " passed" in res.stdout, res.stdout[-3000:] + res.stderr[-1000:]


@pytest.mark.parametrize("beta", [1.0, 0.5])
def test_gradients_below_the_normal_range_accumulate(mb, dev, beta):
    """Float32 outputs: subnormal products and old values are kept as they are (beta = 1 is added by the memory).  The
    products are 64 and 128 times 2^-140, the old values multiples of 2^-148: every sum is exact."""
    edge = torch.tensor([0, 64], dtype=torch.int32, device=dev)
    x, y = torch.full((64, 128), 2.0 ** -70, device=dev).bfloat16(), torch.full((64, 64), 2.0 ** -70, device=dev).bfloat16()
    for old in (0.0, 6.0 * 2.0 ** -148, -100.0 * 2.0 ** -148, -2.0 ** -126, 2.0 ** -126):
        db = mb.gemm_grouped_grad_(torch.full((1, 64, 128), old, device=dev), y, x, edge, beta=beta)
        d = mb.gemm_grouped_(torch.full((64, 64), old, device=dev), x, x.view(1, 64, 128), edge, beta=beta)
        mb.synchronize_status(dev)
        assert bool((db.double() == 2.0 ** -134 + beta * old).all()) and bool((d.double() == 2.0 ** -133 + beta * old).all())


def test_outputs_over_operands_are_refused(mb, dev):
    """Tiles are written while others still read: an output that shares memory with an operand would depend on the order."""
    rows, width, groups = 48, 64, 3
    edge = torch.tensor([0, 5, 20, 48], dtype=torch.int32, device=dev)
    flat = torch.zeros(4 * groups * width * width, dtype=torch.bfloat16, device=dev)
    x, w = flat[:rows * width].view(rows, width), flat[rows * width:][:groups * width * width].view(groups, width, width)
    free = flat[2 * groups * width * width:]
    y, g = free[:rows * width].view(rows, width), free[rows * width:][:groups * width * width].view(groups, width, width)
    mb.gemm_grouped_(y, x, w, edge)
    mb.gemm_grouped_(y, x, w.transpose(1, 2), edge)
    mb.gemm_grouped_grad_(g, y, x, edge)
    shifted = flat[8:8 + rows * width].view(rows, width)
    for call in (lambda: mb.gemm_grouped_(x, x, w, edge), lambda: mb.gemm_grouped_(shifted, x, w, edge),
                 lambda: mb.gemm_grouped_(w[2, :48], x, w, edge), lambda: mb.gemm_grouped_(w[2, :48], x, w.transpose(1, 2), edge),
                 lambda: mb.gemm_grouped_grad_(g, y, g[1, :48], edge), lambda: mb.gemm_grouped_grad_(g, g[2, 16:], x, edge),
                 lambda: mb.gemm_grouped_grad_(w, y, shifted, edge)):
        with pytest.raises(mb.MoyeError) as e:
            call()
        assert e.value.code == -1, str(e.value)
    # beside one another in a wider array: rows of A and D, weights and their gradient
    gen = torch.Generator(device=dev).manual_seed(2)
    both = torch.randn(rows, 2 * width, generator=gen, device=dev).bfloat16()
    ws = torch.randn(groups, width, 2 * width, generator=gen, device=dev).bfloat16()
    want = mb.gemm_grouped_(y, both[:, :width].contiguous(), ws[:, :, :width].contiguous(), edge)
    mb.gemm_grouped_(both[:, width:], both[:, :width], ws[:, :, :width], edge)
    assert torch.equal(both[:, width:], want)
    mb.gemm_grouped_grad_(ws[:, :, width:], want, both[:, :width], edge)
    assert torch.equal(ws[:, :, width:], mb.gemm_grouped_grad_(g, want, both[:, :width].contiguous(), edge))
    mb.synchronize_status(dev)
