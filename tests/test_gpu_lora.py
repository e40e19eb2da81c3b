"""Low-rank adapters of many requests on the GPU: `gemm_lora_` against 64-bit products of every request.  The value is
C + s * sum over R of (sum over K): in fp32 off by at most (K + R + 4) * 2^-23 of the sum of magnitudes; the product of
rank R may be carried as a high and a low 16-bit part, off by 2^-16 of itself, when the output has 16 bits; the
output rounding adds eps / 2 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# borders (None: a request per row), rows, adapters of the requests, N, K, R, count
CASES = [
    (None, 1, [0], 8, 8, 8, 1),
    (None, 5, [2, -1, 0, 7, 2], 1001, 520, 24, 3),                           # none, and a number that does not exist
    ([0, 3, 3, 40, 41], 41, [1, 0, 0, -1], 136, 4096, 16, 2),                # an empty request, one without an adapter
    ([2, 130, 300], 310, [3, 1], 2056, 1000, 64, 4),                         # rows before and behind every request
    ([0, 129, 257, 700], 700, [0, 0, 2], 264, 264, 128, 3),                  # the largest rank, long requests
    (list(range(0, 65)), 64, [i % 7 for i in range(64)], 4096, 512, 8, 7),
    ([0, 1000], 1000, [0], 1, 16, 40, 1),
    ([0, 1, 2, 200, 201, 460, 461], 461, [0, 1, 2, 3, 4, 5], 512, 1024, 32, 6),
]


def make(case, kind, dev, seed=1):
    offsets, rows, which, n, k, rank, count = case
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device=dev) * scale).to(DT[kind])
    x, a, b = r(rows, k), r(count, rank, k, scale=k ** -0.5), r(count, n, rank, scale=rank ** -0.5)
    scales = torch.rand(count, generator=gen, device=dev) + 0.5
    edge = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=dev)
    return x, a, b, scales, torch.tensor(which, dtype=torch.int32, device=dev), edge


def check(got, c, x, a, b, scales, which, offsets, out, untouched):
    rank, k = a.shape[1:]
    offsets = list(range(len(which) + 1)) if offsets is None else offsets
    inside = torch.zeros(len(c), dtype=torch.bool, device=c.device)
    for q, w in enumerate(which):
        s = slice(offsets[q], offsets[q + 1])
        inside[s] = True
        if not 0 <= w < len(a):
            assert torch.equal(got[s], c[s])
            continue
        f = 1.0 if scales is None else float(scales[w])
        want = c[s].double() + f * ((x[s].double() @ a[w].double().T) @ b[w].double().T)
        mag = f * ((x[s].double().abs() @ a[w].double().abs().T) @ b[w].double().abs().T)
        tol = (k + rank + 4) * 2.0 ** -23 * (mag + c[s].double().abs())
        if out != torch.float32:
            tol = tol + 2.0 ** -16 * mag + torch.finfo(out).eps / 2 * want.abs() + torch.finfo(out).tiny * torch.finfo(out).eps
        assert bool(((got[s].double() - want).abs() <= tol).all())
    assert torch.equal(got[~inside], untouched[~inside])


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_lora(mb, dev, case, kind, out):
    offsets, rows, which, n, k, rank, count = CASES[case]
    ot = DT[kind] if out == "same" else torch.float32
    x, a, b, scales, w, edge = make(CASES[case], kind, dev)
    c = torch.randn(rows, n, device=dev).to(ot)
    d0 = torch.full_like(c, -3.0)
    d = d0.clone()
    assert mb.gemm_lora_(d, x, a, b, w, edge, scales=scales, C=c) is d
    check(d, c, x, a, b, scales, which, offsets, ot, d0)
    inplace = c.clone()
    mb.gemm_lora_(inplace, x, a, b, w, edge)
    check(inplace, c, x, a, b, None, which, offsets, ot, c)
    mb.synchronize_status(dev)


# sizes at which requests share their factors on the tensor cores: tiles of 1 to 128 rows in one launch, turned (up to 32
# rows) and not, a cluster of CTAs per tile and one CTA per tile, outputs that TMA can and cannot write, every part of R
TILES = [
    ([0, 1, 3, 20, 52, 85, 213, 341, 800], 805, [3, 0, 1, -1, 2, 3, 9, 0], 1001, 520, 64, 4),
    ([2, 3, 20, 52, 85, 213, 341, 800], 800, [0, 1, 2, 2, 3, -1, 1], 1000, 520, 72, 4),
    ([0, 3000], 3000, [0], 520, 136, 128, 1),
    ([0, 4000, 4000, 4001], 4001, [1, 0, 0], 264, 4096, 8, 2),
    (list(range(0, 8001, 40)), 8000, [i % 4 for i in range(200)], 264, 200, 24, 3),
    (list(range(0, 1537, 32)), 1536, [i % 5 for i in range(48)], 131, 1032, 48, 5),
]


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("case", range(len(TILES)))
def test_lora_tiles(mb, dev, case, kind, out):
    offsets, rows, which, n, k, rank, count = TILES[case]
    ot = DT[kind] if out == "same" else torch.float32
    x, a, b, scales, w, edge = make(TILES[case], kind, dev)
    x[:offsets[0]], x[offsets[-1]:] = float("nan"), float("inf")
    c = torch.randn(rows, n + 9, device=dev).to(ot)[:, :n]
    if n % 8 == 0:
        c = c.contiguous()
    d0 = torch.full((rows, n), -3.0, device=dev).to(ot)
    d = d0.clone()
    mb.gemm_lora_(d, x, a, b, w, edge, scales=scales, C=c)
    mb.synchronize_status(dev)
    check(d, c, x, a, b, scales, which, offsets, ot, d0)
    wide = torch.full((rows, n + 24), 5.0, device=dev).to(ot)
    inplace = wide[:, 8:8 + n]
    inplace.copy_(c)
    mb.gemm_lora_(inplace, x, a, b, w, edge)
    check(inplace, c, x, a, b, None, which, offsets, ot, c)
    assert bool((wide[:, :8] == 5).all()) and bool((wide[:, 8 + n:] == 5).all())
    mb.synchronize_status(dev)


def test_pitched_views_and_moye_arrays(mb, dev):
    offsets, which, n, k, rank = [0, 5, 200], [1, 0], 100, 64, 16
    gen = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev).to(torch.bfloat16)
    x, a, b = r(200, 2 * k)[:, 8:8 + k], r(2, rank + 3, k + 8)[:, 1:1 + rank, 8:8 + k], r(2, n + 1, rank + 8)[:, 1:, :rank]
    base = r(200, n + 9)
    big = base.clone()
    d, c = big[:, 3:3 + n], r(200, n + 1)[:, 1:]
    edge, w = torch.tensor(offsets, dtype=torch.int32, device=dev), torch.tensor(which, dtype=torch.int32, device=dev)
    mb.gemm_lora_(mb.MoYeArray(d), mb.MoYeArray(x), a, b, w, edge, C=mb.MoYeArray(c))
    check(d, c, x, a, b, None, which, offsets, torch.bfloat16, d)
    assert torch.equal(big[:, :3], base[:, :3]) and torch.equal(big[:, 3 + n:], base[:, 3 + n:])


def test_the_pitch_of_a_single_row_says_nothing(mb, dev):
    case = ([0, 1], 1, [0], 272000, 272000, 128, 1)  # long enough for the tiles of the tensor cores
    x, a, b, scales, w, edge = make(case, "bf16", dev)
    one = lambda t: t.as_strided(t.shape, (t.shape[1] + 3, 1))
    c = torch.randn(1, 272000, device=dev).to(torch.bfloat16)
    got = mb.gemm_lora_(one(torch.zeros_like(c)), one(x), a, b, w, edge, scales, C=one(c))
    mb.synchronize_status(dev)
    check(got, c, x, a, b, scales, [0], [0, 1], torch.bfloat16, c)


def test_infinities_stay_in_their_rows(mb, dev):
    x, a, b, scales, w, edge = make(CASES[3], "bf16", dev)
    x[:2], x[300:], x[129] = float("nan"), float("inf"), float("inf")
    d = torch.zeros(310, 2056, device=dev)
    mb.gemm_lora_(d, x, a, b, w, edge)
    bad = ~d.isfinite().all(1)
    assert bad.nonzero().view(-1).tolist() == [129]


@pytest.mark.parametrize("size", [1e-6, 3e5])
@pytest.mark.parametrize("offsets", [[0, 3000], [0, 20], [0, 1, 2], list(range(0, 40 * 200, 40)), list(range(0, 30 * 160, 30))])
def test_the_range_of_f16(mb, dev, offsets, size):
    """The product of rank R may leave the range of f16 (65504; steps of 2^-24 near zero) where the operands and the result
    do not: its 16-bit parts are taken relative to the row's largest."""
    rows, n, k, rank, count = offsets[-1], 264, 512, 24, 3
    gen = torch.Generator(device=dev).manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)
    up, down = (size ** 0.5 * 0.2, 1.0) if size > 1 else (size ** 0.5, 1.0)
    x, a = (r(rows, k) * up).half(), (r(count, rank, k) * up * k ** -0.5).half()
    b = (r(count, n, rank) * min(down / size, 6e4 / 5)).half()
    which = [i % count for i in range(len(offsets) - 1)]
    edge, w = torch.tensor(offsets, dtype=torch.int32, device=dev), torch.tensor(which, dtype=torch.int32, device=dev)
    c = r(rows, n)
    d = mb.gemm_lora_(torch.empty_like(c), x, a, b, w, edge, C=c)
    assert bool(d.isfinite().all())
    check(d, c, x, a, b, None, which, offsets, torch.float32, d)


def test_an_infinity_stays_one(mb, dev):
    """One infinite product of rank R: the outputs it reaches are infinite, not undefined."""
    for kind in ("f16", "bf16"):
        for rows, k, n in ((1, 64, 40), (20, 64, 40), (300, 64, 40), (6000, 512, 264)):
            x, a, b = torch.ones(rows, k, device=dev).to(DT[kind]), torch.zeros(1, 8, k, device=dev).to(DT[kind]), torch.ones(1, n, 8, device=dev).to(DT[kind])
            x[rows // 2, 0] = float("inf")
            a[0, 3, 0] = 1.0
            a[0, 3, 1] = 1.0
            x[:, 2:] = 0
            d = mb.gemm_lora_(torch.zeros(rows, n, device=dev), x, a[:, 3:4].expand(1, 8, k).contiguous(), b, torch.zeros(1, dtype=torch.int32, device=dev),
                              torch.tensor([0, rows], dtype=torch.int32, device=dev))
            assert bool((d[rows // 2] == float("inf")).all()) and int((~d.isfinite()).any(1).sum()) == 1


def test_beside_a_projection_captured(mb, dev):
    """A decoding step: the shared projection by `gemm_`, the adapters in place behind it, captured once and replayed
    with other tokens and other adapters."""
    rows, n, k, rank, count = 12, 512, 256, 16, 5
    gen = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device=dev) * scale).to(torch.bfloat16)
    x, w, a, b = r(rows, k), r(n, k, scale=k ** -0.5), r(count, rank, k, scale=k ** -0.5), r(count, n, rank, scale=rank ** -0.5)
    which = torch.arange(rows, dtype=torch.int32, device=dev) % (count + 1)
    y = torch.empty(rows, n, dtype=torch.bfloat16, device=dev)

    def step():
        mb.matmul(x, w, y)
        mb.gemm_lora_(y, x, a, b, which)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(2):
        x.copy_(r(rows, k))
        which.copy_((which + i) % (count + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        plain = torch.empty_like(y)
        mb.matmul(x, w, plain)
        check(got, plain, x, a, b, None, which.tolist(), None, torch.bfloat16, got)
    mb.synchronize_status(dev)


def test_same_bits_every_time(mb, dev):
    for case in (CASES[1], CASES[3], TILES[0], TILES[2], TILES[5]):
        x, a, b, scales, w, edge = make(case, "bf16", dev)
        rows, n = case[1], case[3]
        outs = [mb.gemm_lora_(torch.zeros(rows, n, device=dev), x, a, b, w, edge, scales) for _ in range(3)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_no_rows_and_no_requests(mb, dev):
    a, b = torch.ones(2, 8, 16, dtype=torch.bfloat16, device=dev), torch.ones(2, 24, 8, dtype=torch.bfloat16, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    mb.gemm_lora_(torch.empty(0, 24, device=dev), torch.empty(0, 16, dtype=torch.bfloat16, device=dev), a, b, none)
    d = torch.full((3, 24), 5.0, device=dev)
    x = torch.ones(3, 16, dtype=torch.bfloat16, device=dev)
    mb.gemm_lora_(d, x, a, b, none, torch.zeros(1, dtype=torch.int32, device=dev))
    mb.gemm_lora_(d, x, a, b, torch.zeros(2, dtype=torch.int32, device=dev), torch.tensor([-5, 0, 0], dtype=torch.int32, device=dev))
    assert bool((d == 5).all())
    # borders behind the array's end stop at it, borders that run backwards make an empty request
    mb.gemm_lora_(d, x, a, b, torch.zeros(3, dtype=torch.int32, device=dev), torch.tensor([-5, 2, 1, 99], dtype=torch.int32, device=dev))
    mb.synchronize_status(dev)
    assert bool((d == 5 + 16 * 8).all())


def test_refusals(mb, dev):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    which, edge = torch.zeros(2, dtype=torch.int32, device=dev), torch.tensor([0, 1, 4], dtype=torch.int32, device=dev)

    def refused(code, *args, **kw):
        with pytest.raises(mb.MoyeError) as e:
            mb.gemm_lora_(*args, **kw)
        assert e.value.code == code, str(e.value)

    ok = (z(4, 32), z(4, 64), z(3, 16, 64), z(3, 32, 16), which, edge)
    mb.gemm_lora_(*ok)
    for code, i, bad in ((-4, 0, z(4, 40)), (-4, 1, z(5, 64)), (-4, 2, z(2, 16, 64)), (-4, 3, z(3, 32, 8)), (-4, 2, z(16, 64)),
                         (-2, 0, z(4, 32, dtype=torch.float16)), (-2, 1, z(4, 64, dtype=torch.float16)), (-2, 3, z(3, 32, 16, dtype=torch.float32)),
                         (-3, 0, z(32, 4).t()), (-3, 1, z(64, 4).t()), (-3, 2, z(3, 64, 16).transpose(1, 2)), (-3, 3, z(1, 32, 16).expand(3, 32, 16)),
                         (-5, 1, z(4, 68)[:, :64]), (-5, 2, z(3, 16, 68)[:, :, :64]), (-5, 3, z(3, 32, 20)[:, :, :16]),
                         (-1, 4, which.long()), (-4, 5, edge[:2]), (-1, 5, edge.long())):
        args = list(ok)
        args[i] = bad
        refused(code, *args)
    refused(-4, z(4, 32), z(4, 64), z(3, 12, 64), z(3, 32, 12), which, edge)        # rank 12
    refused(-4, z(4, 32), z(4, 64), z(3, 136, 64), z(3, 32, 136), which, edge)      # rank 136
    refused(-4, z(4, 32), z(4, 60), z(3, 16, 60), z(3, 32, 16), which, edge)        # K = 60
    refused(-1, z(4, 32), z(4, 64), z(3, 16, 64), z(3, 32, 16), which)              # 2 requests, 4 rows, no borders
    refused(-4, *ok, scales=torch.ones(2, device=dev))
    refused(-1, *ok, scales=torch.ones(3, device=dev, dtype=torch.float64))
    refused(-2, *ok, C=z(4, 32, dtype=torch.float32))
    refused(-4, *ok, C=z(4, 40))
    torch.cuda.synchronize()


# requests, K, N, R: a row each, turned tiles on several CTAs and on one, longer tiles on several CTAs and on one
SCALED = [(list(range(0, 9)), 512, 264, 24), (list(range(0, 601, 30)), 4096, 1000, 24), (list(range(0, 4801, 30)), 512, 264, 24),
          ([0, 150, 300], 2048, 4096, 64), (list(range(0, 8001, 40)), 512, 264, 24)]


@pytest.mark.parametrize("out", ["same", "f32"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(SCALED)))
def test_scales_of_any_size_and_rows_of_zeros(mb, dev, case, kind, out):
    """Scales far from 1, negative and zero; rows of X and an adapter that are zero leave C as it is, whatever the scale."""
    offsets, k, n, rank = SCALED[case]
    rows, requests, size = offsets[-1], len(offsets) - 1, [4.0, 64.0, -8.0, 0.0, 1e30, -2.0 ** -40]
    ot = DT[kind] if out == "same" else torch.float32
    which = [i % len(size) for i in range(requests)]
    x, a, b, _, w, edge = make((offsets, rows, which, n, k, rank, len(size)), kind, dev)
    x[::3] = 0
    x[1] = torch.finfo(DT[kind]).tiny  # a row whose product is far below 1
    a[4] = 0
    scales = torch.tensor(size, device=dev)
    c = torch.randn(rows, n, device=dev).to(ot)
    got = mb.gemm_lora_(torch.full_like(c, float("nan")), x, a, b, w, edge, scales, C=c)
    mb.synchronize_status(dev)
    assert torch.equal(got[::3], c[::3])
    for q, i in enumerate(which):
        s = slice(offsets[q], offsets[q + 1])
        if size[i] == 0 or i == 4:
            assert torch.equal(got[s], c[s])
        add = size[i] * ((x[s].double() @ a[i].double().T) @ b[i].double().T)
        mag = abs(size[i]) * ((x[s].double().abs() @ a[i].double().abs().T) @ b[i].double().abs().T)
        want = c[s].double() + add
        tol = (k + rank + 4) * 2.0 ** -23 * (mag + c[s].double().abs())
        if ot != torch.float32:
            tol = tol + 2.0 ** -16 * mag + torch.finfo(ot).eps / 2 * want.abs() + torch.finfo(ot).tiny * torch.finfo(ot).eps
        assert bool(((got[s].double() - want).abs() <= tol).all())


def running(offsets, rows):
    """Borders inside the array, none below an earlier one."""
    out, high = [], 0
    for o in offsets:
        high = max(high, min(max(o, 0), rows))
        out.append(high)
    return out


# the last three reach the tiles of the tensor cores: two requests that ask for the same rows, borders that fall by one
# in the middle of 400 requests (more than the CTA has threads), and a first border behind the rest
BACKWARDS = [([0, 4, 1, 3, 9], 12, 64, 136, 16), ([-3, 5, 2, 7, 99], 9, 64, 136, 16), ([6, 2, 4, 8], 9, 64, 136, 16),
             ([0, 3000, 0, 3000], 3000, 1024, 1000, 64),
             ([40 * i - 41 * (i % 50 == 49) for i in range(401)], 16000, 512, 264, 24),
             ([700, 0, 300, 1200, 1100, 2000, 5000], 3000, 1024, 131, 64)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(BACKWARDS)))
def test_borders_that_run_backwards(mb, dev, case, in_place):
    """Every row belongs to one request at most, the same in both kernels, and is added to once."""
    offsets, rows, k, n, rank = BACKWARDS[case]
    which = [i % 5 - 1 for i in range(1, len(offsets))]
    x, a, b, scales, w, edge = make((offsets, rows, which, n, k, rank, 4), "bf16", dev)
    c = torch.randn(rows, n, device=dev)
    d0 = c.clone() if in_place else torch.full_like(c, -3.0)
    got = mb.gemm_lora_(d0.clone(), x, a, b, w, edge, scales, C=None if in_place else c)
    if in_place:
        got2 = c.clone()
        mb.gemm_lora_(got2, x, a, b, w, edge, scales, C=got2)
        assert torch.equal(got, got2)
    mb.synchronize_status(dev)
    check(got, c, x, a, b, scales, which, running(offsets, rows), torch.float32, d0)


@pytest.mark.parametrize("case", [([0, 3, 9], 9, [1, 0], 64, 64, 16, 2), ([0, 3000], 3000, [1], 520, 520, 64, 2)])
def test_columns_of_one_wider_array(mb, dev, case):
    offsets, rows, which, n, k, rank, count = case
    x, a, b, scales, w, edge = make(case, "bf16", dev)
    c = torch.randn(rows, n, device=dev).bfloat16()
    wide = torch.zeros(rows, k + 2 * n, dtype=torch.bfloat16, device=dev)
    xs, cs, d = wide[:, :k], wide[:, k:k + n], wide[:, k + n:]
    xs.copy_(x)
    cs.copy_(c)
    got = mb.gemm_lora_(d, xs, a, b, w, edge, scales, C=cs)
    mb.synchronize_status(dev)
    check(got, c, x, a, b, scales, which, offsets, torch.bfloat16, d)
    assert torch.equal(xs, x) and torch.equal(cs, c)
    for kw in ({"C": wide[:, k + n - 8:k + 2 * n - 8]}, {"C": None}):
        with pytest.raises(mb.MoyeError) as e:
            mb.gemm_lora_(d if kw["C"] is not None else wide[:, k - 8:k + n - 8], xs, a, b, w, edge, scales, **kw)
        assert e.value.code == -1


@pytest.mark.parametrize("case", range(len(SCALED)))
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_an_infinite_factor_beside_large_values(mb, dev, kind, case):
    """An adapter with one infinite element: its product of rank R is infinite beside finite ones above the range of f16
    and of the other sign, and the sum is infinite, not undefined.  Requests of the other adapter have finite sums."""
    offsets, k, n, rank = SCALED[case]
    rows, requests = offsets[-1], len(offsets) - 1
    x, a, b = (torch.zeros(*s, dtype=DT[kind], device=dev) for s in ((rows, k), (2, rank, k), (2, n, rank)))
    x[:, 0], x[:, 1] = 1.0, 256.0
    a[0, 0, 0], a[1, 0, 0], a[:, 1:, 1] = float("inf"), 1.0, 32768.0   # the first product infinite or 1, the others 2^23
    b[:] = -1.0
    b[:, :, 0] = 1.0
    which = (torch.arange(requests, device=dev) % 2).to(torch.int32)
    d = mb.gemm_lora_(torch.zeros(rows, n, device=dev), x, a, b, which, torch.tensor(offsets, dtype=torch.int32, device=dev))
    mb.synchronize_status(dev)
    mine = which.repeat_interleave(torch.tensor(offsets, device=dev).diff())
    assert bool((d[mine == 0] == float("inf")).all())
    # 1 - (R - 1) 2^23, a sum of R terms in fp32: off by at most (R + 4) * 2^-23 of the magnitudes
    assert bool(((d[mine == 1].double() - (1 - (rank - 1) * 2.0 ** 23)).abs() <= (rank + 4) * 2.0 ** -23 * rank * 2.0 ** 23).all())
