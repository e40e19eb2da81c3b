"""Rows sorted by group and back on the GPU: `group_rows`, `gather_rows_`, `combine_rows_`, `combine_rows_grad_` against
plain 64-bit forms.  Whole numbers have to be equal.  A value is a sum of `c` products in fp32 and one rounding to the
element type: off by at most (c + 1) * 2^-24 of the sum of magnitudes, and eps / 2 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# tokens, choices, groups, width, type: one row, odd and unaligned widths, more entries than one CTA sorts, the most groups
CASES = [(1, 1, 1, 8, "bf16"), (1, 8, 8, 5000, "f16"), (5, 3, 4, 1, "f32"), (33, 2, 7, 130, "bf16"), (300, 1, 1, 64, "f32"),
         (2039, 3, 17, 101, "f32"), (513, 8, 128, 2048, "bf16"), (700, 9, 1024, 33, "f16"), (4100, 2, 1024, 16, "bf16"),
         (97, 20, 31, 520, "f32"), (50, 40, 9, 264, "bf16"), (12, 67, 5, 33, "f16")]


def ids_for(tokens, choices, groups, seed, dtype=torch.int64, dropped=0.2):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, groups, (tokens, choices), generator=gen)
    out = torch.tensor([-1, groups, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (tokens, choices), generator=gen)]
    return torch.where(torch.rand(tokens, choices, generator=gen) < dropped, out, ids).to(dtype)


def sorted_by_hand(ids, groups):
    flat = ids.reshape(-1).tolist()
    order = [i for g in range(groups) for i, v in enumerate(flat) if v == g] if groups <= 64 else \
        sorted((i for i, v in enumerate(flat) if 0 <= v < groups), key=lambda i: flat[i])
    counts = [0] * groups
    inverse = [-1] * len(flat)
    for p, i in enumerate(order):
        counts[flat[i]] += 1
        inverse[i] = p
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    return order + [-1] * (len(flat) - len(order)), offsets, inverse


def close(got, want, mag, terms, dtype):
    """|got - want| <= (terms + 1) * 2^-24 * mag + eps / 2 * |want| (+ the smallest step of f16)."""
    tol = (terms + 1) * 2.0 ** -24 * mag + (torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
                                            if dtype != torch.float32 else 0)
    return bool(((got.double() - want).abs() <= tol).all())


def data(tokens, choices, width, dtype, dev, seed=3):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)
    return (r(tokens, width).to(dtype), r(tokens * choices, width).to(dtype), torch.softmax(r(tokens, choices), 1), r(tokens, width).to(dtype))


@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,choices,groups", [(0, 2, 5), (1, 1, 1), (31, 3, 4), (4096, 1, 64), (4097, 1, 64), (700, 9, 1024), (20000, 8, 128), (33000, 1, 1024)])
def test_group_rows(mb, dev, tokens, choices, groups, id_type):
    ids = ids_for(tokens, choices, groups, 5, id_type)
    plan = mb.group_rows(ids.to(dev), groups)
    order, offsets, inverse = sorted_by_hand(ids, groups)
    assert plan.order.tolist() == order and plan.offsets.tolist() == offsets and plan.inverse.reshape(-1).tolist() == inverse
    # the plan is filled again in place, from a strided view and from one column
    wide = ids_for(tokens, choices + 2, groups, 6, id_type).to(dev)
    mb.group_rows_(plan, wide[:, 1:choices + 1])
    order, offsets, inverse = sorted_by_hand(wide[:, 1:choices + 1].cpu(), groups)
    assert plan.order.tolist() == order and plan.offsets.tolist() == offsets and plan.inverse.reshape(-1).tolist() == inverse
    one = mb.group_rows(wide[:, 0], groups)
    assert one.order.tolist() == sorted_by_hand(wide[:, :1].cpu(), groups)[0] and one.inverse.shape == (tokens, 1)


def test_group_rows_extremes(mb, dev):
    for ids, groups in ((torch.full((9000,), 3), 7), (torch.full((50, 2), -1), 3), (torch.arange(1024).flip(0), 1024)):
        plan = mb.group_rows(ids.to(dev), groups)
        order, offsets, inverse = sorted_by_hand(ids, groups)
        assert plan.order.tolist() == order and plan.offsets.tolist() == offsets and plan.inverse.reshape(-1).tolist() == inverse


@pytest.mark.parametrize("tokens,choices,groups,width,kind", CASES)
def test_there_and_back(mb, dev, tokens, choices, groups, width, kind):
    dt = DT[kind]
    ids = ids_for(tokens, choices, groups, 7)
    plan = mb.group_rows(ids.to(dev), groups)
    x, ys, w, dy = data(tokens, choices, width, dt, dev)
    inv = plan.inverse.long()
    kept = int(plan.offsets[-1])
    assert kept == int((inv >= 0).sum())
    has = inv >= 0

    xs = torch.full_like(ys, float("nan"))
    assert mb.gather_rows_(xs, x, plan) is xs
    assert torch.equal(xs[:kept], x[plan.order[:kept].long() // choices]) and bool(xs[kept:].isnan().all())

    mine = torch.where(has[:, :, None], ys.double()[inv.clamp(min=0)], 0.0)
    for weights in (w, w.to(torch.float16), w.to(torch.bfloat16), None):
        ww = torch.ones(tokens, choices, dtype=torch.float64, device=dev) if weights is None else weights.double()
        out = torch.full((tokens, width), float("nan"), dtype=dt, device=dev)
        mb.combine_rows_(out, ys, plan, weights)
        terms = mine * ww[:, :, None]
        assert close(out, terms.sum(1), terms.abs().sum(1), choices, dt)

    d_ys, d_w = torch.full_like(ys, float("nan")), torch.full_like(w, float("nan"))
    mb.combine_rows_grad_(d_ys, d_w, dy, ys, plan, w)
    assert bool(d_ys[kept:].isnan().all())
    want = dy.double()[plan.order[:kept].long() // choices] * w.double().reshape(-1)[plan.order[:kept].long()][:, None]
    assert close(d_ys[:kept], want, want.abs(), 1, dt)
    prod = mine * dy.double()[:, None, :]
    # a dot product of `width` terms in fp32, in any order
    assert bool(((d_w.double() - prod.sum(2)).abs() <= (width + 1) * 2.0 ** -24 * prod.abs().sum(2)).all())
    assert bool((d_w[~has] == 0).all())


def test_gradients_against_differences(mb, dev):
    """combine is linear in the rows and in the weights: a difference of its outputs is the derivative up to rounding.
    Every output is off by at most 4 * 2^-24 of a sum of magnitudes below 64 here, a difference over a step of 1 by twice
    that times the 24 outputs' |dy| <= 5: below 24 * 5 * 2 * 4 * 64 * 2^-24 = 0.0037."""
    tokens, choices, width = 6, 3, 4
    plan = mb.group_rows(ids_for(tokens, choices, 5, 11).to(dev), 5)
    x, ys, w, dy = data(tokens, choices, width, torch.float32, dev)

    def value(ys, w):
        return float((mb.combine_rows_(torch.empty_like(x), ys, plan, w).double() * dy.double()).sum())

    d_ys, d_w = mb.combine_rows_grad_(torch.zeros_like(ys), torch.empty_like(w), dy, ys, plan, w)
    base = value(ys, w)
    for t, d in ((ys, d_ys), (w, d_w)):
        for i in range(t.numel()):
            moved = t.clone()
            moved.view(-1)[i] += 1.0
            got = value(moved, w) - base if t is ys else value(ys, moved) - base
            assert abs(got - float(d.reshape(-1)[i])) < 0.0037
    # gather's gradient: <gather(x), g> moved along x
    g = torch.randn_like(ys)
    kept = int(plan.offsets[-1])
    dx = mb.combine_rows_(torch.empty_like(x), g, plan)
    for i in range(x.numel()):
        moved = x.clone()
        moved.view(-1)[i] += 1.0
        f = [(mb.gather_rows_(torch.zeros_like(ys), v, plan)[:kept].double() * g[:kept].double()).sum() for v in (moved, x)]
        assert abs(float(f[0] - f[1]) - float(dx.view(-1)[i])) < 0.0037


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.int16, torch.int64])
@pytest.mark.parametrize("width", [48, 50])
def test_gather_moves_any_element(mb, dev, dtype, width):
    plan = mb.group_rows(ids_for(70, 2, 6, 13).to(dev), 6)
    raw = torch.randint(0, 127, (70, width), device=dev, dtype=torch.int8).repeat_interleave(torch.empty(0, dtype=dtype).element_size(), 1)
    src = raw.view(dtype)
    dst = torch.zeros(140, width, dtype=torch.int8, device=dev).to(dtype) if dtype != torch.float8_e4m3fn else \
        torch.zeros(140, width, dtype=torch.int8, device=dev).view(dtype)
    mb.gather_rows_(dst, src, plan)
    kept = int(plan.offsets[-1])
    assert torch.equal(dst.view(torch.int8)[:kept], raw[plan.order[:kept].long() // 2])


def test_pitched_and_unaligned_views(mb, dev):
    tokens, choices, width = 61, 2, 96
    plan = mb.group_rows(ids_for(tokens, choices, 5, 17, dropped=0.0).to(dev), 5)
    for shift in (8, 3):   # rows on 16 bytes, and rows on none
        x = torch.randn(tokens, 2 * width, device=dev).to(torch.bfloat16)[:, shift:shift + width]
        big = torch.full((tokens * choices, 2 * width), 7.0, dtype=torch.bfloat16, device=dev)
        xs = big[:, shift:shift + width]
        mb.gather_rows_(mb.MoYeArray(xs), mb.MoYeArray(x), plan)
        assert torch.equal(xs, x[plan.order.long() // choices])
        assert bool((big[:, :shift] == 7).all()) and bool((big[:, shift + width:] == 7).all())
        out = torch.full((tokens, 2 * width), 7.0, dtype=torch.bfloat16, device=dev)
        w = torch.rand(choices, tokens, device=dev).t()          # a transposed view
        mb.combine_rows_(out[:, shift:shift + width], xs, plan, w)
        terms = xs.double()[plan.inverse.long()] * w.double()[:, :, None]
        assert close(out[:, shift:shift + width], terms.sum(1), terms.abs().sum(1), choices, torch.bfloat16)
        assert bool((out[:, :shift] == 7).all()) and bool((out[:, shift + width:] == 7).all())


def test_broadcast_inputs(mb, dev):
    """A gradient that is the same for all tokens (an expanded row) is read as it is."""
    plan = mb.group_rows(ids_for(30, 2, 4, 29).to(dev), 4)
    x, ys, w, dy = data(30, 2, 64, torch.float32, dev)
    one = dy[:1].expand(30, 64)
    got = mb.combine_rows_grad_(torch.zeros_like(ys), torch.empty_like(w), one, ys, plan, w)
    want = mb.combine_rows_grad_(torch.zeros_like(ys), torch.empty_like(w), one.contiguous(), ys, plan, w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(mb.gather_rows_(torch.zeros_like(ys), one, plan), mb.gather_rows_(torch.zeros_like(ys), one.contiguous(), plan))
    with pytest.raises(mb.MoyeError):
        mb.combine_rows_(torch.zeros(1, 64, device=dev).expand(30, 64), ys, plan)


def test_infinities_stay_in_their_rows(mb, dev):
    ids = torch.tensor([[0, 1], [1, -1], [-1, -1], [2, 0]], device=dev)
    plan = mb.group_rows(ids, 3)
    ys = torch.ones(8, 16, device=dev)
    ys[int(plan.inverse[0, 0])] = float("inf")
    ys[int(plan.offsets[-1]):] = float("nan")
    out = mb.combine_rows_(torch.empty(4, 16, device=dev), ys, plan, torch.ones(4, 2, device=dev))
    assert bool(out[0].isinf().all()) and bool((out[1] == 1).all()) and bool((out[2] == 0).all()) and bool((out[3] == 2).all())


def test_another_stream_and_a_captured_replay(mb, dev):
    tokens, choices, groups, width = 300, 4, 16, 256
    ids = ids_for(tokens, choices, groups, 19).to(dev)
    plan = mb.group_rows(ids, groups)
    x, ys, w, _ = data(tokens, choices, width, torch.bfloat16, dev)
    xs, out = torch.zeros_like(ys), torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mb.group_rows_(plan, ids)
        mb.gather_rows_(xs, x, plan)
        mb.combine_rows_(out, xs, plan, w)
    torch.cuda.synchronize()
    first = (xs.clone(), out.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mb.group_rows_(plan, ids)
        mb.gather_rows_(xs, x, plan)
        mb.combine_rows_(out, xs, plan, w)
    for seed in (19, 23):
        ids.copy_(ids_for(tokens, choices, groups, seed))
        xs.zero_()
        graph.replay()
        torch.cuda.synchronize()
        fresh = mb.group_rows(ids, groups)
        assert torch.equal(plan.order, fresh.order) and torch.equal(plan.offsets, fresh.offsets) and torch.equal(plan.inverse, fresh.inverse)
        want = mb.gather_rows_(torch.zeros_like(xs), x, fresh)
        assert torch.equal(xs, want) and torch.equal(out, mb.combine_rows_(torch.empty_like(x), want, fresh, w))
        if seed == 19:
            assert torch.equal(xs, first[0]) and torch.equal(out, first[1])


def test_refusals(mb, dev):
    f = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)
    ids = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    plan = mb.group_rows(ids, 3)

    def refused(code, fn, *args, **kw):
        with pytest.raises(mb.MoyeError) as e:
            fn(*args, **kw)
        assert e.value.code == code, str(e.value)

    refused(-4, mb.group_rows, ids, 0)
    refused(-4, mb.group_rows, ids, 1025)
    refused(-2, mb.group_rows, ids.float(), 3)
    refused(-4, mb.group_rows_, plan, ids[:3])
    refused(-4, mb.gather_rows_, f(7, 16), f(4, 16), plan)            # not tokens * choices rows
    refused(-4, mb.gather_rows_, f(8, 16), f(4, 8), plan)
    refused(-2, mb.gather_rows_, f(8, 16), f(4, 16, dtype=torch.float32), plan)
    refused(-3, mb.gather_rows_, f(16, 8).t(), f(4, 16), plan)        # rows of dst are not contiguous
    for n in (3, 5):                                                   # not the plan's tokens
        refused(-4, mb.gather_rows_, f(2 * n, 16), f(n, 16), plan)
        refused(-4, mb.combine_rows_, f(n, 16), f(2 * n, 16), plan)
        wn = torch.zeros(n, 2, device=dev)
        refused(-4, mb.combine_rows_grad_, f(2 * n, 16), wn, f(n, 16), f(2 * n, 16), plan, wn)
    both = f(8, 16)
    refused(-1, mb.gather_rows_, both, both[4:], plan)                # overlap
    refused(-1, mb.combine_rows_, both[:4], both, plan)
    refused(-2, mb.combine_rows_, f(4, 16, dtype=torch.int16), f(8, 16, dtype=torch.int16), plan)
    refused(-4, mb.combine_rows_, f(4, 16), f(8, 16), plan, torch.zeros(4, 3, device=dev))
    refused(-2, mb.combine_rows_, f(4, 16), f(8, 16), plan, torch.zeros(4, 2, device=dev, dtype=torch.int32))
    w = torch.zeros(4, 2, device=dev)
    refused(-2, mb.combine_rows_grad_, f(8, 16), w.half(), f(4, 16), f(8, 16), plan, w)
    refused(-1, mb.combine_rows_grad_, both, w.clone(), f(4, 16), both, plan, w)
    with pytest.raises(RuntimeError):
        mb.gather_rows_(torch.zeros(8, 16), torch.zeros(4, 16), plan)
    torch.cuda.synchronize()


def test_an_element_of_its_own_for_every_weight_gradient(mb, dev):
    ids = torch.zeros(4, 2, dtype=torch.int64, device=dev)
    plan = mb.group_rows(ids, 3)
    ones, w = torch.ones(8, 16, device=dev), torch.ones(4, 2, device=dev)
    z = lambda *s: torch.zeros(*s, device=dev)
    for bad in (z(4, 1).expand(4, 2), z(1, 2).expand(4, 2), z(1, 1).expand(4, 2), z(9).as_strided((4, 2), (1, 1)), z(9).as_strided((4, 2), (1, 2)),
                z(9).as_strided((4, 2), (2, 2))):
        with pytest.raises(mb.MoyeError) as e:
            mb.combine_rows_grad_(z(8, 16), bad, ones[:4], ones, plan, w)
        assert e.value.code == -3, str(e.value)
    for good in (z(4, 2), z(2, 4).t(), z(8, 6)[::2, 1::4], z(3, 9).t()[:8:2, :2]):
        mb.combine_rows_grad_(z(8, 16), good, ones[:4], ones, plan, w)
        assert bool((good == 16).all())
    one = mb.group_rows(ids[:1], 3)   # a single token, a single choice: their strides say nothing
    for shape, stride, p in (((1, 2), (0, 1), one), ((4, 1), (2, 0), mb.group_rows(ids[:, 0], 3))):
        good = z(8).as_strided(shape, stride)
        n = shape[0] * shape[1]
        mb.combine_rows_grad_(z(n, 16), good, ones[:shape[0]], ones[:n], p, w[:shape[0], :shape[1]])
        assert bool((good == 16).all())
    mb.synchronize_status(dev)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("choices", [2, 5])
def test_rows_of_width_zero(mb, dev, choices, kind):
    """Nothing to move; the gradients of the weights are empty sums."""
    ids = ids_for(7, choices, 3, 31).to(dev)
    plan = mb.group_rows(ids, 3)
    x, ys = torch.empty(7, 0, dtype=DT[kind], device=dev), torch.empty(7 * choices, 0, dtype=DT[kind], device=dev)
    w, dw = torch.ones(7, choices, device=dev), torch.full((7, choices), float("nan"), device=dev)
    mb.gather_rows_(ys, x, plan)
    mb.combine_rows_(x, ys, plan, w)
    mb.combine_rows_grad_(ys, dw, x, ys, plan, w)
    mb.combine_rows_grad_(ys.clone(), dw, x, ys, plan, w)
    mb.synchronize_status(dev)
    assert bool((dw == 0).all())


def test_columns_of_one_wider_array(mb, dev):
    """Arrays that lie beside one another in one buffer share no element; shifted by a column they do."""
    tokens, choices, width = 37, 2, 40
    ids = ids_for(tokens, choices, 5, 37).to(dev)
    plan = mb.group_rows(ids, 5)
    x, ys, w, dy = data(tokens, choices, width, torch.bfloat16, dev)
    n = tokens * choices
    wide = torch.zeros(n, 4 * width, dtype=torch.bfloat16, device=dev)
    part = lambda i, rows=n, shift=0: wide[:rows, i * width + shift:(i + 1) * width + shift]
    refused = lambda fn, *args: pytest.raises(mb.MoyeError, fn, *args).value.code == -1
    part(0, tokens).copy_(x)
    mb.gather_rows_(part(1), part(0, tokens), plan)
    kept = int(plan.offsets[-1])
    assert torch.equal(part(1)[:kept], x[plan.order[:kept].long() // choices])
    part(2).copy_(ys)
    part(0, tokens).copy_(dy)
    want = mb.combine_rows_grad_(torch.zeros_like(ys), torch.zeros_like(w), dy, ys, plan, w)
    got = mb.combine_rows_grad_(part(3), torch.zeros_like(w), part(0, tokens), part(2), plan, w)
    assert torch.equal(got[0][:kept], want[0][:kept]) and torch.equal(got[1], want[1])
    mb.combine_rows_(part(0, tokens), part(2), plan, w)
    assert torch.equal(part(0, tokens), mb.combine_rows_(torch.empty_like(x), ys, plan, w))
    for shift in (-1, 1):
        assert refused(mb.gather_rows_, part(1), part(1 + shift, tokens, -shift), plan)
        assert refused(mb.combine_rows_, part(1 + shift, tokens, -shift), part(1), plan, w)
        assert refused(mb.combine_rows_grad_, part(1), w.clone(), part(3, tokens), part(1 + shift, n, -shift), plan, w)
    assert refused(mb.gather_rows_, part(1), wide.view(-1)[:tokens * width].view(tokens, width), plan)  # another pitch, the same memory
    mb.synchronize_status(dev)


def test_weight_gradients_that_interleave(mb, dev):
    """Strides whose rows lie in one another without sharing an element."""
    plan = mb.group_rows(torch.zeros(4, 3, dtype=torch.int64, device=dev), 3)
    ones, w = torch.ones(12, 16, device=dev), torch.ones(4, 3, device=dev)
    for stride in ((5, 2), (2, 9), (7, 3), (3, 4), (4, 3)):
        flat = torch.zeros(64, device=dev)
        mb.combine_rows_grad_(torch.zeros(12, 16, device=dev), flat.as_strided((4, 3), stride), ones[:4], ones, plan, w)
        assert bool((flat.as_strided((4, 3), stride) == 16).all()) and int((flat != 0).sum()) == 12
    for stride in ((4, 2), (2, 3), (3, 3), (2, 6)):
        with pytest.raises(mb.MoyeError) as e:
            mb.combine_rows_grad_(torch.zeros(12, 16, device=dev), torch.zeros(64, device=dev).as_strided((4, 3), stride), ones[:4], ones, plan, w)
        assert e.value.code == -3
    mb.synchronize_status(dev)


@pytest.mark.parametrize("wt", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_gradients_with_16_bit_weights(mb, dev, kind, wt):
    """Weights and their gradients in 16 bits: the dot product of `width` terms in fp32, then one rounding."""
    tokens, choices, width = 130, 5, 72
    plan = mb.group_rows(ids_for(tokens, choices, 9, 41).to(dev), 9)
    x, ys, w, dy = data(tokens, choices, width, DT[kind], dev)
    w = w.to(DT[wt])
    d_ys, d_w = mb.combine_rows_grad_(torch.full_like(ys, float("nan")), torch.full_like(w, float("nan")), dy, ys, plan, w)
    mb.synchronize_status(dev)
    inv, kept = plan.inverse.long(), int(plan.offsets[-1])
    has = inv >= 0
    at = plan.order[:kept].long()
    want = dy.double()[at // choices] * w.double().reshape(-1)[at][:, None]
    assert close(d_ys[:kept], want, want.abs(), 1, DT[kind]) and bool(d_ys[kept:].isnan().all())
    prod = torch.where(has[:, :, None], ys.double()[inv.clamp(min=0)], 0.0) * dy.double()[:, None, :]
    assert close(d_w, prod.sum(2), prod.abs().sum(2), width, DT[wt]) and bool((d_w[~has] == 0).all())
