"""The row-group calls' compiled way into the library (csrc/calls.cpp) beside the way through ctypes: the same entry points,
hence the same bits; what the compiled way does not take, the other one does or refuses."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def everything(mb, dev, stream=None, wrap=lambda x: x):
    """One call of each operator on seeded inputs; the results."""
    gen = torch.Generator(device=dev).manual_seed(7)
    r = lambda *s, dtype=torch.bfloat16: torch.randn(*s, generator=gen, device=dev).to(dtype)
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device=dev, dtype=dtype)
    ids = torch.randint(-1, 5, (70, 3), generator=gen, device=dev)
    x, w1, weights = r(70, 64), r(5, 48, 64), r(70, 3, dtype=torch.float32)
    a, b, which = r(4, 16, 64), r(4, 48, 16), torch.tensor([3, -1, 0], dtype=torch.int32, device=dev)
    edge, scales, c = torch.tensor([0, 1, 30, 69], dtype=torch.int32, device=dev), r(4, dtype=torch.float32), r(70, 48)
    torch.cuda.synchronize()
    s = None if stream is None else stream.cuda_stream
    plan = mb.group_rows(ids, 5)
    torch.cuda.synchronize()
    if s is not None:
        mb.group_rows_(plan, ids, stream=s)
    xs, ys, y, dys, dw, dx, dw1, d, e = z(210, 64), z(210, 48), z(70, 48), z(210, 48), z(70, 3, dtype=torch.float32), z(210, 64), z(5, 48, 64), z(70, 48), c.clone()
    torch.cuda.synchronize()
    mb.gather_rows_(wrap(xs), x, plan, stream=s)
    mb.gemm_grouped_(wrap(ys), xs, w1, plan, alpha=0.5, stream=s)
    mb.combine_rows_(wrap(y), ys, plan, weights, stream=s)
    mb.combine_rows_grad_(wrap(dys), dw, y, ys, plan, weights, stream=s)
    mb.gemm_grouped_(wrap(dx), dys, w1.transpose(1, 2), plan.offsets, stream=s)
    mb.gemm_grouped_grad_(wrap(dw1), dys, xs, plan, 1, 0, stream=s)
    mb.gemm_lora_(wrap(d), x, a, b, which, edge, scales=scales, C=c, stream=s)
    mb.gemm_lora_(wrap(e), x, a, b, torch.arange(70, dtype=torch.int32, device=dev) % 5, stream=s)
    torch.cuda.synchronize()
    mb.synchronize_status(dev)
    n = int(plan.offsets[-1])
    return [plan.order, plan.offsets, plan.inverse, xs[:n], ys[:n], y, dys[:n], dw, dx[:n], dw1, d, e]


def same(p, q):
    return all(torch.equal(u, v) for u, v in zip(p, q))


def test_both_ways_give_the_same_bits(mb, dev, monkeypatch):
    mb.synchronize_status(dev)  # the library is loaded, this thread has its handle
    assert mb._lib.calls is not None
    assert mb._lib.calls.gather_rows(torch.zeros(2, 8, device=dev), torch.zeros(2, 8, device=dev),
                                     torch.zeros(7, dtype=torch.int32, device=dev), 2, 1, None) in (0, 1)
    taken = everything(mb, dev)
    side = torch.cuda.Stream(dev)
    assert same(taken, everything(mb, dev, side))
    assert same(taken, everything(mb, dev, wrap=mb.MoYeArray))  # no tensors: the way through ctypes
    monkeypatch.setattr(mb._lib, "calls", None)
    assert same(taken, everything(mb, dev))


def test_the_compiled_way_is_taken(mb, dev, monkeypatch):
    everything(mb, dev)

    def never(*args):
        raise AssertionError("the call went through ctypes")

    monkeypatch.setattr(mb.grouped, "_call", never)
    everything(mb, dev)


def test_a_new_thread_and_the_current_stream(mb, dev):
    want = everything(mb, dev)
    got = []

    def work():
        side = torch.cuda.Stream(dev)
        for _ in range(2):  # first without a handle of this thread, then with one
            with torch.cuda.stream(side):
                got.append(everything(mb, dev))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(same(want, g) for g in got)


def test_a_captured_call_follows_the_capturing_stream(mb, dev):
    ids = torch.zeros(9, 2, dtype=torch.int64, device=dev)
    x, xs = torch.randn(9, 32, device=dev), torch.zeros(18, 32, device=dev)
    plan = mb.group_rows(ids, 4)
    mb.gather_rows_(xs, x, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mb.group_rows_(plan, ids)
        mb.gather_rows_(xs, x, plan)
        inside = mb.group_rows(ids, 4)  # its tensors are the graph's
    ids.copy_(torch.arange(18, device=dev).view(9, 2) % 4)
    xs.zero_()
    graph.replay()
    torch.cuda.synchronize()
    order = torch.argsort(ids.flatten(), stable=True)
    assert torch.equal(plan.order.long(), order) and torch.equal(inside.order.long(), order)
    assert torch.equal(xs, x[order // 2])


def test_errors_of_the_compiled_way(mb, dev):
    everything(mb, dev)
    f = lambda *s: torch.zeros(*s, device=dev)
    plan = mb.group_rows(torch.zeros(4, 2, dtype=torch.int64, device=dev), 3)
    both = f(8, 16)
    for code, call in ((-1, lambda: mb.gather_rows_(both, both[4:], plan)), (-3, lambda: mb.gather_rows_(f(16, 8).t(), f(4, 16), plan)),
                       (-2, lambda: mb.group_rows(f(4), 3)), (-4, lambda: mb.group_rows_(plan, torch.zeros(3, 2, dtype=torch.int64, device=dev)))):
        with pytest.raises(mb.MoyeError) as e:
            call()
        assert e.value.code == code and str(e.value)
    for bad in (None, 3, "x", [1.0]):
        with pytest.raises((TypeError, AttributeError)):
            mb.gather_rows_(bad, f(4, 16), plan)
        with pytest.raises((TypeError, AttributeError)):
            mb.group_rows(bad, 3)
    with pytest.raises((TypeError, ValueError)):
        mb.gemm_grouped_(f(4, 8).half(), f(4, 8).half(), f(3, 8, 8).half(), plan, alpha="one")
    with pytest.raises(OverflowError):
        mb.gemm_grouped_(f(4, 8).half(), f(4, 8).half(), f(3, 8, 8).half(), plan, alpha=10 ** 400)
    torch.cuda.synchronize()
