"""The row-group operators without a GPU: host arrays are refused, descriptors are the ABI's, the entry points check
their handle first."""
import ctypes

import pytest
import torch


def test_host_arrays_are_refused(mb):
    x, y, b = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(3, 16, 16)
    ids, which = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, dtype=torch.int32)
    plan = mb.RowGroups(4, 2, 3, "cpu")
    for call in (lambda: mb.group_rows(ids, 3), lambda: mb.group_rows_(plan, ids), lambda: mb.gather_rows_(y, x, plan),
                 lambda: mb.combine_rows_(x, y, plan), lambda: mb.combine_rows_grad_(y, x, x, y, plan, x),
                 lambda: mb.gemm_grouped_(y, y, b, plan), lambda: mb.gemm_grouped_grad_(b, y, y, plan),
                 lambda: mb.gemm_lora_(x, x, b, b, which)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError):
        mb.gather_rows_([1], x, plan)
    with pytest.raises(TypeError):
        mb.group_rows([1, 2], 3)
    with pytest.raises(mb.MoyeError):
        mb.group_rows(torch.zeros(2, 2, 2, dtype=torch.int64), 3)


def test_plan_shapes(mb):
    p = mb.RowGroups(5, 3, 7, "cpu")
    assert p.order.shape == (15,) and p.inverse.shape == (5, 3) and p.offsets.shape == (8,)
    assert all(t.dtype == torch.int32 and t.is_contiguous() for t in (p.order, p.inverse, p.offsets))
    spans = sorted((t.data_ptr(), t.data_ptr() + 4 * t.numel()) for t in (p.order, p.inverse, p.offsets))
    assert spans[0][1] <= spans[1][0] and spans[1][1] <= spans[2][0]


@pytest.mark.parametrize("rank", [1, 2, 3, 4])
def test_packed_descriptor_is_the_structure(mb, rank):
    shape, stride = [3 + i for i in range(rank)], [1000 ** (i + 1) for i in range(rank)]
    packed = mb._lib.pack_tensor(0x7F0000001230, mb._lib.BF16, shape, stride)
    assert packed == bytes(mb._lib.make_tensor(0x7F0000001230, mb._lib.BF16, shape, stride))
    assert len(packed) == ctypes.sizeof(mb._lib.Tensor)


def test_entry_points_check_their_handle(mb):
    lib = mb._lib.load()
    f, z = ctypes.c_float(1), None
    assert lib.moye_b200_group_rows(z, z, 1, z, z, z, z) == -1
    assert lib.moye_b200_gather_rows(z, z, z, z, 1, z) == -1
    assert lib.moye_b200_combine_rows(z, z, z, z, z, 1, z) == -1
    assert lib.moye_b200_combine_rows_grad(z, z, z, z, z, z, z, 1, z) == -1
    assert lib.moye_b200_gemm_grouped(z, z, z, z, z, f, f, z) == -1
    assert lib.moye_b200_gemm_grouped_grad(z, z, z, z, z, f, f, z) == -1
    assert lib.moye_b200_gemm_lora(z, z, z, z, z, z, z, z, 0, z, z) == -1
    assert b"null handle" in lib.moye_b200_last_error()


def test_the_compiled_calls_leave_what_is_not_plain(mb):
    """Arrays that are not on a device, wrong types, wrong argument counts: not taken (1), never an exception or a launch."""
    mb._lib.load()
    calls = mb._lib.calls
    assert calls is not None, "lib/moye_calls.so was not built"
    x, v = torch.zeros(4, 8), torch.zeros(20, dtype=torch.int32)
    for odd in (x, None, 3, "x", torch.zeros(4, 8).to_sparse(), torch.zeros(4, 8, dtype=torch.complex64)):
        assert calls.gather_rows(odd, x, v, 4, 2, None) == 1
        assert calls.combine_rows(x, odd, v, 4, 2, None, None) == 1
        assert calls.combine_rows_grad(x, x, odd, x, v, 4, 2, x, None) == 1
        assert calls.gemm_grouped(odd, x, x, v, 0, 1.0, 0.0, None) == 1
        assert calls.gemm_grouped_grad(x, odd, x, v, 0, 1.0, 0.0, None) == 1
        assert calls.gemm_lora(odd, x, x, x, v, None, None, None, None) == 1
        assert calls.group_rows(odd, v, 4, 2, 3, None) == 1
        assert calls.new_plan(odd, 3) == 1
    assert calls.new_plan(x) == 1 and calls.gather_rows() == 1 and calls.group_rows(v, v, 10 ** 30, 2, 3, None) == 1


def test_without_the_compiled_calls_there_is_the_way_through_ctypes(mb, tmp_path, monkeypatch):
    lib = mb._lib.load()
    monkeypatch.setattr(mb._lib, "LIB_PATH", str(tmp_path / "libmoye_b200.so"))
    assert mb._lib._load_calls(lib) is None                    # not built
    (tmp_path / "moye_calls.so").write_bytes(b"no library")
    assert mb._lib._load_calls(lib) is None                    # cannot be loaded


def test_compiled_calls_for_another_torch_are_not_loaded(mb, tmp_path, monkeypatch):
    """The module reads tensors by torch's layout of them: one that was built for another torch, interpreter or version of
    the library is left alone, and built again."""
    import shutil
    import sys

    lib = mb._lib.load()
    build = sys.modules[mb._lib.calls_marker.__module__]
    own = open(build.OUT_CALLS, "rb").read()
    marker = mb._lib.calls_marker(lib.moye_b200_version())
    assert marker in own and torch.__version__.encode() in marker and sys.implementation.cache_tag.encode() in marker
    monkeypatch.setattr(mb._lib, "LIB_PATH", str(tmp_path / "libmoye_b200.so"))
    other = tmp_path / "moye_calls.so"
    shutil.copy(build.OUT_CALLS, other)
    assert mb._lib._load_calls(lib) is not None
    for a, b in ((torch.__version__, "0" * len(torch.__version__)), (sys.implementation.cache_tag, "x" * len(sys.implementation.cache_tag)),
                 (f"library {lib.moye_b200_version()}", "library 999")):
        other.unlink()  # a file of its own: the one before may be mapped
        other.write_bytes(own.replace(marker, marker.replace(a.encode(), b.encode())))
        assert mb._lib._load_calls(lib) is None
    monkeypatch.setattr(build, "OUT_CALLS", str(other))
    assert marker in open(build.build_calls(), "rb").read()
