"""What the 4-bit and rotary entry points refuse, and which calls have no effect (no GPU needed: nothing is launched)."""
import numpy as np
import pytest


def _host(pkg, shape, itemsize=1, strides=None, shift=0):
    buf = np.zeros(int(np.prod(shape)) * itemsize + 64, dtype=np.uint8)
    addr = (buf.ctypes.data + 15) // 16 * 16 + shift
    return pkg.MemRef(addr, shape, strides, keepalive=buf)


def _coded(pkg, rows, cols):
    return tuple(_host(pkg, shape) for shape in pkg.mxf4_shapes(rows, cols))


@pytest.fixture()
def nothing_launched(hom):
    hom.clear_error()
    before = hom.launch_count()
    yield
    hom.clear_error()
    assert hom.launch_count() == before


def _refused(pkg, code, text, call, *args, **kwargs):
    with pytest.raises(pkg.HomError) as e:
        call(*args, **kwargs)
    assert e.value.code == code and text in e.value.message, e.value


@pytest.mark.parametrize("name,element", [("homQuantizeMxF4F16", 2), ("homQuantizeMxF4F32", 4)])
def test_quantize_refusals(pkg, hom, nothing_launched, name, element):
    call = getattr(hom, name)
    q, s = _coded(pkg, 5, 40)
    x = _host(pkg, (5, 40), element)
    _refused(pkg, 1, "rank 2 or 3", call, None, q, s)
    _refused(pkg, 1, "rank 2 or 3", call, _host(pkg, (200,), element), q, s)
    _refused(pkg, 1, "rank 2 or 3", call, x, None, s)
    _refused(pkg, 1, "contiguous", call, _host(pkg, (5, 40), element, (80, 2)), q, s)
    _refused(pkg, 1, "scales of Q", call, x, q, None)
    _refused(pkg, 1, "scales of Q", call, x, q, _host(pkg, (1, 2, 512)))
    _refused(pkg, 1, "whole blocks", call, x, _host(pkg, (5, 20)), s)
    _refused(pkg, 1, "need codes", call, _host(pkg, (5, 70), element), q, s)
    _refused(pkg, 1, "need codes", call, _host(pkg, (4, 40), element), q, s)
    _refused(pkg, 1, "need codes", call, x, q, s, True)
    _refused(pkg, 2, "transposed", call, _host(pkg, (2, 40, 5), element), *_coded(pkg, 5, 80), True)
    _refused(pkg, 1, "16-byte aligned", call, x, _host(pkg, (5, 32), shift=8), s)
    _refused(pkg, 1, "16-byte aligned", call, x, q, _host(pkg, (1, 1, 512), shift=4))
    _refused(pkg, 1, "aligned to its elements", call, _host(pkg, (5, 40), element, shift=1), q, s)
    _refused(pkg, 2, "2^30", call, pkg.MemRef(16, (1, (1 << 30) + 1)), q, s)
    _refused(pkg, 2, "2^30 rows", call, pkg.MemRef(16, (1 << 20, 1 << 11, 1)), q, s)
    both = _host(pkg, (1024,))
    _refused(pkg, 1, "overlaps", call, pkg.MemRef(both.data_ptr, (5, 40)), pkg.MemRef(both.data_ptr + 64, (5, 32)), s)
    _refused(pkg, 1, "overlaps", call, x, pkg.MemRef(both.data_ptr, (5, 32)), pkg.MemRef(both.data_ptr + 144, (1, 1, 512)))


@pytest.mark.parametrize("name,element", [("homDequantizeMxF4F16", 2), ("homDequantizeMxF4F32", 4)])
def test_dequantize_refusals(pkg, hom, nothing_launched, name, element):
    call = getattr(hom, name)
    q, s = _coded(pkg, 5, 40)
    _refused(pkg, 1, "rank 2 or 3", call, q, s, None)
    _refused(pkg, 1, "do not hold", call, q, s, _host(pkg, (5, 65), element))
    _refused(pkg, 1, "do not hold", call, q, s, _host(pkg, (6, 40), element))
    _refused(pkg, 1, "contiguous", call, q, s, _host(pkg, (5, 40), element, (48, 1)))
    _refused(pkg, 1, "aligned to its elements", call, q, s, _host(pkg, (5, 40), element, shift=1))
    _refused(pkg, 1, "overlaps", call, q, s, pkg.MemRef(q.data_ptr, (5, 40)))


def test_product_refusals(pkg, hom, nothing_launched):
    a, b = _coded(pkg, 6, 64), _coded(pkg, 16, 64)
    d = _host(pkg, (6, 16), 2)
    call = hom.homGemmMxF4F16
    _refused(pkg, 1, "rank 2 or 3", call, None, a[1], *b, None, d)
    _refused(pkg, 1, "scales of A", call, a[0], _host(pkg, (2, 1, 512)), *b, None, d)
    _refused(pkg, 1, "scales of B", call, *a, b[0], _host(pkg, (1, 1, 256)), None, d)
    _refused(pkg, 1, "inner dimensions", call, *a, *_coded(pkg, 16, 96), None, d)
    _refused(pkg, 1, "D must be", call, *a, *b, None, _host(pkg, (6, 8), 2))
    _refused(pkg, 1, "D must be", call, *a, *b, None, _host(pkg, (2, 3, 16), 2))
    _refused(pkg, 1, "contiguous", call, *a, *b, None, _host(pkg, (6, 16), 2, (32, 1)))
    _refused(pkg, 2, "batch 1", call, *a, _host(pkg, (2, 8, 32)), b[1], None, d)
    _refused(pkg, 2, "activation", call, *a, *b, None, d, 2)
    _refused(pkg, 1, "needs a contiguous C", call, *a, *b, None, d, 0, 1.0, 1.0)
    _refused(pkg, 1, "C must be", call, *a, *b, _host(pkg, (3, 16), 2), d, 0, 1.0, 1.0)
    _refused(pkg, 1, "needs a contiguous C", call, *a, *b, _host(pkg, (6, 8), 2), d, 0, 1.0, 1.0)
    _refused(pkg, 1, "16-byte aligned", call, *a, *b, None, _host(pkg, (6, 16), 2, shift=8))
    _refused(pkg, 1, "C is not", call, *a, *b, _host(pkg, (6, 16), 2, shift=8), d, 0, 1.0, 1.0)
    _refused(pkg, 1, "overlaps", call, *a, *b, None, pkg.MemRef(a[0].data_ptr + 16, (6, 16)))
    room = _host(pkg, (7, 16), 2)
    _refused(pkg, 1, "overlaps", call, *a, *b, pkg.MemRef(room.data_ptr + 32, (6, 16)), pkg.MemRef(room.data_ptr, (6, 16)),
             0, 1.0, 1.0)
    _refused(pkg, 2, "K == 0", call, _host(pkg, (6, 0)), _host(pkg, (1, 0, 512)), _host(pkg, (16, 0)),
             _host(pkg, (1, 0, 512)), None, d)


@pytest.mark.parametrize("name,element", [("homRotaryF16", 2), ("homRotaryF32", 4)])
def test_rotary_refusals(pkg, hom, nothing_launched, name, element):
    call = getattr(hom, name)
    x, out = _host(pkg, (2, 3, 4, 8), element), _host(pkg, (2, 3, 4, 8), element)
    f, pos = _host(pkg, (4,), 8), _host(pkg, (2, 3), 8)
    _refused(pkg, 1, "[bs, seq, heads, d]", call, None, None, f, out)
    _refused(pkg, 1, "[bs, seq, heads, d]", call, _host(pkg, (2, 3, 32), element), None, f, out)
    _refused(pkg, 1, "different shapes", call, x, None, f, _host(pkg, (2, 3, 4, 16), element))
    _refused(pkg, 1, "Frequencies", call, x, None, None, out)
    _refused(pkg, 1, "Frequencies", call, x, None, _host(pkg, (0,), 8), out)
    _refused(pkg, 1, "Frequencies", call, x, None, _host(pkg, (4,), 8, (2,)), out)
    _refused(pkg, 1, "a head has 8", call, x, None, _host(pkg, (5,), 8), out)
    big = _host(pkg, (1, 1, 1, 1026), element)
    _refused(pkg, 2, "512 frequencies", call, big, None, _host(pkg, (513,), 8), big)
    for bad in (_host(pkg, (3, 2), 8), _host(pkg, (6,), 8), _host(pkg, (2, 3), 8, (6, 2)), _host(pkg, (2, 3), 8, shift=4)):
        _refused(pkg, 1, "Positions", call, x, bad, f, out)
    for bad in (float("nan"), float("inf")):
        _refused(pkg, 1, "magnitude", call, x, pos, f, out, magnitude=bad)
    _refused(pkg, 1, "last dimension", call, _host(pkg, (2, 3, 4, 8), 2 * element, (192, 64, 16, 2)), None, f, out)
    _refused(pkg, 1, "last dimension", call, x, None, f, _host(pkg, (2, 3, 4, 8), 2 * element, (192, 64, 16, 2)))
    _refused(pkg, 2, "strides", call, _host(pkg, (2, 3, 4, 8), element, (-96, 32, 8, 1)), None, f, out)
    _refused(pkg, 1, "share memory", call, x, None, f, _host(pkg, (2, 3, 4, 8), element, (0, 32, 8, 1)))
    _refused(pkg, 1, "share memory", call, x, None, f, _host(pkg, (2, 3, 4, 8), element, (96, 32, 7, 1)))
    _refused(pkg, 1, "overlaps", call, x, None, f, pkg.MemRef(x.data_ptr + 16 * element, (2, 3, 4, 8)))
    _refused(pkg, 1, "overlaps", call, x, None, pkg.MemRef(out.data_ptr + 16, (4,)), out)
    _refused(pkg, 1, "overlaps", call, x, pkg.MemRef(out.data_ptr + 16, (2, 3)), f, out)
    _refused(pkg, 1, "aligned to its elements", call, _host(pkg, (2, 3, 4, 8), element, shift=1), None, f, out)
    _refused(pkg, 2, "2^30", call, pkg.MemRef(16, ((1 << 30) + 1, 1, 1, 8)), None, f, pkg.MemRef(16, ((1 << 30) + 1, 1, 1, 8)))


def test_rotary_overlap_is_a_matter_of_address_ranges(pkg, hom, nothing_launched):
    """Two groups of heads of one packed buffer share no element and are refused all the same, as are dimensions of Out
    that interleave."""
    packed = _host(pkg, (2, 3, 12, 8), 2)
    query, key = (pkg.MemRef(packed.data_ptr + 2 * 8 * first, (2, 3, 4, 8), (288, 96, 8, 1)) for first in (0, 4))
    f = _host(pkg, (4,), 8)
    _refused(pkg, 1, "overlaps", hom.homRotaryF16, query, None, f, key)
    _refused(pkg, 1, "overlaps", hom.homRotaryF16, key, None, f, query)
    out = _host(pkg, (8, 8), 2)  # pieces of eight at 0, 2, 4 and 3, 5, 7
    _refused(pkg, 1, "share memory", hom.homRotaryF16, _host(pkg, (2, 3, 1, 8), 2), None, f,
             pkg.MemRef(out.data_ptr, (2, 3, 1, 8), (24, 16, 8, 1)))


def test_frequency_refusals(pkg, hom, nothing_launched):
    f = _host(pkg, (4,), 8)
    call = hom.homRotaryFrequencies
    _refused(pkg, 1, "Frequencies", call, None)
    _refused(pkg, 2, "512", call, _host(pkg, (513,), 8))
    for bad in (dict(base=0.0), dict(base=float("inf")), dict(scaling="linear", factor=0.0),
                dict(scaling="base", factor=float("nan")), dict(scaling="parts", factor=2.0),
                dict(scaling="parts", factor=2.0, original_length=2048.0, beta_fast=1.0, beta_slow=1.0)):
        _refused(pkg, 1, "needs a positive base", call, f, **bad)


def test_calls_without_elements_have_no_effect(pkg, hom, nothing_launched):
    import torch

    for rows, cols in ((0, 64), (5, 0), (0, 0)):
        q, s = (torch.empty(shape, dtype=torch.uint8) for shape in pkg.mxf4_shapes(rows, cols))
        x = torch.empty((rows, cols), dtype=torch.float16)
        hom.homQuantizeMxF4F16(x, q, s)
        hom.homDequantizeMxF4F16(q, s, x)
    a = [torch.empty(shape, dtype=torch.uint8) for shape in pkg.mxf4_shapes(0, 64)]
    b = _coded(pkg, 16, 64)
    hom.homGemmMxF4F16(*a, *b, None, torch.empty((0, 16), dtype=torch.float16))
    hom.homGemmMxF4F16(*b, *a, None, torch.empty((16, 0), dtype=torch.float16))
    f = _host(pkg, (4,), 8)
    for shape in ((0, 3, 4, 8), (2, 0, 4, 8), (2, 3, 0, 8)):
        x = torch.empty(shape, dtype=torch.float32)
        hom.homRotaryF32(x, None, f, x)
        hom.homRotaryF32(x, torch.empty(shape[:2], dtype=torch.int64), f, x)


def test_direct_calls_and_ctypes_agree(pkg, hom, nothing_launched):
    """The two ways the binding has of calling: the same refusals, argument errors as exceptions, tensors or descriptors."""
    import torch

    through = [pkg.RunnerUtils(direct=False)]
    assert through[0]._calls is None
    if pkg.CALLS_MODULE.exists():
        assert hom._calls is not None
        through.append(hom)
    q, s = _coded(pkg, 5, 40)
    x, rot = torch.zeros((5, 41), dtype=torch.float16), _host(pkg, (2, 3, 4, 8), 2)
    a, b = _coded(pkg, 6, 64), _coded(pkg, 16, 64)
    empty = [torch.empty(shape, dtype=torch.uint8) for shape in pkg.mxf4_shapes(0, 64)]
    for h in through:
        _refused(pkg, 1, "need codes", h.homQuantizeMxF4F16, torch.zeros((5, 70), dtype=torch.float16), q, s)
        _refused(pkg, 1, "need codes", h.homQuantizeMxF4F32, x, q, s, transposed=True)
        _refused(pkg, 1, "do not hold", h.homDequantizeMxF4F16, q, s, torch.zeros((5, 70), dtype=torch.float16))
        _refused(pkg, 1, "do not hold", h.homDequantizeMxF4F32, q, s, _host(pkg, (6, 40), 4))
        _refused(pkg, 2, "activation 5", h.homGemmMxF4F16, *a, *b, None, _host(pkg, (6, 16), 2), activation=5)
        _refused(pkg, 1, "needs a contiguous C", h.homGemmMxF4F16, *a, *b, None, _host(pkg, (6, 16), 2), beta=1)
        _refused(pkg, 1, "Frequencies", h.homRotaryF16, rot, None, None, rot)
        _refused(pkg, 1, "magnitude", h.homRotaryF32, rot, None, _host(pkg, (4,), 8), rot, magnitude=float("inf"))
        h.homQuantizeMxF4F16(torch.empty((0, 64), dtype=torch.float16), *empty)
        with pytest.raises(Exception) as e:
            h.homQuantizeMxF4F16("no tensor", q, s)
        assert not isinstance(e.value, pkg.HomError)
        with pytest.raises(Exception) as e:
            h.homGemmMxF4F16(*a, *b, None, _host(pkg, (6, 16), 2), alpha="one")
        assert not isinstance(e.value, pkg.HomError)


def test_a_failed_build_of_the_direct_calls_is_no_failed_build(tmp_path, monkeypatch, capsys):
    """The module is optional: what cannot be compiled is left out, an outdated one of an earlier build included."""
    import importlib.util
    import stat
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("hom_build_calls", Path(__file__).parents[1] / "hands-on-mlir_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    compiler = tmp_path / "gcc"
    compiler.write_text("#!/bin/sh\necho no such option >&2\nexit 1\n")
    compiler.chmod(compiler.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("PATH", str(tmp_path))
    headers = tmp_path / "include"
    headers.mkdir()
    (headers / "Python.h").write_text("")
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(headers)})
    old = tmp_path / build.CALLS_MODULE
    old.write_bytes(b"")
    build._build_calls(tmp_path, tmp_path / build.RUNNER_LIB.name, True, False)
    assert not old.exists() and "no such option" in capsys.readouterr().out


def test_descriptors_of_a_derived_class_and_of_a_second_package(pkg, hom, nothing_launched):
    """Both ways of calling take what is a MemRef by inheritance, and a package loaded a second time under another name
    leaves the first one's calls as they were."""
    import importlib.util
    import sys
    from pathlib import Path

    class Named(pkg.MemRef):
        pass

    q, s = _coded(pkg, 5, 40)
    x = Named(q.data_ptr, (5, 70))
    path = Path(pkg.__file__)
    spec = importlib.util.spec_from_file_location("hom_second", path, submodule_search_locations=[str(path.parent)])
    second = importlib.util.module_from_spec(spec)
    sys.modules["hom_second"] = second
    try:
        spec.loader.exec_module(second)
        other = second.RunnerUtils()
        assert second.MemRef is not pkg.MemRef
        for h in (pkg.RunnerUtils(direct=False), hom):
            _refused(pkg, 1, "need codes", h.homQuantizeMxF4F16, x, q, s)
        with pytest.raises(second.HomError):
            other.homQuantizeMxF4F16(second.MemRef(q.data_ptr, (5, 70)), *(second.MemRef(t.data_ptr, t.shape) for t in (q, s)))
    finally:
        del sys.modules["hom_second"]
