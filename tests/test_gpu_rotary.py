"""Rotary positions against 64 bits: layouts, parts of a head, strides, far positions, gradients."""
import numpy as np
import pytest

import mxf4_reference as ref
from util import to_dev

pytestmark = pytest.mark.gpu


def _frequencies(half, base=10000.0):
    return base ** (-np.arange(half) / half)


def _call(hom, x):
    import torch
    return hom.homRotaryF16 if x.dtype == torch.float16 else hom.homRotaryF32


def _check(got, x, positions, freq, interleaved, backward, magnitude):
    want = ref.rotary(x, positions, freq, interleaved, backward, magnitude)
    tol = ref.rotary_tolerance(x, want, freq, interleaved, magnitude, np.finfo(got.dtype).eps)
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (err - tol).max()
    half = len(freq)
    assert np.array_equal(got[..., 2 * half:], x[..., 2 * half:])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bs,seq,heads,d,half", [
    (1, 1, 1, 2, 1), (1, 1, 16, 64, 32), (2, 5, 3, 64, 32), (3, 7, 24, 64, 16), (2, 3, 5, 80, 20), (1, 9, 2, 33, 16),
    (2, 4, 3, 66, 33), (1, 300, 12, 64, 32), (1, 2, 1, 1024, 512), (2, 2, 40, 128, 24), (1, 3, 200, 64, 32),
])
def test_rotary_layouts(hom, cuda, bs, seq, heads, d, half, interleaved, dtype):
    import torch

    rng = np.random.default_rng(bs + seq + heads + d)
    x = rng.standard_normal((bs, seq, heads, d)).astype(dtype)
    freq = _frequencies(half)
    tf = to_dev(freq, cuda)
    for positions, backward, magnitude in ((None, False, 1.0), (rng.integers(-5, 1 << 20, (bs, seq)), True, 1.25),
                                           (rng.integers(0, 4096, (1, seq)), False, -0.5)):
        tx = to_dev(x, cuda)
        out = torch.full((bs, seq + 1, heads, d), 3.0, dtype=tx.dtype, device=cuda)
        tp = None if positions is None else to_dev(positions, cuda)
        # `out` is a view with a longer batch stride: the extra token must stay as it is
        _call(hom, tx)(tx, tp, tf, out[:, :seq], interleaved, backward, magnitude)
        got = out.cpu().numpy()
        assert (got[:, seq] == 3).all()
        assert np.array_equal(tx.cpu().numpy(), x)
        full = None if positions is None else np.broadcast_to(positions, (bs, seq))
        _check(got[:, :seq], x, full, freq, interleaved, backward, magnitude)
        _call(hom, tx)(tx, tp, tf, tx, interleaved, backward, magnitude)  # in place
        assert torch.equal(tx, out[:, :seq])


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_views(hom, cuda, interleaved, dtype):
    """Heads before tokens, odd strides and starts, a batch that is read from one broadcast sequence, and the query and
    key heads of a packed buffer whose values stay as they are."""
    import torch

    rng = np.random.default_rng(3)
    freq = _frequencies(32)
    tf = to_dev(freq, cuda)
    call = hom.homRotaryF16 if dtype == np.float16 else hom.homRotaryF32
    x = rng.standard_normal((2, 6, 9, 64)).astype(dtype)  # [bs, heads, seq, d]
    tx = to_dev(x, cuda)
    call(tx.transpose(1, 2), None, tf, tx.transpose(1, 2), interleaved)
    _check(tx.cpu().numpy().transpose(0, 2, 1, 3), x.transpose(0, 2, 1, 3), None, freq, interleaved, False, 1.0)

    store = torch.from_numpy(rng.standard_normal(4 * 5 * 7 * 67 + 1).astype(dtype)).to(cuda)
    view = store[1:].view(4, 5, 7, 67)[..., :64]
    before, x = store.clone(), view.cpu().numpy()
    out = torch.empty((4, 5, 7, 64), dtype=store.dtype, device=cuda)
    call(view, None, tf, out, interleaved)
    _check(out.cpu().numpy(), x, None, freq, interleaved, False, 1.0)
    assert torch.equal(store, before)
    call(view, None, tf, view, interleaved)
    assert torch.equal(view, out)
    changed = torch.zeros_like(store, dtype=torch.bool)
    changed[1:].view(4, 5, 7, 67)[..., :64] = True
    assert torch.equal(store[~changed], before[~changed])

    one = to_dev(rng.standard_normal((1, 5, 3, 64)).astype(dtype), cuda)
    out = torch.empty((4, 5, 3, 64), dtype=one.dtype, device=cuda)
    positions = rng.integers(0, 1000, (4, 5))
    call(one.expand(4, 5, 3, 64), to_dev(positions, cuda), tf, out, interleaved)
    _check(out.cpu().numpy(), np.broadcast_to(one.cpu().numpy(), (4, 5, 3, 64)), positions, freq, interleaved, False, 1.0)

    qkv = to_dev(rng.standard_normal((2, 9, 3 * 4 * 64)).astype(dtype), cuda)
    before = qkv.clone()
    turned = qkv.view(2, 9, 12, 64)[:, :, :8]
    call(turned, None, tf, turned, interleaved)
    _check(turned.cpu().numpy(), before.view(2, 9, 12, 64)[:, :, :8].cpu().numpy(), None, freq, interleaved, False, 1.0)
    assert torch.equal(qkv.view(2, 9, 12, 64)[:, :, 8:], before.view(2, 9, 12, 64)[:, :, 8:])


def test_rotary_beyond_32_bit_offsets(hom, cuda):
    """Two sequences 2^31 + 64 elements apart, turned in place in a 4 GB buffer."""
    import torch

    far = (1 << 31) + 64
    store = torch.zeros(far + 2 * 4 * 64, dtype=torch.float16, device=cuda)
    view = store.as_strided((2, 2, 4, 64), (far, 4 * 64, 64, 1))
    x = np.random.default_rng(8).standard_normal((2, 2, 4, 64)).astype(np.float16)
    view.copy_(to_dev(x, cuda))
    freq = _frequencies(32)
    positions = np.array([[0, 5], [1 << 33, (1 << 33) + 1]])
    hom.homRotaryF16(view, to_dev(positions, cuda), to_dev(freq, cuda), view)
    _check(view.cpu().numpy(), x, positions, freq, False, False, 1.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(hom, cuda, interleaved):
    """The backward call is the transpose of the forward one, and agrees with differences of it."""
    import torch

    rng = np.random.default_rng(11)
    shape = (2, 6, 3, 40)
    freq = to_dev(_frequencies(16), cuda)
    positions = to_dev(rng.integers(0, 100000, (2, 6)), cuda)
    x, g = (to_dev(rng.standard_normal(shape).astype(np.float32), cuda) for _ in range(2))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    hom.homRotaryF32(x, positions, freq, y, interleaved, False, 1.5)
    hom.homRotaryF32(g, positions, freq, dx, interleaved, True, 1.5)
    left, right = (y.double() * g.double()).sum().item(), (x.double() * dx.double()).sum().item()
    # 1440 products of numbers of size one, each of which carries the rotation's error
    assert abs(left - right) <= 1440 * 1.5 * 4 * (2.5e-7 + 5 * 2.0 ** -24)
    step = 2.0 ** -6  # the call is linear: any step gives the derivative, a power of two adds no rounding of its own
    for at in [(0, 0, 0, 0), (1, 5, 2, 17), (0, 3, 1, 31), (1, 2, 0, 39), (1, 5, 1, 8)]:
        ends = []
        for sign in (1, -1):
            moved = x.clone()
            moved[at] += sign * step
            out = torch.empty_like(x)
            hom.homRotaryF32(moved, positions, freq, out, interleaved, False, 1.5)
            ends.append((out.double() * g.double()).sum().item())
            size = moved[at].double().item()
        slope = (ends[0] - ends[1]) / (2 * step)
        # two outputs change; each end carries fp32 errors of values of size four, the moved value half a step
        assert abs(slope - dx[at].item()) <= 2 * 4 * 4 * 1.5 * 3e-7 / step + abs(size) * 1e-6


@pytest.mark.parametrize("half", [1, 2, 32, 512])
def test_frequencies(hom, cuda, half):
    import torch

    out = torch.full((half + 1,), 7.0, dtype=torch.float64, device=cuda)
    i = np.arange(half)
    plain = 10000.0 ** (-i / half)
    base = 10000.0 * (8.0 ** (half / (half - 1)) if half > 1 else 1.0)
    turns = 2048 * plain / (2 * np.pi)
    keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0, 1)
    for scaling, want in (("none", plain), ("linear", plain / 8), ("base", base ** (-i / half)),
                          ("parts", plain * (keep + (1 - keep) / 8))):
        hom.homRotaryFrequencies(out[:half], 10000.0, scaling, 8.0, 2048.0)
        got = out.cpu().numpy()
        assert got[-1] == 7.0
        # a power's relative error grows with its exponent: ln(10000 * 64) < 14 steps, and a few for the rest
        assert np.abs(got[:-1] / want - 1).max() <= 40 * 2.0 ** -53, scaling


def test_rotary_on_another_stream_and_in_graphs(hom, cuda):
    import torch

    rng = np.random.default_rng(2)
    freq = torch.empty(32, dtype=torch.float64, device=cuda)
    hom.homRotaryFrequencies(freq)
    x = [to_dev(rng.standard_normal((4, 33, 8, 64)).astype(np.float16), cuda) for _ in range(2)]
    want = [torch.empty_like(v) for v in x]
    for v, w in zip(x, want):
        hom.homRotaryF16(v, None, freq, w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    try:
        hom.set_stream(stream.cuda_stream)
        graphs = []
        with torch.cuda.stream(stream):
            for v in x:
                out = torch.zeros_like(v)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    hom.homRotaryF16(v, None, freq, out)
                graphs.append((graph, out))
            for _ in range(2):
                for (graph, out), w in zip(graphs, want):
                    out.zero_()
                    graph.replay()
                    stream.synchronize()
                    assert torch.equal(out, w)
    finally:
        stream.synchronize()
        hom.use_torch_stream()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("bs,seq,heads,d,half", [(1, 1, 1, 4, 2), (2, 5, 3, 68, 34), (2, 3, 4, 50, 18), (1, 7, 5, 20, 2),
                                                 (3, 11, 7, 100, 50), (1, 300, 12, 64, 10), (2, 2, 33, 36, 6)])
def test_rotary_in_pieces_of_two_elements(hom, cuda, bs, seq, heads, d, half, interleaved, dtype):
    test_rotary_layouts(hom, cuda, bs, seq, heads, d, half, interleaved, dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pitch,half", [(66, 32), (70, 16), (66, 24)])
def test_rotary_heads_whose_pitch_allows_two_elements(hom, cuda, interleaved, dtype, pitch, half):
    import torch

    rng = np.random.default_rng(pitch + half)
    store = torch.from_numpy(rng.standard_normal((3, 9, 5, pitch)).astype(dtype)).to(cuda)
    view, before = store[..., :64], store.clone()
    freq = _frequencies(half)
    x = view.cpu().numpy()
    out = torch.empty((3, 9, 5, 64), dtype=store.dtype, device=cuda)
    call = _call(hom, store)
    call(view, None, to_dev(freq, cuda), out, interleaved)
    _check(out.cpu().numpy(), x, None, freq, interleaved, False, 1.0)
    call(view, None, to_dev(freq, cuda), view, interleaved)  # in place: a lane keeps its turns where the pairs allow it
    assert torch.equal(view, out) and torch.equal(store[..., 64:], before[..., 64:])
