"""Microscaled 4-bit floating point: conversion bit for bit, the product against 64 bits."""
import numpy as np
import pytest

import mxf4_reference as ref
from util import to_dev

pytestmark = pytest.mark.gpu


def _buffers(pkg, cuda, rows, cols, fill=0xA5):
    """Codes and scales inside larger buffers whose other bytes must stay as they are."""
    import torch

    out = []
    for shape in pkg.mxf4_shapes(rows, cols):
        n = int(np.prod(shape))
        whole = torch.full((n + 512,), fill, dtype=torch.uint8, device=cuda)
        out.append((whole[256:256 + n].view(shape), whole))
    return out


def _assert_guards(buffers):
    for view, whole in buffers:
        n = view.numel()
        assert bool((whole[:256] == 0xA5).all()) and bool((whole[256 + n:] == 0xA5).all())


def _awkward(rng, rows, cols, dtype):
    """Blocks of every size, ties, zeros, negative zeros, subnormals, single large values."""
    x = rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-6, 6, (rows, 1)))
    grid = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.5, 4.0], (rows, cols)) * rng.choice([-1, 1], (rows, cols))
    x = np.where(rng.random((rows, cols)) < 0.4, grid * 2.0 ** rng.integers(-3, 3), x)
    x[rng.random((rows, cols)) < 0.1] = 0.0
    x[rng.random((rows, cols)) < 0.05] = -0.0
    if rows > 2:
        x[1] = 0.0
        x[2] = rng.integers(-9, 9, cols) * (2.0 ** -24 if dtype == np.float16 else 2.0 ** -140)
    if rows > 3:
        x[3, ::7] = 60000.0
    return x.astype(dtype)


SHAPES = [(1, 1), (1, 32), (3, 31), (5, 33), (33, 96), (127, 256), (128, 264), (129, 257), (70, 1000), (260, 513),
          (4, 4099), (300, 1003), (389, 2050)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_bit_for_bit_and_back(hom, pkg, cuda, rows, cols, transposed, dtype):
    import torch

    x = _awkward(np.random.default_rng(rows * 7 + cols), rows, cols, dtype)
    (q, q_all), (s, s_all) = buffers = _buffers(pkg, cuda, rows, cols)
    there = hom.homQuantizeMxF4F16 if dtype == np.float16 else hom.homQuantizeMxF4F32
    there(to_dev(x.T if transposed else x, cuda), q, s, transposed)
    codes, scales = ref.quantize(x)
    assert np.array_equal(s.cpu().numpy(), ref.tile_scales(scales))
    assert np.array_equal(q.cpu().numpy(), codes)
    _assert_guards(buffers)
    want = ref.values(codes, ref.tile_scales(scales))[:, :cols]
    for name, t in (("homDequantizeMxF4F16", torch.float16), ("homDequantizeMxF4F32", torch.float32)):
        out = torch.full((rows + 2, cols), 9.0, dtype=t, device=cuda)
        getattr(hom, name)(q, s, out[1:rows + 1])
        got = out.cpu().numpy()
        assert (got[0] == 9).all() and (got[-1] == 9).all()
        if dtype == np.float32 and t == torch.float16:
            with np.errstate(over="ignore"):
                assert np.array_equal(got[1:-1], want.astype(np.float16))
        else:
            assert np.array_equal(got[1:-1].astype(np.float64), want)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("transposed", [False, True])
def test_not_a_number_blocks(hom, pkg, cuda, transposed, dtype):
    import torch

    x = np.random.default_rng(5).standard_normal((40, 100)).astype(dtype)
    x[0, 3], x[1, 40], x[2, 99], x[39, 64] = np.nan, np.inf, -np.inf, -np.nan
    (q, _), (s, _) = _buffers(pkg, cuda, 40, 100)
    f16 = dtype == np.float16
    (hom.homQuantizeMxF4F16 if f16 else hom.homQuantizeMxF4F32)(to_dev(x.T if transposed else x, cuda), q, s, transposed)
    codes, scales = ref.quantize(x)
    assert np.array_equal(q.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), ref.tile_scales(scales))
    out = torch.empty((40, 100), dtype=torch.float16 if f16 else torch.float32, device=cuda)
    (hom.homDequantizeMxF4F16 if f16 else hom.homDequantizeMxF4F32)(q, s, out)
    got = out.cpu().numpy()
    nan = np.zeros((40, 4), bool)
    nan[0, 0] = nan[1, 1] = nan[2, 3] = nan[39, 2] = True
    assert np.array_equal(np.isnan(got), nan.repeat(32, 1)[:, :100])


def test_unaligned_and_offset_operands(hom, pkg, cuda):
    """An X that starts on an odd element, named by a descriptor's offset."""
    import torch

    x = np.random.default_rng(6).standard_normal((9, 64)).astype(np.float16)
    store = torch.zeros(9 * 64 + 3, dtype=torch.float16, device=cuda)
    store[3:] = to_dev(x, cuda).reshape(-1)
    (q, _), (s, _) = _buffers(pkg, cuda, 9, 64)
    hom.homQuantizeMxF4F16(pkg.MemRef(store.data_ptr(), (9, 64), offset=3, keepalive=store), q, s)
    codes, scales = ref.quantize(x)
    assert np.array_equal(q.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), ref.tile_scales(scales))
    out = torch.zeros(9 * 64 + 3, dtype=torch.float32, device=cuda)
    hom.homDequantizeMxF4F32(q, s, pkg.MemRef(out.data_ptr(), (3, 3, 64), offset=1, keepalive=out))
    got = out.cpu().numpy()
    assert got[0] == 0 and (got[-2:] == 0).all()
    assert np.array_equal(got[1:-2].reshape(9, 64).astype(np.float64), ref.values(codes, ref.tile_scales(scales)))


# ------------------------------------------------------------------------------------------ product

def _operands(rng, m, n, k, spread):
    """Random codes; scales within `spread` powers of two."""
    out = []
    for rows in (m, n):
        blocks = -(-k // 32)
        nibbles = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
        nibbles[:, k:] = 0
        codes = nibbles[:, 0::2] | (nibbles[:, 1::2] << 4)
        scales = (127 + rng.integers(-spread, spread + 1, (rows, blocks))).astype(np.uint8)
        out += [codes, ref.tile_scales(scales)]
    return out


def _product(hom, cuda, a, sa, b, sb, c, d, act=0, alpha=1.0, beta=0.0):
    hom.homGemmMxF4F16(*(to_dev(t, cuda) for t in (a, sa, b, sb)), c, d, act, alpha, beta)


# one and two rows; one wave of small tiles with K in one, two and four parts; CTA pairs with A resident and not; N that
# is no multiple of 8 in each
PRODUCTS = [(1, 8, 32), (1, 4096, 1024), (2, 1, 32), (2, 333, 5000), (7, 33, 96), (16, 768, 4096), (33, 77, 2100),
            (127, 129, 256), (128, 128, 288), (129, 200, 544), (385, 1001, 808), (300, 1000, 800), (640, 512, 1056),
            (1100, 2304, 768), (2500, 1024, 520), (1001, 2001, 1060), (3900, 2400, 300), (4001, 2391, 600),
            (5, 72, 40000), (900, 1288, 2500), (100, 1001, 3000), (130, 1000, 2600), (128, 4000, 4200), (200, 777, 4100),
            (20, 640, 1700), (4001, 2390, 600), (9500, 70, 300)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_representable_sums_is_exact(hom, cuda, m, n, k):
    """With one scale for all blocks every partial sum is a whole number of quarters below 2^24: nothing is rounded
    but the result, whatever the order of the additions."""
    import torch

    rng = np.random.default_rng(m + n + k)
    a, sa, b, sb = _operands(rng, m, n, k, 0)
    want = ref.values(a, sa) @ ref.values(b, sb).T
    d = torch.full((m + 2, n), 5.0, dtype=torch.float16, device=cuda)
    inner = d[1:m + 1]
    if n % 8 == 0:
        _product(hom, cuda, a, sa, b, sb, None, inner)
        got = d.cpu().numpy()
        assert (got[0] == 5).all() and (got[-1] == 5).all()
        got = got[1:-1]
    else:
        out = torch.full((m, n), 5.0, dtype=torch.float16, device=cuda)
        _product(hom, cuda, a, sa, b, sb, None, out)
        got = out.cpu().numpy()
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(np.float16))


@pytest.mark.parametrize("act,alpha,beta,row", [(0, 1.0, 0.0, False), (1, 1.0, 1.0, True), (0, 1.0, 1.0, False),
                                                (1, 0.25, -2.0, False), (0, 0.5, 3.0, True), (1, 1.0, 0.0, False)])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_with_epilogue(hom, cuda, m, n, k, act, alpha, beta, row):
    import torch

    rng = np.random.default_rng(m * 3 + n + k + act)
    a, sa, b, sb = _operands(rng, m, n, k, 3)
    va, vb = ref.values(a, sa), ref.values(b, sb)
    alpha /= float(np.sqrt(k)) * 8 if alpha != 1.0 else 1.0
    if alpha == 1.0:  # keep the results near one: exact powers of two on B's scales
        shift = int(np.log2(np.sqrt(k))) + 4
        sb = np.where(sb > 0, sb - shift, 0).astype(np.uint8)
        vb = vb * 2.0 ** -shift
    c = rng.standard_normal((1 if row else m, n)).astype(np.float16)
    v = alpha * (va @ vb.T) + beta * c.astype(np.float64)
    want = ref.gelu(v) if act else v
    # K additions of products with at most half a step each, of the sum of magnitudes; one step each for alpha, beta
    # and C; the slope of GELU is below 1.13 and its own error below 1e-6; half a step of fp16
    size = abs(alpha) * (np.abs(va) @ np.abs(vb).T)
    tol = 1.13 * ((k + 2) * 2.0 ** -24 * size + 2 * 2.0 ** -24 * np.abs(beta * c)) + 1e-6 * act
    tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    tc = to_dev(c, cuda)
    out = torch.full((m, n), 5.0, dtype=torch.float16, device=cuda)
    _product(hom, cuda, a, sa, b, sb, tc if beta else None, out, act, alpha, beta)
    err = np.abs(out.cpu().numpy().astype(np.float64) - want)
    assert (err <= tol).all(), (err - tol).max()
    again = torch.empty_like(out)
    _product(hom, cuda, a, sa, b, sb, tc if beta else None, again, act, alpha, beta)
    assert torch.equal(again, out), "the order of the additions is fixed"
    if beta and not row:  # C is D
        _product(hom, cuda, a, sa, b, sb, tc, tc, act, alpha, beta)
        assert torch.equal(tc, out)


def test_product_takes_every_scale_to_its_own_block(hom, cuda):
    """One nonzero pair of values per (row, column): the result is the product of its two scales."""
    import torch

    m, n, k = 300, 264, 416
    rng = np.random.default_rng(9)
    for trial in range(4):
        block, lane = int(rng.integers(0, k // 32)), int(rng.integers(0, 32))
        at = block * 32 + lane
        out = []
        for rows in (m, n):
            nibbles = np.zeros((rows, k), np.uint8)
            nibbles[:, at] = 2  # 1.0
            scales = (127 + rng.integers(-5, 6, (rows, k // 32))).astype(np.uint8)
            out += [nibbles[:, 0::2] | (nibbles[:, 1::2] << 4), ref.tile_scales(scales)]
        d = torch.empty((m, n), dtype=torch.float16, device=cuda)
        _product(hom, cuda, *out, None, d)
        want = ref.values(out[0], out[1]) @ ref.values(out[2], out[3]).T
        assert np.array_equal(d.cpu().numpy().astype(np.float64), want), trial


def test_not_a_number_stays_in_its_row_and_column(hom, cuda):
    import torch

    m, n, k = 200, 136, 320
    a, sa, b, sb = _operands(np.random.default_rng(3), m, n, k, 1)
    sa = sa.copy()
    sa[150 // 128, 5 // 4, 150 % 32 * 16 + 150 // 32 % 4 * 4 + 5 % 4] = 255
    sb = sb.copy()
    sb[7 // 128, 9 // 4, 7 % 32 * 16 + 7 // 32 % 4 * 4 + 9 % 4] = 255
    d = torch.empty((m, n), dtype=torch.float16, device=cuda)
    _product(hom, cuda, a, sa, b, sb, None, d)
    bad = np.isnan(d.cpu().numpy())
    want = np.zeros((m, n), bool)
    want[150], want[:, 7] = True, True
    assert np.array_equal(bad, want)


def test_extreme_scales(hom, cuda):
    """The largest and smallest scales of one operand against the other's: the product is an ordinary number."""
    import torch

    m, n, k = 130, 64, 64
    rng = np.random.default_rng(4)
    a, b = (rng.integers(0, 256, (rows, k // 2)).astype(np.uint8) for rows in (m, n))
    for high, low in ((250, 4), (240, 14), (127, 127)):
        sa = ref.tile_scales(np.full((m, 2), high, np.uint8))
        sb = ref.tile_scales(np.full((n, 2), low, np.uint8))
        d = torch.empty((m, n), dtype=torch.float16, device=cuda)
        _product(hom, cuda, a, sa, b, sb, None, d)
        want = ref.values(a, sa) @ ref.values(b, sb).T
        assert np.array_equal(d.cpu().numpy(), want.astype(np.float16)), (high, low)


@pytest.mark.parametrize("cols,rows", [(2080, 1048582), (2083, 1048581)])
def test_offsets_beyond_32_bits(hom, pkg, cuda, cols, rows):
    """More than 2^31 values.  They are codes times one, with a largest value of each block between 4 and 6: they come
    back as they were, and so does their product with the identity, plus themselves."""
    import torch

    rng = np.random.default_rng(31)
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float16)
    part = grid[rng.integers(0, 8, (4099, cols))] * rng.choice([-1, 1], (4099, cols)).astype(np.float16)
    part[:, ::32] = grid[rng.integers(6, 8, part[:, ::32].shape)]
    part = to_dev(part, cuda)
    x = part.repeat(-(-rows // 4099), 1)[:rows]
    assert x.numel() > 2 ** 31 and x.is_contiguous()

    def coded(n):
        return [torch.empty(s, dtype=torch.uint8, device=cuda) for s in pkg.mxf4_shapes(n, cols)]

    q, eye, out = coded(rows), coded(cols), torch.empty_like(x)
    hom.homQuantizeMxF4F16(x, *q)
    hom.homDequantizeMxF4F16(*q, out)
    hom.synchronize()
    assert torch.equal(out, x)
    hom.homQuantizeMxF4F16(torch.eye(cols, dtype=torch.float16, device=cuda), *eye)
    out.fill_(7.0)
    hom.homGemmMxF4F16(*q, *eye, None, out)
    hom.synchronize()
    assert torch.equal(out, x)
    hom.homGemmMxF4F16(*q, *eye, out, out, beta=1.0)
    hom.synchronize()
    assert torch.equal(out, x * 2)
    turned = x.t().contiguous()
    del out, x
    again = coded(rows)
    hom.homQuantizeMxF4F16(turned, *again, True)
    hom.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(q, again))


def test_streams_graphs_and_declared_weights(hom, pkg, cuda):
    """The same calls eagerly, on another stream, and replayed from two graphs whose replays alternate; the weight is
    quantised into its buffers by the stream itself."""
    import torch

    m, n, k = 200, 512, 768
    rng = np.random.default_rng(12)
    w = to_dev(rng.standard_normal((1, k, n)).astype(np.float16), cuda)
    xs = [to_dev(rng.standard_normal((m, k)).astype(np.float16), cuda) for _ in range(2)]
    (bq, _), (bs, _) = _buffers(pkg, cuda, n, k)
    hom.homQuantizeMxF4F16(w, bq, bs, True)
    codes, scales = ref.quantize(w[0].T.cpu().numpy())
    assert np.array_equal(bq.cpu().numpy(), codes) and np.array_equal(bs.cpu().numpy(), ref.tile_scales(scales))

    def step(x, q, s, d):
        hom.homQuantizeMxF4F16(x, q, s)
        hom.homGemmMxF4F16(q, s, bq, bs, None, d, 1)

    def fresh():
        return [v for v, _ in _buffers(pkg, cuda, m, k)] + [torch.empty((m, n), dtype=torch.float16, device=cuda)]

    want = []
    for x in xs:
        buffers = fresh()
        step(x, *buffers)
        want.append(buffers[-1].clone())
    assert not torch.equal(want[0], want[1])
    hom.declare_weights(bq)
    hom.declare_weights(bs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    try:
        hom.set_stream(stream.cuda_stream)
        graphs = []
        with torch.cuda.stream(stream):
            for x in xs:
                buffers = fresh()
                step(x, *buffers)
                stream.synchronize()
                assert torch.equal(buffers[-1], want[len(graphs)])
                buffers[-1].zero_()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    step(x, *buffers)
                graphs.append((graph, buffers))
            for _ in range(3):
                for (graph, buffers), w_ in zip(graphs, want):
                    buffers[-1].zero_()
                    graph.replay()
                    stream.synchronize()
                    assert torch.equal(buffers[-1], w_)
    finally:
        stream.synchronize()
        hom.use_torch_stream()
        hom.forget_weights(bq)
        hom.forget_weights(bs)


def test_two_threads_on_two_streams(hom, pkg, cuda):
    """Calls of two host threads overlap on the device and in the library."""
    import threading

    import torch

    rng = np.random.default_rng(21)
    jobs = []
    for m, n, k in ((1, 512, 768), (96, 328, 1280), (3000, 2304, 768), (500, 2403, 640)):
        a, sa, b, sb = (to_dev(t, cuda) for t in _operands(rng, m, n, k, 2))
        want = torch.empty((m, n), dtype=torch.float16, device=cuda)
        hom.homGemmMxF4F16(a, sa, b, sb, None, want, 1, 0.01)
        jobs.append(((a, sa, b, sb), want))
    hom.synchronize()
    bad = []

    def work(order):
        stream = torch.cuda.Stream()
        hom.set_stream(stream.cuda_stream)
        outs = []
        for _ in range(10):
            for i in order:
                operands, want = jobs[i]
                with torch.cuda.stream(stream):
                    d = torch.empty_like(want)
                hom.homGemmMxF4F16(*operands, None, d, 1, 0.01)
                outs.append((i, d))
        hom.synchronize()
        bad.extend(i for i, d in outs if not torch.equal(d, jobs[i][1]))

    threads = [threading.Thread(target=work, args=(order,)) for order in ((0, 1, 2, 3), (3, 2, 1, 0))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("m", [1, 2, 200, 3000])
def test_declared_weights_and_their_rewriting(hom, pkg, cuda, m):
    """Every form of the product with a declared weight, and right behind a call that quantises another weight into the
    declared buffers, with nothing that waits in between."""
    import torch

    n, k = 2048, 1600
    rng = np.random.default_rng(m)
    x = to_dev(rng.standard_normal((m, k)).astype(np.float16), cuda)
    ws = [to_dev(rng.standard_normal((n, k)).astype(np.float32), cuda) for _ in range(2)]
    (aq, _), (as_, _) = _buffers(pkg, cuda, m, k)
    (bq, b_all), (bs, s_all) = _buffers(pkg, cuda, n, k)
    d = [torch.empty((m, n), dtype=torch.float16, device=cuda) for _ in range(6)]
    for w, out in zip(ws, d):
        hom.homQuantizeMxF4F32(w, bq, bs)
        hom.homQuantizeMxF4F16(x, aq, as_)
        hom.homGemmMxF4F16(aq, as_, bq, bs, None, out)
    hom.synchronize()
    assert not torch.equal(d[0], d[1])
    try:
        for _ in range(3):
            # (one declaration around the codes, more than they take)
            hom.declare_weights(b_all)
            hom.declare_weights(bs)
            hom.homQuantizeMxF4F16(x, aq, as_)
            hom.homGemmMxF4F16(aq, as_, bq, bs, None, d[2])
            for w, out in zip(ws, d[3:5]):
                hom.homQuantizeMxF4F32(w, bq, bs)
                hom.homQuantizeMxF4F16(x, aq, as_)
                hom.homGemmMxF4F16(aq, as_, bq, bs, None, out)
            hom.synchronize()
            assert torch.equal(d[2], d[1]) and torch.equal(d[3], d[0]) and torch.equal(d[4], d[1])
    finally:
        hom.forget_weights(b_all)
        hom.forget_weights(bs)


@pytest.mark.parametrize("rows,dtype", [(2, np.float16), (1, np.float32)])
def test_quantize_transposed_with_a_long_k(hom, pkg, cuda, rows, dtype):
    """More than 2^16 scale tiles along K."""
    cols = 128 * 65536 + 33
    x = np.random.default_rng(rows).standard_normal((cols, rows)).astype(dtype)
    (q, q_all), (s, s_all) = buffers = _buffers(pkg, cuda, rows, cols)
    (hom.homQuantizeMxF4F16 if dtype == np.float16 else hom.homQuantizeMxF4F32)(to_dev(x, cuda), q, s, True)
    q, s = q.cpu().numpy(), s.cpu().numpy()
    _assert_guards(buffers)
    for first in (0, 128 * 32768, 128 * 65535, 128 * 65536):  # blocks are independent of one another
        part = x[first:first + 128].T
        codes, scales = ref.quantize(part)
        assert np.array_equal(q[:, first // 2:first // 2 + codes.shape[1]], codes)
        assert np.array_equal(s[:, first // 128:first // 128 + 1], ref.tile_scales(scales))
    rq, rs = ([v for v, _ in _buffers(pkg, cuda, rows, cols)])
    (hom.homQuantizeMxF4F16 if dtype == np.float16 else hom.homQuantizeMxF4F32)(to_dev(x.T, cuda), rq, rs)
    assert np.array_equal(rq.cpu().numpy(), q) and np.array_equal(rs.cpu().numpy(), s)


@pytest.mark.parametrize("act,row", [(0, True), (1, False)])
@pytest.mark.parametrize("m,n,k", [(1100, 2304, 768), (2500, 1024, 520), (3900, 2400, 300), (900, 1288, 2500), (9500, 264, 300),
                                   (1001, 2001, 1060), (4001, 2390, 600), (300, 1000, 800), (2, 333, 5000)])
def test_bias_without_gelu_and_residual_with_it(hom, cuda, m, n, k, act, row):
    """An ordinary projection's row of C, and a matrix C under GELU, neither of them scaled."""
    test_product_with_epilogue(hom, cuda, m, n, k, act, 1.0, 1.0, row)


@pytest.mark.parametrize("declared", [False, True])
@pytest.mark.parametrize("m,n,k", [(65536, 264, 1000), (65536, 263, 1000), (200000, 40, 1000), (66000, 600, 250),
                                   (40000, 520, 1500), (70001, 258, 700)])
def test_many_row_blocks_on_a_pair_are_exact(hom, cuda, m, n, k, declared):
    """A pair that goes through three to eleven row blocks of A, kept in shared memory (K up to 1024) or not, and as many
    turns of its accumulators and stages; the weight fetched early or not.  Sums as in the exact test above."""
    import torch

    rng = np.random.default_rng(m + n)
    blocks = -(-k // 32)
    coded, values = [], []
    for rows in (m, n):
        nibbles = rng.integers(0, 16, (rows, blocks * 32), dtype=np.uint8)
        nibbles[:, k:] = 0
        scales = np.zeros((-(-rows // 128), -(-blocks // 4), 512), np.uint8)
        r, b = np.arange(rows)[:, None], np.arange(blocks)[None]
        scales[r // 128, b // 4, r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = 127
        coded += [to_dev(nibbles[:, 0::2] | (nibbles[:, 1::2] << 4), cuda), to_dev(scales, cuda)]
        table = np.concatenate([ref.VALUES, -ref.VALUES]).astype(np.float32)
        values.append(table[nibbles])  # (sums of whole quarters below 2^24: exact in fp32 too)
    want = values[0] @ values[1].T
    assert np.abs(want).max() < 2 ** 16
    row = rng.integers(-8, 9, (1, n)).astype(np.float16)
    out, biased = (torch.full((m, n), 5.0, dtype=torch.float16, device=cuda) for _ in range(2))
    torch.cuda.synchronize()
    if declared:
        for t in coded[2:]:
            hom.declare_weights(t)
    try:
        hom.homGemmMxF4F16(*coded, None, out)
        hom.homGemmMxF4F16(*coded, to_dev(row, cuda), biased, 0, 1.0, 1.0)
        hom.synchronize()
    finally:
        if declared:
            for t in coded[2:]:
                hom.forget_weights(t)
    assert np.array_equal(out.cpu().numpy(), want.astype(np.float16))
    assert np.array_equal(biased.cpu().numpy(), (want + row.astype(np.float32)).astype(np.float16))
