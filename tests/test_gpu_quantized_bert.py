"""The 4-bit and rotary operators together, as an encoder layer uses them: called one after the other, and through the
replay program."""
import numpy as np
import pytest

import mxf4_reference as ref
from util import assert_bits_equal, drift_fractions, to_dev

pytestmark = pytest.mark.gpu


def _model(seed, seq, hidden=256, heads=4, ffn=512, layers=2):
    from hands_on_mlir_b200.bert_program import BertConfig
    cfg = BertConfig(layers=layers, hidden=hidden, heads=heads, ffn=ffn, vocab=500)
    rng = np.random.default_rng(seed)
    w = {n: rng.normal(0, 0.05, cfg.weight_shape(n, seq)).astype(np.float16) for n in cfg.weight_names()}
    return cfg, w, rng


def _inputs(cfg, rng, lens, seq):
    ids = rng.integers(0, cfg.vocab, (len(lens), seq)).astype(np.int64)
    mask = (np.arange(seq)[None, :] < np.array(lens)[:, None]).astype(np.int64)
    return ids, mask, rng.integers(0, 2, ids.shape).astype(np.int64)


def _layernorm(x):
    mean = x.mean(-1, keepdims=True)
    return (x - mean) / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + 1e-12)


def _close(got, want, tol, what):
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (what, (err - tol).max())


def test_attention_half_of_a_layer(hom, pkg, cuda):
    """Quantise, QKV product, rotary in the packed buffer, attention, quantise, output product onto the residual,
    LayerNorm; each stage against 64 bits of what the stage before it left."""
    import torch

    bs, seq, heads = 3, 77, 4
    hidden, rows = 64 * heads, bs * seq
    rng = np.random.default_rng(1)
    x = rng.standard_normal((bs, seq, hidden)).astype(np.float16)
    wqkv, wo = (rng.normal(0, hidden ** -0.5, (1, hidden, n)).astype(np.float16) for n in (3 * hidden, hidden))
    lens = [77, 1, 40]
    cu = to_dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), cuda)
    freq = torch.empty(32, dtype=torch.float64, device=cuda)

    def coded(n, k):
        return [torch.empty(s, dtype=torch.uint8, device=cuda) for s in pkg.mxf4_shapes(n, k)]

    half = dict(dtype=torch.float16, device=cuda)
    tx, qx, qo = to_dev(x, cuda), coded(rows, hidden), coded(rows, hidden)
    bqkv, bo = coded(3 * hidden, hidden), coded(hidden, hidden)
    qkv, packed = torch.empty((rows, 3 * hidden), **half), torch.empty((rows, 3 * hidden), **half)
    ctx, out = torch.empty((bs, seq, hidden), **half), tx.clone()
    hom.homRotaryFrequencies(freq)
    hom.homQuantizeMxF4F16(to_dev(wqkv, cuda), *bqkv, True)
    hom.homQuantizeMxF4F16(to_dev(wo, cuda), *bo, True)
    hom.homQuantizeMxF4F16(tx, *qx)
    hom.homGemmMxF4F16(*qx, *bqkv, None, qkv)
    packed.copy_(qkv)
    turned = packed.view(bs, seq, 3 * heads, 64)[:, :, :2 * heads]
    hom.homRotaryF16(turned, None, freq, turned)
    hom.nvteBertAttentionF16(packed.view(bs, seq, 3 * hidden), cu, ctx, 0.125, heads)
    hom.homQuantizeMxF4F16(ctx, *qo)
    hom.homGemmMxF4F16(*qo, *bo, out.view(rows, hidden), out.view(rows, hidden), beta=1.0)
    summed = out.clone()
    hom.nvteLayernormF16(out, 1e-12)
    hom.synchronize()

    def host(t):
        return t.cpu().numpy()

    for q, v in ((qx, x), (qo, host(ctx))):
        codes, scales = ref.quantize(v.reshape(rows, hidden))
        assert np.array_equal(host(q[0]), codes) and np.array_equal(host(q[1]), ref.tile_scales(scales))
    for got, a, b, c in ((qkv, qx, bqkv, 0.0), (summed.view(rows, hidden), qo, bo, x.reshape(rows, hidden).astype(float))):
        va, vb = (ref.values(host(t[0]), host(t[1])) for t in (a, b))
        want = va @ vb.T + c
        size = np.abs(va) @ np.abs(vb).T + np.abs(c)
        _close(host(got), want, (hidden + 2) * 2.0 ** -24 * size + np.abs(want) * 2.0 ** -11 + 2.0 ** -25, "product")
    before, f = host(qkv).reshape(bs, seq, 3 * heads, 64), host(freq)
    want = ref.rotary(before[:, :, :2 * heads], None, f)
    _close(host(turned), want, ref.rotary_tolerance(before[:, :, :2 * heads], want, f, False, 1.0, 2.0 ** -10), "rotary")
    assert np.array_equal(host(packed).reshape(before.shape)[:, :, 2 * heads:], before[:, :, 2 * heads:])
    want = _layernorm(host(summed).astype(np.float64))
    # fp32 statistics of 256 values and half a step of the result
    _close(host(out), want, np.abs(want) * (2.0 ** -11 + 300 * 2.0 ** -24) + 1e-6, "LayerNorm")


@pytest.mark.parametrize("nk", [False, True])
@pytest.mark.parametrize("fused", [0, 1, 2])
def test_program_with_rotary_positions(hom, cuda, nk, fused):
    """Against the encoder in 64 bits with turned queries and keys; zeros as the position table.  The bound is the
    end-to-end one of the fp16 encoder."""
    from hands_on_mlir_b200.bert_program import BertProgram

    seq, lens = 90, [90, 33, 1]
    cfg, w, rng = _model(5, seq)
    w["pos_emb"] = np.zeros_like(w["pos_emb"])
    ids, mask, types = _inputs(cfg, rng, lens, seq)
    prog = BertProgram(cfg, len(lens), seq, weights_nk=nk, fused_layernorm=fused)
    stored = {n: np.ascontiguousarray(v.transpose(0, 2, 1)) if nk and n[0] == "w" and n != "word_emb" else v
              for n, v in w.items()}
    prog.set_weights({k: to_dev(v, cuda) for k, v in stored.items()})
    args = [to_dev(v, cuda) for v in (ids, mask, types)]
    plain = prog.result_to_torch(prog.forward(*args)).cpu().numpy()
    before, launches = hom.launch_count(), prog.launches_per_forward()
    prog.set_rotary(base=500.0, scaling="linear", factor=2.0, magnitude=1.1)
    assert prog.launches_per_forward() == launches + cfg.layers and hom.launch_count() == before + 1
    got = prog.result_to_torch(prog.forward(*args)).cpu().numpy()
    for _ in range(2):
        again = prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy()
        assert_bits_equal(again, got, "graph replay")
    hom.synchronize()

    freq = 500.0 ** (-np.arange(32) / 32) / 2.0
    x = _layernorm(w["word_emb"][0].astype(float)[ids] + w["type_emb"][0].astype(float)[types])
    heads = cfg.heads
    for i in range(cfg.layers):
        m = {k: w[f"{k}_{i}"][0].astype(float) for k in ("wqkv", "wo", "w1", "w2")}
        qkv = (x @ m["wqkv"]).reshape(len(lens), seq, 3 * heads, 64)
        qkv[:, :, :2 * heads] = ref.rotary(qkv[:, :, :2 * heads], None, freq, magnitude=1.1)
        q, k, v = (t.transpose(0, 2, 1, 3) for t in np.split(qkv, 3, axis=2))
        s = np.where(mask[:, None, None, :] > 0, q @ k.transpose(0, 1, 3, 2) * 0.125, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        ctx = (p / p.sum(-1, keepdims=True) @ v).transpose(0, 2, 1, 3).reshape(x.shape)
        x = _layernorm(ctx @ m["wo"] + x)
        x = _layernorm(ref.gelu(x @ m["w1"]) @ m["w2"] + x)
    for b, n in enumerate(lens):
        assert drift_fractions(got[b, :n], x[b, :n])[2] == 0.0, b
    # at position 0 of a one-token sequence nothing is turned but the stretched scores of one key: no change
    assert_bits_equal(got[2, :1], plain[2, :1], "one token at position 0")
    assert drift_fractions(plain[0], x[0])[2] > 0.0
    prog.close()


@pytest.mark.parametrize("nk", [False, True])
def test_program_with_quantized_projections(hom, pkg, cuda, nk):
    """The program is the sequence of the tested calls, bit for bit: eagerly, from a graph, from host buffers."""
    import torch
    from hands_on_mlir_b200.bert_program import BertProgram

    seq, lens = 70, [70, 9]
    bs = len(lens)
    cfg, w, rng = _model(8, seq, hidden=192, heads=3, ffn=416)
    ids, mask, types = _inputs(cfg, rng, lens, seq)
    prog = BertProgram(cfg, bs, seq, weights_nk=nk)
    tw = {n: to_dev(v.transpose(0, 2, 1) if nk and n[0] == "w" and n != "word_emb" else v, cuda) for n, v in w.items()}
    prog.set_weights(tw)
    args = [to_dev(v, cuda) for v in (ids, mask, types)]
    plain = prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy()
    plain = prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy()
    prog.quantize_weights()
    prog.set_rotary()
    got = prog.result_to_torch(prog.forward(*args)).cpu().numpy()
    launches = hom.launch_count()
    prog.forward(*args)
    assert hom.launch_count() - launches == prog.launches_per_forward() == 6 + 12 * cfg.layers
    for _ in range(3):
        assert_bits_equal(prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy(), got, "graph replay")
    pinned = [torch.from_numpy(v).pin_memory() for v in (ids, mask, types)]
    out = torch.empty((bs, seq, cfg.hidden), dtype=torch.float16).pin_memory()
    prog.forward_host(*pinned, out)
    assert_bits_equal(out.numpy(), got, "host buffers")
    for _ in range(4):
        prog.forward_host_async(*pinned, out, use_graph=True)
        prog.wait_host()
        assert_bits_equal(out.numpy(), got, "pipelined host buffers")

    # the same calls by hand
    h, rows = cfg.hidden, bs * seq
    half = dict(dtype=torch.float16, device=cuda)
    x, rest = torch.empty((bs, seq, h), **half), torch.empty((bs, seq, h), **half)
    cu, freq = torch.empty(bs + 1, dtype=torch.int32, device=cuda), torch.empty(32, dtype=torch.float64, device=cuda)
    hom.homRotaryFrequencies(freq)
    hom.thrustCuSeqLenI64(args[1], cu)
    hom.thrustGatherF16(args[0], tw["word_emb"], x)
    hom.thrustGatherF16(args[2], tw["type_emb"], rest)
    hom.thrustElementwiseAddF16(x, rest, x)
    hom.thrustElementwiseAddF16(x, tw["pos_emb"], x)
    hom.nvteLayernormF16(x, cfg.eps)

    def product(a, name, d, act=0, beta=0.0):
        k, n = a.shape[-1], d.shape[-1]
        qa, qb = ([torch.empty(s, dtype=torch.uint8, device=cuda) for s in pkg.mxf4_shapes(r, k)] for r in (rows, n))
        hom.homQuantizeMxF4F16(a.view(rows, k), *qa)
        hom.homQuantizeMxF4F16(tw[name], *qb, not nk)
        hom.homGemmMxF4F16(*qa, *qb, d.view(rows, n), d.view(rows, n), act, 1.0, beta)

    qkv, ctx, ffn = (torch.empty((bs, seq, n), **half) for n in (3 * h, h, cfg.ffn))
    for i in range(cfg.layers):
        product(x, f"wqkv_{i}", qkv)
        turned = qkv.view(bs, seq, 3 * cfg.heads, 64)[:, :, :2 * cfg.heads]
        hom.homRotaryF16(turned, None, freq, turned)
        hom.nvteBertAttentionF16(qkv, cu, ctx, 0.125, cfg.heads)
        product(ctx, f"wo_{i}", x, beta=1.0)
        hom.nvteLayernormF16(x, cfg.eps)
        product(x, f"w1_{i}", ffn, act=1)
        product(ffn, f"w2_{i}", x, beta=1.0)
        hom.nvteLayernormF16(x, cfg.eps)
    hom.synchronize()
    assert_bits_equal(x.cpu().numpy(), got, "the same calls by hand")
    assert not np.array_equal(plain, got)
    prog.close()


def test_a_refused_option_changes_nothing(hom, pkg, cuda):
    from hands_on_mlir_b200.bert_program import BertProgram

    cfg, w, rng = _model(4, 16, layers=1)
    args = [to_dev(v, cuda) for v in _inputs(cfg, rng, [16, 5], 16)]
    prog = BertProgram(cfg, 2, 16)
    prog.set_weights({k: to_dev(v, cuda) for k, v in w.items()})
    plain = prog.result_to_torch(prog.forward(*args)).cpu().numpy()
    prog.set_rotary(base=100.0, magnitude=1.2)
    prog.quantize_weights()
    want = prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy()
    assert not np.array_equal(plain, want)
    for bad in (dict(base=-1.0), dict(scaling="linear", factor=0.0), dict(magnitude=float("inf"))):
        with pytest.raises(pkg.HomError):
            prog.set_rotary(**bad)
        for graph in (True, True):
            assert_bits_equal(prog.result_to_torch(prog.forward(*args, use_graph=graph)).cpu().numpy(), want, str(bad))
    prog.close()


def test_program_refusals_and_new_weights(hom, pkg, cuda):
    from hands_on_mlir_b200.bert_program import BertProgram

    seq = 16
    cfg, w, rng = _model(2, seq, layers=1)
    ids, mask, types = _inputs(cfg, rng, [16, 5], seq)
    args = [to_dev(v, cuda) for v in (ids, mask, types)]
    fused = BertProgram(cfg, 2, seq, fused_layernorm=1)
    with pytest.raises(pkg.HomError):
        fused.quantize_weights()  # nothing bound
    fused.set_weights({k: to_dev(v, cuda) for k, v in w.items()})
    with pytest.raises(pkg.HomError):
        fused.quantize_weights()
    with pytest.raises(pkg.HomError):
        fused.set_rotary(base=-1.0)
    with pytest.raises(pkg.HomError):
        fused.set_rotary(magnitude=float("nan"))
    fused.close()

    prog = BertProgram(cfg, 2, seq)
    tw = {k: to_dev(v, cuda) for k, v in w.items()}
    prog.set_weights(tw)
    prog.quantize_weights()
    first = prog.result_to_torch(prog.forward(*args)).cpu().numpy()
    other = {k: to_dev(v, cuda) for k, v in _model(3, seq, layers=1)[1].items()}
    prog.set_weights(other)
    with pytest.raises(pkg.HomError):
        prog.forward(*args)
    hom.clear_error()
    prog.quantize_weights()
    second = prog.result_to_torch(prog.forward(*args, use_graph=True)).cpu().numpy()
    assert not np.array_equal(first, second)
    tw["wqkv_0"].mul_(1.0)
    prog.set_weights(tw)
    prog.quantize_weights()
    for graph in (False, True, True):
        assert_bits_equal(prog.result_to_torch(prog.forward(*args, use_graph=graph)).cpu().numpy(), first, "back again")
    prog.close()
