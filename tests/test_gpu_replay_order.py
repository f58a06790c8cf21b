"""Forwards of a program issued one after the other on the default stream, with nothing between them that waits: each
takes milliseconds, far longer than the host needs to issue the next."""
import numpy as np
import pytest

from util import to_dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fused", [0, 2])
def test_forwards_back_to_back_on_the_default_stream(hom, cuda, fused):
    import torch
    from hands_on_mlir_b200.bert_program import BertConfig, BertProgram

    assert torch.cuda.current_stream().cuda_stream == 0
    batch, seq = 32, 512
    cfg = BertConfig(layers=4, hidden=1024, heads=16, ffn=4096, vocab=500)
    rng = np.random.default_rng(17)
    weights = {n: to_dev(rng.normal(0, 0.03, cfg.weight_shape(n, seq)).astype(np.float16), cuda) for n in cfg.weight_names()}
    lens = rng.integers(1, seq + 1, batch)
    args = [to_dev(v, cuda) for v in (rng.integers(0, cfg.vocab, (batch, seq)).astype(np.int64),
                                      (np.arange(seq)[None] < lens[:, None]).astype(np.int64),
                                      rng.integers(0, 2, (batch, seq)).astype(np.int64))]
    prog = BertProgram(cfg, batch, seq, fused_layernorm=fused)
    prog.set_weights(weights)

    def results(graphs):
        return [prog.result_to_torch(prog.forward(*args, use_graph=g)) for g in graphs]

    def agree(got, want):
        assert bool(want.isfinite().all())
        for i, r in enumerate(got):
            assert torch.equal(r, want), i

    want = results([False])[0]
    hom.synchronize()
    agree(results([False, False, True, True, True, False, True]), want)
    prog.set_rotary()
    if fused == 0:
        prog.quantize_weights()
    changed = results([False, True, True, True])
    want = results([False])[0]
    hom.synchronize()
    agree(changed, want)
    prog.close()
