"""Run in a fresh process: the library's first calls on the device are captured into a graph, under the strictest capture
mode; its replays must leave what eager calls leave.  Prints `ok`."""
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from __graft_entry__ import load_package  # noqa: E402

pkg = load_package()
hom = pkg.runner()
torch.manual_seed(0)
m, k, n = int(sys.argv[1]), 512, 640
x, w = (torch.randn(s, device="cuda").half() for s in ((m, k), (1, k, n)))
freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)


def coded(rows):
    return [torch.empty(s, dtype=torch.uint8, device="cuda") for s in pkg.mxf4_shapes(rows, k)]


a, b = coded(m), coded(n)
out = torch.empty((1, m, n // 64, 64), dtype=torch.float16, device="cuda")


def calls():
    hom.homQuantizeMxF4F16(x, *a)
    hom.homQuantizeMxF4F16(w, *b, True)
    hom.homGemmMxF4F16(*a, *b, None, out.view(m, n), 1)
    hom.homRotaryF16(out, None, freq, out)


stream = torch.cuda.Stream()
stream.wait_stream(torch.cuda.current_stream())
hom.set_stream(stream.cuda_stream)
with torch.cuda.stream(stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="global"):
        calls()
    graph.replay()
    stream.synchronize()
    first = out.clone()
    out.zero_()
    calls()
    stream.synchronize()
    assert torch.equal(first, out) and bool(first.isfinite().all()) and bool(first.any())
hom.synchronize()
print("ok")
