"""GPU: a grouped call of 64 rows whose K split joins over the workspace, captured with
and without a warm-up; a difference is reported by linear, tile and size."""
import pytest
import torch

import int4_hip
from _synth import randn
from test_gpu_gemm import DEV, _weights

pytestmark = pytest.mark.gpu
SHAPES = [(2048, 2048), (512, 2048), (512, 2048), (2048, 2048), (8192, 2048), (8192, 2048), (2048, 8192)]


def _report(got, want):
    """Where two lists of outputs differ: linear, its shape, how many elements in which tiles
    of 128 columns, over which rows, by how much, and what stands there."""
    lines = []
    for i, (a, b) in enumerate(zip(got, want)):
        bad = a.view(torch.int16) != b.view(torch.int16)
        if bad.any():
            rows, cols = bad.nonzero(as_tuple=True)
            off = (a.float() - b.float()).abs()[bad]
            lines.append(f"linear {i} (N, K = {SHAPES[i]}): {int(bad.sum())} of {bad.numel()} in column tiles "
                         f"{sorted(set((cols // 128).tolist()))}, rows {rows.min()}..{rows.max()}, off by up to "
                         f"{off.max().item():.4g} (outputs of {b.float().std().item():.3g}), "
                         f"{int((a[bad] == 0).sum())} of them zero; first got {a[bad][:4].tolist()} for "
                         f"{b[bad][:4].tolist()}")
    return "; ".join(lines)


@pytest.mark.parametrize("warm", [True, False])
def test_captured_64_row_block(warm):
    ws = [_weights(N, K, 128, seed=700 + i) for i, (N, K) in enumerate(SHAPES)]
    xs = [randn((64, K), seed=710 + i).to(DEV) for i, (N, K) in enumerate(SHAPES)]
    eager = int4_hip.w4a16_matmul_grouped(xs, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    if warm:
        with torch.cuda.stream(side):
            other = int4_hip.w4a16_matmul_grouped(xs, ws)
        torch.cuda.current_stream().wait_stream(side)
        assert not (said := _report(other, eager)), said
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = int4_hip.w4a16_matmul_grouped(xs, ws)
    for replay in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert not (said := _report(outs, eager)), f"replay {replay}: {said}"
        again = int4_hip.w4a16_matmul_grouped(xs, ws)  # eager work between replays
        assert not (said := _report(again, eager)), f"eager after replay {replay}: {said}"
