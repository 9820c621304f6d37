"""A call that takes two pieces of scratch has two: activations that are not 16-byte
aligned are copied into one, and the route they are copied for (parts of K, or slabs
of dequantized weights ahead of a library product) uses another."""
import pytest
import torch

from test_gpu_workspace import _bf
from ubridge_amd import ops, synth

pytestmark = pytest.mark.gpu


def misaligned(a):
    buf = torch.zeros(a.numel() + 1, dtype=a.dtype, device=a.device)
    buf[1:] = a.reshape(-1)
    m = buf[1:].view(a.shape)
    assert m.data_ptr() % 16 == 2
    return m


@pytest.mark.parametrize("M,K,N", [(2, 8192, 1032), (16, 8192, 1032), (72, 4096, 1544), (40, 8192, 776), (1096, 768, 1048)])
def test_misaligned_activations(dev, M, K, N):
    qw, sc, qz = synth.make_gptq_w4(K, N, 128, seed=M)
    args = torch.from_numpy(qw).cuda(), _bf(sc), torch.from_numpy(qz).cuda(), 128
    a = _bf(synth.bf16_activations(M, K, seed=M + 1))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = ops.w4a16_gemm(a, *args)
        m = misaligned(a)
        ops.release_workspace(s)
        n = ops.workspace_stats()[0]
        for _ in range(3):
            assert torch.equal(ops.w4a16_gemm(m, *args), want)
        assert ops.workspace_stats()[0] <= n + 2
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = ops.w4a16_gemm(m, *args)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(ops.w4a16_gemm(m, *args), want)
    del graph
    ops.release_workspace(s)
    assert ops.workspace_stats()[0] == n
