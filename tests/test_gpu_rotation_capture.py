"""A complex128 rotation table whose first use is a captured call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_table_converted_in_a_capture_is_not_kept():
    """The conversion runs with the graph's replays; an eager call before them converts for itself."""
    from flashvsr_sm89_ops import fused_rms_rope
    L, D = 256, 256
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1, L, D, generator=g).bfloat16().cuda()
    w = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    ang = torch.rand(L, 64, generator=g, dtype=torch.float64)
    table = torch.polar(torch.ones_like(ang), ang)
    want = fused_rms_rope(x, w, table.to(torch.complex64).cuda())
    freqs = table.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fused_rms_rope(x, w, freqs)
    assert torch.equal(fused_rms_rope(x, w, freqs), want)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(fused_rms_rope(x, w, freqs), want)
