"""Column sums (bias gradients): rows split over workgroups and joined in a fixed order, against 64 bits; two calls give equal bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 8), (7, 13, 16), (128, 256, 256), (129, 257, 264), (1000, 31, 32), (12544, 768, 768), (333, 3000, 3008), (40001, 40, 48)])
def test_column_sums(rows, cols, ld, scaled):
    from vilmedic_amd import ops
    from vilmedic_amd._lib import check, lib, ptr, stream
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(rows, ld, generator=g).to(torch.bfloat16)
    start = torch.randn(cols + 3, generator=g)
    scale = torch.tensor([0.37], device=dev()) if scaled else None
    xd = x.to(dev())
    outs = []
    for _ in range(2):
        out = start.to(dev())
        ops.colsum(xd, out, cols=cols, scale_dev=scale)
        outs.append(out.cpu())
    alone = start.to(dev())                                   # the form without a workspace
    check(lib().vm_colsum_bf16(ptr(xd), ld, ptr(alone), rows, cols, ptr(scale), stream()), "vm_colsum_bf16")
    assert torch.equal(outs[0], outs[1])
    f = float(scale.cpu()) if scaled else 1.0
    want = start[:cols].double() + f * x[:, :cols].double().sum(0)
    # fp32 sums in any order: half a step for each addition, of at most the sum of magnitudes, the scale's product and the last addition
    tol = 2.0 ** -24 * ((rows + 2) * f * x[:, :cols].double().abs().sum(0) + 2 * want.abs() + start[:cols].double().abs()) * 1.01
    for out in (outs[0], alone.cpu()):
        assert bool(((out[:cols].double() - want).abs() <= tol).all())
        assert torch.equal(out[cols:], start[cols:])


def test_column_sums_in_a_graph_replayed_beside_eager_calls():
    from vilmedic_amd import ops
    x = torch.randn(5000, 96, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev())
    other = torch.randn(5000, 96, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev())
    want, out = torch.zeros(96, device=dev()), torch.zeros(96, device=dev())
    ops.colsum(x, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.colsum(x, torch.zeros(96, device=dev()))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.zero_()
        ops.colsum(x, out)
    for _ in range(4):
        graph.replay()
        ops.colsum(other, torch.zeros(96, device=dev()))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
