"""Descriptors that the whole-layer call cannot follow: found on the device before a byte is fetched by them."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("matrix,off", [(0, 8), (1, 16), (2, 128)])
def test_an_offset_that_is_not_aligned(matrix, off):
    """One picked expert's matrix begins between two blocks: DSGX_ERR_FORMAT, the routed experts left out, the shared one and the
    residual there; with the descriptor mended the next call is right."""
    from dsgx10_b200 import _lib, moe, synth
    H, I, E, topk, M = 1024, 512, 8, 2, 3
    layer = synth.Int4Layer.on_device(H, I, E, 41, "cuda")
    shp, wr = moe.shape(H, I, E, topk, fmt=_lib.FMT_INT4), synth.router_weights(E, H, 42).cuda()
    x, lw = synth.activations(M, H, 43).cuda(), layer.layer_w()
    block = moe.MoeBlock(shp, wr)
    want, idx, _ = block.run(lw, x, res=x)
    want, e = want.clone(), int(idx[1, 0])
    d = layer.desc.view(torch.int64).view(E * 3, -1)
    d[e * 3 + matrix, 0] += off
    got = block.run(lw, x, res=x)[0]
    torch.cuda.synchronize()
    assert moe.ws_status(block.ws) == _lib.ERR_FORMAT and not torch.equal(got, want) and bool(got.isfinite().all())
    d[e * 3 + matrix, 0] -= off
    block.ws[:4].zero_()
    assert torch.equal(block.run(lw, x, res=x)[0], want) and moe.ws_status(block.ws) == 0
