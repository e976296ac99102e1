"""A bounded wait of the whole-layer kernel that runs out: reported, and the workspace is ready for the next call."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,shared", [(3, True), (11, False)])
def test_a_wait_that_runs_out(M, shared):
    """The counter of the router's logits, the workspace's first word behind the status, begins one too low: the routing CTAs never see
    them complete and every other CTA waits for a table that does not come, a second or two in all.  Eleven rows are two launches, of
    which the second is right."""
    from dsgx10_b200 import _lib, moe, synth
    H, I, E, topk = 1024, 512, 16, 4
    shp = moe.shape(H, I, E, topk, fmt=_lib.FMT_INT4)
    layer, wr = synth.Int4Layer.on_device(H, I, E, 61, "cuda", shared=shared), synth.router_weights(E, H, 62).cuda()
    x, lw = synth.activations(M, H, 63).cuda(), layer.layer_w()
    want = moe.MoeBlock(shp, wr).run(lw, x)[0].clone()
    block = moe.MoeBlock(shp, wr)
    block.ws[256:260].view(torch.int32).fill_(-1)
    got = block.run(lw, x)[0]
    torch.cuda.synchronize()
    assert moe.ws_status(block.ws) == _lib.ERR_DEVICE_WAIT
    assert torch.equal(got[8:], want[8:])
    block.ws[:4].zero_()
    for _ in range(2):
        got = block.run(lw, x)[0]
        torch.cuda.synchronize()
        assert moe.ws_status(block.ws) == 0 and torch.equal(got, want)
