"""The whole-layer call held closely to 64 bits: rows in the mean, every element of its stages (tests/block_util.py)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _layer(H, I, E, seed, fmt=2, shared=True):
    """Any zero points, in the block layout on the device (packing full widths through the host takes minutes)."""
    from dsgx10_b200 import synth
    if fmt == 3:
        return synth.Bf16Layer(H, I, E, seed, device="cuda", shared=shared)
    layer = synth.Int4Layer.on_device(H, I, E, seed, "cuda", shared=shared)
    z = layer.pool.view(-1, 2368)[:, 2304:]
    z.copy_(torch.randint(0, 256, z.shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return layer


def _run(H, I, E, topk, M, fmt=2, shared=True, res=False, **kw):
    from dsgx10_b200 import moe, synth
    from tests import block_util as U
    layer = _layer(H, I, E, H + E, fmt, shared)
    block = moe.MoeBlock(moe.shape(H, I, E, topk, fmt=fmt, **kw), synth.router_weights(E, H, 3).cuda())
    x = synth.activations(M, H, 4).cuda()
    r = synth.activations(M, H, 5).cuda() if res else None
    got, idx, w = block.run(layer.layer_w(), x, res=r)
    torch.cuda.synchronize()
    assert moe.ws_status(block.ws) == 0
    out, parts = U.reference(layer, x, idx.long(), w, r, shared)
    ratio = U.check_rows(got, out, parts)
    assert ratio <= 1, ratio
    h, y = U.stages(block, H, I)
    U.check_stages(layer, x, idx.long(), w, h, y, got, r, shared)


@pytest.mark.parametrize("M", [1, 2, 4, 5, 8])
def test_small(M):
    _run(1024, 512, 16, 4, M, res=M == 2)


@pytest.mark.parametrize("H,I,E,topk,M,kw", [
    (512, 512, 4, 4, 8, {}),                                       # one task a unit; all eight rows on every expert
    (1024, 2048, 24, 8, 3, dict(score_fn=1)),
    (2560, 1536, 20, 5, 7, dict(score_fn=2, route_scale=1.5)),     # odd numbers of blocks along K, tasks of two and of one
    (4096, 4096, 6, 3, 6, dict(score_fn=1)),                       # down tiles as large as x's
    (2048, 1024, 64, 8, 8, dict(n_group=8, topk_group=4, route_scale=2.5, shared=False)),
    (1024, 1024, 8, 2, 5, dict(fmt=3)),
    (1024, 512, 8, 4, 4, dict(fmt=3, shared=False)),
])
def test_shapes(H, I, E, topk, M, kw):
    _run(H, I, E, topk, M, **kw)


@pytest.mark.parametrize("M", [1, 4, 8])
def test_full_widths_and_all_experts(M):
    """hidden 6144, 168 experts of 2048, top-8 softmax, shared expert."""
    _run(6144, 2048, 168, 8, M, score_fn=1)


def test_the_four_launches_are_as_near_as_their_roundings():
    """dsgx_moe_layer_decode rounds W (three times), g, u and h to bf16 where this call does not: six roundings of at most 2^-8 of a
    value, independent, each passed on like the value it is in, so a row is apart by at most sqrt(6) 2^-8 of its parts; both outputs
    are rounded once."""
    from dsgx10_b200 import moe, synth
    from tests import block_util as U
    for H, I, E, topk, M in ((1024, 512, 16, 4, 3), (6144, 2048, 24, 8, 4)):
        layer = _layer(H, I, E, 9)
        shp, wr, x = moe.shape(H, I, E, topk, fmt=2, score_fn=1), synth.router_weights(E, H, 10).cuda(), synth.activations(M, H, 11).cuda()
        got, idx, w = moe.MoeBlock(shp, wr).run(layer.layer_w(), x)
        four = moe.LayerStep(shp, wr).run(layer.layer_w(), x)
        torch.cuda.synchronize()
        out, parts = U.reference(layer, x, idx.long(), w)
        apart = (got.double() - four.double()).pow(2).sum(1).sqrt()
        assert bool((apart <= 2 * 2.0 ** -8 * out.pow(2).sum(1).sqrt() + 6 ** 0.5 * 2.0 ** -8 * parts.sum(1).sqrt()).all())
        assert U.check_rows(got, out, parts) <= 1 < U.check_rows(four, out, parts)
