"""Rows whose values lie far apart, both 4-bit operators.

A block of 512 k goes to f16 by its largest value's power of two.  What is far below that rounds by at most 2^-35 of the largest (odd k;
2^-39 at even k), which (u + z) s carries into the sum: the term `small` beside the products' other bounds.  An output in f32's
subnormal range is off by half a step of 2^-149 more for each of a row's blocks and joins, in bf16 by 2^-134."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _rows(kind, M, K, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g).double()
    at = torch.arange(M)[:, None] * 7 + torch.arange(0, K, 512)[None, :]      # even and odd places, one a block
    at = at.clamp_max(K - 1)
    if kind == "spread":            # every power of two from 2^-40 to 1 in one block
        x = x * torch.exp2(-torch.randint(0, 41, (M, K), generator=g).double())
    elif kind in ("2^20", "2^30"):  # one value far above the others
        x.scatter_(1, at, 2.0 ** int(kind[2:]))
    elif kind == "subnormal":       # all of a row below bf16's smallest normal number
        x = x * 2.0 ** -128
    elif kind == "largest":         # bf16's largest number, once a block, beside ordinary ones
        x.scatter_(1, at, 3.3895313892515355e38)
    elif kind == "zero":
        x[::2] = 0
        x[1::2, :K // 2] = 0
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("kind", ["spread", "2^20", "2^30", "subnormal", "largest", "zero"])
@pytest.mark.parametrize("M,N,K", [(1, 24, 512), (3, 40, 1300), (7, 300, 2560), (16, 33, 700)])
def test_products(kind, M, N, K):
    from dsgx10_b200 import linear, weights
    from tests.linear_util import random_int4
    wp, s, zp, w, b = random_int4(N, K, 17)
    w, b = torch.from_numpy(w), torch.from_numpy(b)
    x = _rows(kind, M, K, K + M)
    got = linear.linear_decode(linear.LinearW(N, K, torch.from_numpy(weights.pack_linear_int4(wp, s, zp, K=K)).cuda()), x.cuda(), out_dtype=torch.float32)
    xd, nb = x.double(), -(-K // 512)
    top = torch.cat([xd[:, i:i + 512].abs().amax(1, keepdim=True).expand(M, min(512, K - i)) for i in range(0, K, 512)], 1)
    y = xd @ w.T
    tol = 2.0 ** -24 * y.abs() + (80 + nb) * 2.0 ** -23 * (xd.abs() @ b.T) + 2.0 ** -35 * (top @ b.T) + (nb + 8) * 2.0 ** -150
    err = (got.double().cpu() - y).abs()
    assert bool((err <= tol * (1 + 2.0 ** -7)).all()), float((err / tol).max())


@pytest.mark.parametrize("kind", ["spread", "2^20", "subnormal", "zero"])
@pytest.mark.parametrize("M", [2, 7])
def test_layer(kind, M):
    """Every element of the layer's stages, as in the ordinary range."""
    from dsgx10_b200 import moe, synth
    from tests import block_util as U
    H, I, E = 1536, 1024, 12
    layer = synth.Int4Layer.on_device(H, I, E, 31, "cuda")
    z = layer.pool.view(-1, 2368)[:, 2304:]
    z.copy_(torch.randint(0, 256, z.shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)))
    block = moe.MoeBlock(moe.shape(H, I, E, 4, fmt=2), synth.router_weights(E, H, 32).cuda())
    x = _rows(kind, M, H, 33 + M).cuda()
    got, idx, w = block.run(layer.layer_w(), x)
    torch.cuda.synchronize()
    assert moe.ws_status(block.ws) == 0 and bool(got.isfinite().all())
    h, y = U.stages(block, H, I)
    U.check_stages(layer, x, idx.long(), w, h, y, got)
