"""A whole INT4 / BF16 layer in one launch (dsgx_moe_block_decode) against the layer's formula in 64 bits.

Tolerance, by arithmetic, per output element.  With gamma(K) = (80 + K / 512) 2^-23 a product's f32 sum is off by at most gamma A,
A = sum |x| (u + z) s (INT4: see the dense products' tests; bf16 weights: exact products, A = sum |x| |W|).  dg, du for gate and
up; silu's slope is below 1.1, and h is rounded once to bf16.  silu's exponential is the fast one, within 2 + 1.16 |g| steps of
2^-23 by CUDA's error table: below 95 for |g| <= 80 (beyond that silu is g or below 2^-100), with the division's 2 and the
product's half a step less than 128 x 2^-23 = 2^-16 of the value:
    dh = 1.1 dg (|u| + du) + |silu(g)| du + |h| (2^-8 + 2^-16)      (2^-8: half a step of bf16 relative to the value)
    dy = sum_c |W| dh_c + gamma(I) sum_c (|h| + dh)_c (u + z) s
    dout = sum_e w_e dy_e + dy_shared + 2^-20 (sum_e w_e |y_e| + |y_shared| + |res|) + 2^-8 |out|
(the adds of at most eight picks, the shared expert and the residual, and w's last bits, stay below 2^-20 of what is added).
The picks are those of dsgx_route on dsgx_router_logits, bit for bit."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _gamma(K):
    return (80 + K // 512) * 2.0 ** -23


def _canonical(layer, e):
    """(W, bound) f64 of an expert's three matrices on the GPU, from the packed blocks' address rule."""
    from tests.linear_util import unpack
    out = []
    for m, (N, K) in enumerate(((layer.I, layer.H), (layer.I, layer.H), (layer.H, layer.I))):
        if layer.fmt == 3:
            w = torch.from_numpy((layer.bits[e][m].astype(np.uint32) << 16).view(np.float32).astype(np.float64)).cuda()
            out.append((w, w.abs()))
            continue
        off, nb = layer.desc_host[e * 3 + m].off, N // 8 * (K // 512) * 2368
        w, b = unpack(layer.pool[off:off + nb].cpu().numpy(), N, K, bound=True)
        out.append((torch.from_numpy(w).cuda(), torch.from_numpy(b).cuda()))
    return out


def _shared(layer):
    return [(w, w.abs()) for w in (torch.from_numpy((b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)).cuda() for b in layer.sh_bits)]


def _ffn(x, mats):
    """(y, dy) of rows x through one expert."""
    (wg, bg), (wu, bu), (wd, bd) = mats
    g, u, ax = x @ wg.T, x @ wu.T, x.abs()
    dg, du = _gamma(x.shape[1]) * (ax @ bg.T), _gamma(x.shape[1]) * (ax @ bu.T)
    act = g * torch.sigmoid(g)
    h = act * u
    dh = 1.1 * dg * (u.abs() + du) + act.abs() * du + h.abs() * (2.0 ** -8 + 2.0 ** -16)
    return h @ wd.T, dh @ wd.abs().T + _gamma(h.shape[1]) * ((h.abs() + dh) @ bd.T)


def _expect(layer, x, idx, w, res, shared):
    x, w = x.double(), w.double()
    out, tol, size = (torch.zeros_like(x) for _ in range(3))
    for e in torch.unique(idx).tolist():
        m, k = (idx == e).nonzero(as_tuple=True)
        y, dy = _ffn(x[m], _canonical(layer, e))
        out[m] += w[m, k, None] * y
        tol[m] += w[m, k, None] * dy
        size[m] += w[m, k, None] * y.abs()
    if shared:
        y, dy = _ffn(x, _shared(layer))
        out, tol, size = out + y, tol + dy, size + y.abs()
    if res is not None:
        out, size = out + res.double(), size + res.double().abs()
    return out, tol + 2.0 ** -20 * size + 2.0 ** -8 * out.abs() * (1 + 2.0 ** -7)


def _setup(H, I, E, topk, seed, fmt=2, shared=True, zeros=True, **route):
    from dsgx10_b200 import moe, synth
    shp = moe.shape(H, I, E, topk, fmt=fmt, **route)
    layer = (synth.Bf16Layer if fmt == 3 else synth.Int4Layer)(H, I, E, seed, device="cuda", shared=shared)
    if fmt == 2 and zeros:  # asymmetric zero points
        z = layer.pool.view(-1, 2368)[:, 2304:]
        z.copy_(torch.randint(0, 256, z.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed)).cuda())
    return shp, layer, synth.router_weights(E, H, seed + 2).cuda()


def _check(shp, layer, wr, x, bias=None, res=None, shared=True, block=None):
    from dsgx10_b200 import moe
    block = moe.MoeBlock(shp, wr, bias) if block is None else block
    got, idx, w = block.run(layer.layer_w(), x, res=res)
    torch.cuda.synchronize()
    assert moe.ws_status(block.ws) == 0
    want_idx, want_w = moe.route(shp, moe.router_logits(x, wr), bias)
    assert torch.equal(idx, want_idx) and torch.equal(w, want_w)
    out, tol = _expect(layer, x, idx.long(), w, res, shared)
    err = (got.double() - out).abs()
    assert bool((err <= tol + 1e-30).all()), float((err / (tol + 1e-30)).max())
    return block, got.clone()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 7, 8, 11, 16])
def test_rows(M):
    from dsgx10_b200 import synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 300)
    _check(shp, layer, wr, synth.activations(M, 1024, 301 + M).cuda(), res=synth.activations(M, 1024, 400 + M).cuda())


@pytest.mark.parametrize("H,I,E,topk,M,kw", [
    (512, 512, 1, 1, 1, {}),                                            # the smallest layer: one expert, one block along K
    (512, 1536, 3, 3, 8, dict(score_fn=1, shared=False)),               # every row picks every expert: all sets of eight rows
    (2560, 512, 40, 8, 6, dict(score_fn=2, route_scale=1.5)),
    (1536, 1024, 33, 5, 4, dict(score_fn=0, norm_topk=False)),
    (1024, 2048, 64, 8, 7, dict(n_group=8, topk_group=3, route_scale=2.5, shared=False)),
    (6144, 2048, 12, 8, 2, dict(score_fn=1)),                           # full widths, few experts
    (6144, 1024, 10, 4, 8, dict(score_fn=1)),                           # one tile of activations only
    (8192, 512, 4, 2, 8, {}),                                           # the rows in two launches
    (512, 512, 500, 8, 3, {}),
])
def test_shapes(H, I, E, topk, M, kw):
    from dsgx10_b200 import synth
    shared = kw.get("shared", True)
    shp, layer, wr = _setup(H, I, E, topk, H + I + E, **kw)
    bias = torch.randn(E, generator=torch.Generator().manual_seed(5)).cuda() if kw.get("score_fn") == 0 else None
    _check(shp, layer, wr, synth.activations(M, H, 7).cuda(), bias=bias, shared=shared)


@pytest.mark.parametrize("M", [1, 5, 8])
def test_bf16_layer(M):
    from dsgx10_b200 import synth
    shp, layer, wr = _setup(1024, 512, 8, 2, 970, fmt=3, score_fn=1)
    _check(shp, layer, wr, synth.activations(M, 1024, 972 + M).cuda(), res=synth.activations(M, 1024, 9).cuda())


def test_interleaved_shared_expert_same_bits():
    from dsgx10_b200 import _lib, moe, synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 140)
    x = synth.activations(5, 1024, 141).cuda()
    block, got = _check(shp, layer, wr, x)
    gu = np.empty((2 * 512, 1024), np.uint16)
    gu[0::2], gu[1::2] = layer.sh_bits[0], layer.sh_bits[1]
    bgu = torch.from_numpy(synth.tile_bf16(gu)).cuda()
    lw = layer.layer_w()
    lw.sh.bg, lw.sh.bu, lw.sh.bgu = None, None, bgu.data_ptr()
    assert torch.equal(block.run(lw, x)[0], got)
    lw.sh.bu = layer.sh_dev[1].data_ptr()
    with pytest.raises(_lib.DsgxError):
        block.run(lw, x)


def test_rows_do_not_depend_on_each_other_and_runs_repeat():
    """A row alone or with up to fifteen others: the same bits (other unions, other deals of the units); again and again."""
    from dsgx10_b200 import moe, synth
    for H, I, E, topk in ((1024, 512, 16, 4), (2048, 1024, 6, 5)):
        shp, layer, wr = _setup(H, I, E, topk, 131)
        block = moe.MoeBlock(shp, wr)
        x = synth.activations(16, H, 132).cuda()
        lw = layer.layer_w()
        full = block.run(lw, x)[0].clone()
        for _ in range(20):
            assert torch.equal(block.run(lw, x)[0], full)
        for a, b in ((0, 1), (3, 4), (15, 16), (2, 5), (0, 8), (4, 13), (7, 16)):
            assert torch.equal(block.run(lw, x[a:b].contiguous())[0], full[a:b]), (a, b)
        assert moe.ws_status(block.ws) == 0


def test_in_place_graph_and_streams():
    """A chain of layers that share the residual stream, captured and replayed on new inputs; two layers on two streams."""
    from dsgx10_b200 import moe, synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 150)
    blocks = [moe.MoeBlock(shp, wr) for _ in range(2)]
    lw = layer.layer_w()
    xs = [synth.activations(3, 1024, 151 + i).cuda() for i in range(4)]

    def chain(x):  # x += MoE(x), twice, in place
        for b in blocks:
            b.run(lw, x, res=x, out=x)
        return x

    want = [chain(x.clone()) for x in xs]
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(x)
    for i in (2, 0, 3):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want[i])
    one = [blocks[0].run(lw, x, res=x)[0].clone() for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(blocks[i % 2].run(lw, xs[i], res=xs[i])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, one))
    assert all(moe.ws_status(b.ws) == 0 for b in blocks)


def test_a_row_of_nan_leaves_the_others():
    from dsgx10_b200 import moe, synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 160)
    block = moe.MoeBlock(shp, wr)
    x = synth.activations(6, 1024, 161).cuda()
    lw = layer.layer_w()
    clean = block.run(lw, x)[0].clone()
    x[2, 17] = float("nan")
    got = block.run(lw, x)[0]
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(got[keep], clean[keep]) and moe.ws_status(block.ws) == 0
    x[2] = 0
    _check(shp, layer, wr, x, block=block)


def test_with_the_dense_products():
    """The two operators as a model uses them: a projection with its residual, then the layer on the stream."""
    from dsgx10_b200 import linear, moe, synth, weights
    from tests.linear_util import random_int4
    H, M = 1024, 4
    shp, layer, wr = _setup(H, 512, 16, 4, 170)
    wp, s, zp, w, b = random_int4(H, H, 171)
    proj = linear.LinearW(H, H, torch.from_numpy(weights.pack_linear_int4(wp, s, zp)).cuda())
    a, r = synth.activations(M, H, 172).cuda(), synth.activations(M, H, 173).cuda()
    x = linear.linear_decode(proj, a, res=r)
    y = a.double() @ torch.from_numpy(w).cuda().T + r.double()
    tol = 2.0 ** -8 * y.abs() * (1 + 2.0 ** -7) + _gamma(H) * (a.double().abs() @ torch.from_numpy(b).cuda().T) + 2.0 ** -24 * y.abs()
    assert bool(((x.double() - y).abs() <= tol).all())
    _check(shp, layer, wr, x, res=x)


def test_refusals():
    from dsgx10_b200 import _lib, moe, synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 180)
    block = moe.MoeBlock(shp, wr)
    x = synth.activations(2, 1024, 181).cuda()
    lw = layer.layer_w()
    for bad in (x.float(), x[:, :512], x.cpu(), x.T):
        with pytest.raises(ValueError):
            block.run(lw, bad)
    with pytest.raises(ValueError):
        block.run(lw, x, res=x[:1])
    with pytest.raises(ValueError):
        moe.MoeBlock(shp, wr.double())
    with pytest.raises(_lib.DsgxError):
        block.run(lw, synth.activations(17, 1024, 1).cuda())
    fp8 = layer.layer_w()
    fp8.fmt = _lib.FMT_BF16
    with pytest.raises(_lib.DsgxError):
        block.run(fp8, x)
    # descriptors of another format: found on the device, reported, the routed experts left out
    shp16 = moe.shape(1024, 512, 16, 4, fmt=_lib.FMT_BF16)
    b16 = moe.MoeBlock(shp16, wr)
    out, _, _ = b16.run(fp8, x)
    torch.cuda.synchronize()
    assert moe.ws_status(b16.ws) == _lib.ERR_FORMAT
    y, tol = _ffn(x.double(), _shared(layer))
    assert bool(((out.double() - y).abs() <= tol + 2.0 ** -8 * y.abs() + 2.0 ** -20 * y.abs()).all())


def test_layers_and_products_at_once():
    """Layers on one stream while dense products of all divisions (clusters, pairs of them, one CTA) run on two others."""
    from dsgx10_b200 import linear, moe, synth
    shp, layer, wr = _setup(1024, 512, 16, 4, 190)
    blocks, lw = [moe.MoeBlock(shp, wr) for _ in range(2)], layer.layer_w()
    xs = [synth.activations(m, 1024, 191 + m).cuda() for m in (1, 5, 8, 13)]
    ws = []
    for M, N, K in ((1, 4096, 2048), (16, 1000, 9000), (8, 512, 6144), (3, 131, 300)):
        n = -(-N // 8) * -(-K // 512)
        b = torch.randint(0, 256, (n, 2368), dtype=torch.uint8, device="cuda")
        b[:, 2048:2304].view(n, 128, 2)[:, :, 1] = 0x3B
        ws.append((linear.LinearW(N, K, b.view(-1)), synth.activations(M, K, 200 + M).cuda()))
    want = [blocks[0].run(lw, x)[0].clone() for x in xs], [linear.linear_decode(w, x) for w, x in ws]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [], [], []
    for i in range(12):
        with torch.cuda.stream(streams[0]):
            got[0].append(blocks[0].run(lw, xs[i % 4])[0])
        for k in (1, 2):
            with torch.cuda.stream(streams[k]):
                got[k].append([linear.linear_decode(w, x) for w, x in ws])
                if k == 2:
                    got[k][-1].append(blocks[1].run(lw, xs[(i + 1) % 4])[0])
    torch.cuda.synchronize()
    assert all(moe.ws_status(b.ws) == 0 for b in blocks)
    assert all(torch.equal(y, want[0][i % 4]) for i, y in enumerate(got[0]))
    for k in (1, 2):
        for i, ys in enumerate(got[k]):
            assert all(torch.equal(a, b) for a, b in zip(ys[:4], want[1]))
            assert k == 1 or torch.equal(ys[4], want[0][(i + 1) % 4])
