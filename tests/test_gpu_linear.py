"""The dense INT4 products (dsgx_linear_decode) against the formula in 64 bits.

Tolerance, by arithmetic.  The kernel forms sum u x and z sum x of every group of 32 apart and subtracts.  A product u x has at
most 4 + 8 significant bits: exact.  sum u x is two MMAs of 16 products, each adding with at most one truncation (2^-23 of
the running magnitude) a product and one for its accumulator: 34; sum x is 32 adds of 2^-24, times z and into the difference
by one fused multiply-add: 17 x 2^-23; the scale by another one; 16 groups a block and at most nb / 8 + 1 blocks a run in
sequence, the runs' three levels, each 2^-24.  So |y - exact| <= GAMMA A with A = sum |x| (u + z) s and
GAMMA = (34 + 17 + 8 + nb / 16 + 3) 2^-23 < (80 + nb) 2^-23; the one rounding of the output adds 2^-8 |y| (bf16) or 2^-24 |y| (f32).
(x in f16 with its block's power of two is exact for these inputs: none is below 2^-32 of its block's largest.)"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _make(N, K, seed, zeros=True):
    from dsgx10_b200 import weights
    from tests.linear_util import random_int4
    wp, s, zp, w, bound = random_int4(N, K, seed, zeros)
    return torch.from_numpy(weights.pack_linear_int4(wp, s, zp, K=K)).cuda(), torch.from_numpy(w), torch.from_numpy(bound)


def _x(M, K, seed):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def _gamma(K):
    return (80 + -(-K // 512)) * 2.0 ** -23


def _check(got, y, A, K, extra=0.0):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    err = (got.double().cpu() - y).abs()
    tol = (half * y.abs() + _gamma(K) * A + extra) * (1 + 2.0 ** -7) + 1e-38
    assert bool((err <= tol).all()), float((err / tol).max())


SHAPES = [(1, 1, 1), (1, 8, 512), (2, 9, 513), (3, 17, 31), (4, 16, 32), (1, 33, 64), (5, 100, 1000), (8, 257, 2049), (9, 300, 1537),
          (16, 1000, 4100), (16, 40, 12800), (8, 24, 20000), (1, 5000, 700), (4, 4744, 1024), (7, 2400, 3600), (12, 6000, 600), (2, 20001, 96)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("f32", [False, True])
def test_product(M, N, K, f32):
    from dsgx10_b200 import linear
    blocks, w, wb = _make(N, K, 11 * N + K)
    x = _x(M, K, M + K)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = linear.linear_decode(linear.LinearW(N, K, blocks), x.cuda(), out_dtype=torch.float32 if f32 else torch.bfloat16, status=status)
    assert int(status) == 0
    _check(got, x.double() @ w.T, x.double().abs() @ wb.T, K)


@pytest.mark.parametrize("M,N,K", [(1, 7, 40), (4, 1000, 1024), (6, 129, 3000), (16, 520, 5120), (1, 9000, 2048)])
def test_swiglu(M, N, K):
    """h = silu(g) u: an error dg moves silu by at most 1.1 dg (its slope is below 1.1); expf, the division and the product
    are within 8 x 2^-24 of the value."""
    from dsgx10_b200 import linear
    (bg, wg, bwg), (bu, wu, bwu) = _make(N, K, 5), _make(N, K, 6, zeros=False)
    x = _x(M, K, 3)
    got = linear.linear_decode(linear.LinearW(N, K, bg, up=bu), x.cuda())
    g, u = x.double() @ wg.T, x.double() @ wu.T
    dg, du = (_gamma(K) * (x.double().abs() @ w.T) for w in (bwg, bwu))
    act = g * torch.sigmoid(g)
    h = act * u
    _check(got, h, 0 * h, K, extra=1.1 * dg * (u.abs() + du) + act.abs() * du + h.abs() * 8 * 2.0 ** -24)


@pytest.mark.parametrize("f32", [False, True])
def test_residual_and_in_place(f32):
    """One rounding after the residual's add (which rounds once more in f32: 2^-24 of the sum)."""
    from dsgx10_b200 import linear
    M, N, K = 5, 333, 1500
    blocks, w, wb = _make(N, K, 21)
    x, res = _x(M, K, 22), _x(M, N, 23)
    lw = linear.LinearW(N, K, blocks)
    y = x.double() @ w.T + res.double()
    got = linear.linear_decode(lw, x.cuda(), res=res.cuda(), out_dtype=torch.float32 if f32 else torch.bfloat16)
    _check(got, y, x.double().abs() @ wb.T, K, extra=2.0 ** -24 * y.abs())
    if not f32:
        r = res.cuda()
        assert linear.linear_decode(lw, x.cuda(), res=r, out=r) is r and torch.equal(r, got)


def test_rows_do_not_depend_on_each_other():
    """A row alone, among four, eight or sixteen (another kernel, another split of K): the same bits; twice: the same bits."""
    from dsgx10_b200 import linear
    for N, K in ((500, 6144), (2000, 1111), (16, 9000)):
        blocks, _, _ = _make(N, K, N)
        lw = linear.LinearW(N, K, blocks)
        x = _x(16, K, K).cuda()
        all16 = linear.linear_decode(lw, x, out_dtype=torch.float32)
        assert torch.equal(all16, linear.linear_decode(lw, x, out_dtype=torch.float32))
        for m in (1, 3, 4, 5, 8, 9, 13):
            assert torch.equal(linear.linear_decode(lw, x[16 - m:], out_dtype=torch.float32), all16[16 - m:]), (N, K, m)


def test_inf_and_nan_stay_in_their_row():
    from dsgx10_b200 import linear
    N, K = 200, 1030
    blocks, _, _ = _make(N, K, 41)
    lw = linear.LinearW(N, K, blocks)
    for M in (2, 7, 12):
        x = _x(M, K, 42).cuda()
        clean = linear.linear_decode(lw, x)
        bad = x.clone()
        bad[1, 5], bad[M - 1, K - 1] = float("nan"), float("inf")
        got = linear.linear_decode(lw, bad)
        keep = [r for r in range(M) if r not in (1, M - 1)]
        assert torch.equal(got[keep], clean[keep]) and bool(got[1].isnan().all()) and not bool(got[M - 1].isfinite().any())


def test_strided_and_unaligned_rows():
    """Rows of larger tensors, at addresses that are no multiples of 16 bytes: the bits of the packed call; nothing
    outside the rows is written."""
    from dsgx10_b200 import linear
    M, N, K = 6, 77, 1001
    blocks, _, _ = _make(N, K, 51)
    lw = linear.LinearW(N, K, blocks)
    x, res = _x(M, K, 52).cuda(), _x(M, N, 53).cuda()
    want = linear.linear_decode(lw, x, res=res)
    for off, pad in ((0, 7), (3, 12), (8, 8)):
        xs = torch.full((M, K + pad + off), float("nan"), dtype=torch.bfloat16, device="cuda")
        xs[:, off:off + K] = x
        rs = torch.full((M, N + pad + off), float("nan"), dtype=torch.bfloat16, device="cuda")
        rs[:, off:off + N] = res
        os_ = torch.full((M, N + pad + off), 7.0, dtype=torch.bfloat16, device="cuda")
        linear.linear_decode(lw, xs[:, off:off + K], res=rs[:, off:off + N], out=os_[:, off:off + N])
        assert torch.equal(os_[:, off:off + N], want)
        rest = torch.cat([os_[:, :off], os_[:, off + N:]], 1)
        assert bool((rest == 7.0).all())


def test_streams_and_graph():
    """Two streams at once, and a captured chain (gate/up, down with the residual in place) replayed on new inputs: the bits
    of the eager calls."""
    from dsgx10_b200 import linear
    H, I, M = 1024, 1536, 2
    gate, up, down = (_make(n, k, 60 + i)[0] for i, (n, k) in enumerate(((I, H), (I, H), (H, I))))
    gu, down = linear.LinearW(I, H, gate, up=up), linear.LinearW(H, I, down)

    def layer(x, out=None):
        return linear.linear_decode(down, linear.linear_decode(gu, x), res=x, out=out)

    xs = [_x(M, H, 70 + i).cuda() for i in range(6)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, x in enumerate(xs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(layer(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, out = xs[0].clone(), torch.empty_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, out=out)
    for i in (3, 1, 5):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_python_refusals():
    from dsgx10_b200 import linear
    N, K = 64, 700
    blocks, _, _ = _make(N, K, 81)
    lw = linear.LinearW(N, K, blocks)
    x = _x(2, K, 82).cuda()
    for bad in (x.float(), x[:, :-1], x.cpu(), x[0], _x(17, K, 1).cuda(), torch.empty(K, 2, dtype=torch.bfloat16, device="cuda").T,
                x[:0], x[:1].expand(2, K)):
        with pytest.raises(ValueError):
            linear.linear_decode(lw, bad)
    for kw in (dict(res=x), dict(out=x), dict(out=torch.empty(2, N, dtype=torch.float16, device="cuda"))):
        with pytest.raises(ValueError):
            linear.linear_decode(lw, x, **kw)
    for bad in (blocks[:-1], blocks.cpu(), blocks.view(torch.int16)):
        with pytest.raises(ValueError):
            linear.LinearW(N, K, bad)
    from dsgx10_b200 import _lib
    with pytest.raises(_lib.DsgxError):
        linear.linear_decode(linear.LinearW(N, K, blocks, up=blocks), x, res=torch.zeros(2, N, dtype=torch.bfloat16, device="cuda"))


FIRST_USE = """
import torch
from dsgx10_b200 import linear, moe, synth, _lib
cases = []
for M, N, K, up in ((1, 512, 1024, False), (3, 1000, 5000, False), (16, 256, 9000, False), (8, 512, 6144, True)):
    n = -(-N // 8) * -(-K // 512)
    b = torch.randint(0, 256, (n, 2368), dtype=torch.uint8, device="cuda")
    b[:, 2048:2304].view(n, 128, 2)[:, :, 1] = 0x3B
    cases.append((linear.LinearW(N, K, b.view(-1), up=b.view(-1) if up else None), torch.randn(M, K, device="cuda").bfloat16()))
shp = moe.shape(1024, 512, 16, 4, fmt=_lib.FMT_INT4)
layer, wr = synth.Int4Layer.on_device(1024, 512, 16, 5, "cuda"), synth.router_weights(16, 1024, 7).cuda()
block, lw, x = moe.MoeBlock(shp, wr), layer.layer_w(), synth.activations(5, 1024, 6).cuda()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [linear.linear_decode(w, x) for w, x in cases] + [block.run(lw, x)[0]]
graph.replay()
torch.cuda.synchronize()
want = [linear.linear_decode(w, x) for w, x in cases] + [block.run(lw, x)[0]]
assert all(torch.equal(a, b) for a, b in zip(got, want)) and moe.ws_status(block.ws) == 0
print("first use captured")
"""


def test_first_use_inside_a_capture():
    """A process whose first call of each form is captured (device attributes and residencies are asked for on the first call)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_USE], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "first use captured" in r.stdout, r.stdout + r.stderr


def test_prepare_then_product():
    """Weights used by the very next calls, again and again into the same memory: never the bytes that were there before."""
    from dsgx10_b200 import linear
    N, K = 4096, 2048
    x = _x(1, K, 90).cuda()
    made = [_make(N, K, 91 + i)[0] for i in range(2)]
    want = []
    for b in made:
        w = linear.LinearW(N, K, b)
        torch.cuda.synchronize()
        want.append(linear.linear_decode(w, x).clone())
    torch.cuda.synchronize()
    for i in range(40):
        w = linear.LinearW(N, K, made[i % 2])
        got = linear.linear_decode(w, x)
        del w
        assert torch.equal(got, want[i % 2]), i


@pytest.mark.parametrize("M,N,K", [(1, 10, 250000), (6, 40, 60000), (16, 17, 100001)])
def test_long_rows(M, N, K):
    """K over all of a cluster's shared memory, and past it: the rows then go in several launches."""
    from dsgx10_b200 import linear
    blocks, w, wb = _make(N, K, 301)
    x = _x(M, K, 302)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lw = linear.LinearW(N, K, blocks)
    got = linear.linear_decode(lw, x.cuda(), out_dtype=torch.float32, status=status)
    assert int(status) == 0
    _check(got, x.double() @ w.T, x.double().abs() @ wb.T, K)
    assert torch.equal(got[-1:], linear.linear_decode(lw, x[-1:].cuda(), out_dtype=torch.float32))


def test_too_long_rows_are_refused():
    from dsgx10_b200 import _lib, linear
    N, K = 8, 1000000
    w = linear.LinearW(N, K, torch.zeros(-(-K // 512) * 2368, dtype=torch.uint8, device="cuda"))
    for M in (1, 3, 16):
        with pytest.raises(_lib.DsgxError):
            linear.linear_decode(w, torch.zeros(M, K, dtype=torch.bfloat16, device="cuda"))


def test_offsets_past_32_bits():
    """More than 4 GiB of weights, the same 16 rows over and over: every 16 outputs are the bits of a matrix of 16 rows."""
    from dsgx10_b200 import linear
    N, K, M = 1 << 20, 8192, 2
    small, _, _ = _make(16, K, 311)
    x = _x(M, K, 312).cuda()
    want = linear.linear_decode(linear.LinearW(16, K, small), x, out_dtype=torch.float32)
    blocks = small.repeat(N // 16)
    w = linear.LinearW(N, K, blocks)
    assert w.data.numel() > 1 << 32
    del blocks
    got = linear.linear_decode(w, x, out_dtype=torch.float32)
    assert torch.equal(got.view(M, N // 16, 16), want.view(M, 1, 16).expand(M, N // 16, 16))
