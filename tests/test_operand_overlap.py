"""Outputs that would be written over inputs still to be read: refused before anything is launched, so without a GPU."""
import ctypes as C

import pytest

from dsgx10_b200 import _lib


@pytest.mark.parametrize("kw", [
    dict(f32=1, out=0x400000, res=0x400000),                       # four bytes over two that others have not read
    dict(ldo=80, out=0x400000, res=0x400000),                      # other rows than the residual's
    dict(out=0x400000, res=0x400002),                              # one element on
    dict(out=0x400000 + 128, res=0x400000),                        # the next row's place
    dict(out=0x200000 + 2), dict(out=0x200000 + 512 * 2 * 2),   # inside x, x's last row
    dict(out=0x200000 - 64 * 4, f32=1),                            # f32 rows that reach x where bf16 ones would not
    dict(out=0x200000 + 512 * 2 - 2, ldx=576, ldo=576),            # columns of one tensor that overlap by one element
])
def test_products(kw):
    a = dict(x=0x200000, ldx=512, M=3, res=None, ldr=64, out=0x400000, ldo=64, f32=0)
    a.update(kw)
    W = _lib.LinearW(0x600000, 64, 512, _lib.FMT_INT4, 0)
    rc = _lib.lib().dsgx_linear_decode(C.byref(W), a["x"], a["ldx"], a["M"], a["res"], a["ldr"], a["out"], a["ldo"], a["f32"], None, None)
    assert rc == _lib.ERR_ARG


def test_layer():
    from dsgx10_b200 import moe
    shp, one = moe.shape(H=1024, I=512, E=16, topk=4, fmt=_lib.FMT_INT4), 1 << 20
    W, B = _lib.LayerW(pool=one, desc=one, fmt=shp.fmt), _lib.MoeBlock(one, None, one, one, one, None)
    for x, res, out in ((one, None, one + 16), (one + 32, None, one), (one, 4 * one, 4 * one + 2048), (4 * one, one, one + 3 * 2048 - 16),
                        (one, one + 2048, one), (one + 2048, one, one)):
        assert _lib.lib().dsgx_moe_block_decode(C.byref(shp), C.byref(W), x, 3, C.byref(B), res, out, None) == _lib.ERR_ARG, (x, res, out)


def test_prepare_is_not_in_place():
    L, w = _lib.lib(), 1 << 24
    size, src = L.dsgx_linear_bytes(64, 1024, 0), 8 * 2 * 2368
    pair = L.dsgx_linear_bytes(64, 1024, 1)
    for a in ((w, None, w), (w, None, w + src - 16), (w, None, w - size + 16), (w, 2 * w, 2 * w), (2 * w, w, w - pair + 16)):
        assert L.dsgx_linear_prepare(a[0], a[1], _lib.FMT_INT4, 64, 1024, a[2], None) == _lib.ERR_ARG, a


@pytest.mark.gpu
def test_columns_of_one_tensor_and_in_place():
    """x, res and out as columns of one tensor, and a residual in place with a leading dimension of its own: the packed call's bits."""
    torch = pytest.importorskip("torch")
    from dsgx10_b200 import linear, weights
    from tests.linear_util import random_int4
    N, K, M = 72, 520, 7
    wp, s, zp, _, _ = random_int4(N, K, 5)
    w = linear.LinearW(N, K, torch.from_numpy(weights.pack_linear_int4(wp, s, zp)).cuda())
    x, r = (torch.randn(M, n, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).cuda() for n in (K, N))
    want = linear.linear_decode(w, x, res=r)
    t = torch.zeros(M, K + 2 * N, dtype=torch.bfloat16, device="cuda")
    t[:, N:N + K], t[:, N + K:] = x, r
    linear.linear_decode(w, t[:, N:N + K], res=t[:, N + K:], out=t[:, :N])
    assert torch.equal(t[:, :N], want) and torch.equal(t[:, N + K:], r) and torch.equal(t[:, N:N + K], x)
    linear.linear_decode(w, t[:, N:N + K], res=t[:, N + K:], out=t[:, N + K:])
    assert torch.equal(t[:, N + K:], want) and torch.equal(t[:, N:N + K], x)
    f = torch.zeros(M, N, dtype=torch.float32, device="cuda")
    with pytest.raises(Exception):
        linear.linear_decode(w, x, res=f.view(torch.bfloat16)[:, :N], out=f)
