"""The dense INT4 products without a GPU: the packing of any size, and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

from dsgx10_b200 import _lib, weights
from tests.linear_util import random_int4, unpack


@pytest.mark.parametrize("N,K", [(1, 1), (8, 512), (9, 513), (17, 31), (40, 1000), (3, 32)])
@pytest.mark.parametrize("zeros", [False, True])
def test_pack_linear_int4_keeps_every_weight(N, K, zeros):
    wp, s, zp, w, _ = random_int4(N, K, 7 * N + K, zeros)
    blocks = weights.pack_linear_int4(wp, s, zp, K=K)
    assert blocks.size == -(-N // 8) * -(-K // 512) * 2368
    full = unpack(blocks, -(-N // 8) * 8, -(-K // 512) * 512)
    assert (full[:N, :K] == w).all()
    kg = -(-K // 32) * 32   # (what shares a group with a real weight has its scale; behind that the scales are 0)
    assert (full[N:] == 0).all() and (full[:, kg:] == 0).all()


def test_pack_linear_int4_refuses_what_does_not_fit():
    wp, s, zp, _, _ = random_int4(9, 100, 1, True)
    for bad in ((wp[:, :-1], s, zp), (wp, s[:, :-1], zp), (wp, s[:-1], zp), (wp, s, zp[:-1])):
        with pytest.raises(ValueError):
            weights.pack_linear_int4(*bad, K=100)


def test_refused_calls():
    """Every refusal comes before anything is launched, so it shows without a GPU."""
    L = _lib.lib()
    one = 1 << 20   # (an aligned address that nothing reads)

    def call(w=one, N=64, K=512, fmt=_lib.FMT_INT4, glu=0, x=one, ldx=512, M=1, res=None, ldr=64, out=one, ldo=64, f32=0, status=None):
        W = _lib.LinearW(w, N, K, fmt, glu)
        return L.dsgx_linear_decode(C.byref(W), x, ldx, M, res, ldr, out, ldo, f32, status, None)

    assert L.dsgx_linear_decode(None, one, 512, 1, None, 0, one, 64, 0, None, None) == _lib.ERR_ARG
    for kw in (dict(w=None), dict(x=None), dict(out=None), dict(M=0), dict(M=17), dict(ldx=511), dict(ldo=63), dict(res=one, ldr=63),
               dict(w=one + 8), dict(x=one + 1), dict(out=one + 1), dict(out=one + 2, f32=1), dict(res=one + 1), dict(status=one + 2)):
        assert call(**kw) == _lib.ERR_ARG, kw
    for fmt in (_lib.FMT_NVFP4, _lib.FMT_RETIRED, _lib.FMT_BF16, _lib.FMT_FP8, _lib.FMT_MXFP4, 77):
        assert call(fmt=fmt) == _lib.ERR_FORMAT
        assert L.dsgx_linear_prepare(one, None, fmt, 64, 512, one, None) == _lib.ERR_FORMAT
    for N, K in ((0, 512), (64, 0), (-5, 512), (64, (1 << 30) + 1), (1 << 29, 1 << 20)):
        assert call(N=N, K=K, ldx=1 << 31, ldo=1 << 31) == _lib.ERR_SHAPE, (N, K)
        assert L.dsgx_linear_bytes(N, K, 0) == 0 and L.dsgx_linear_prepare(one, None, _lib.FMT_INT4, N, K, one, None) == _lib.ERR_SHAPE
    assert call(glu=1, res=one) == _lib.ERR_UNSUPPORTED
    for a in ((None, None, one), (one, None, None), (one + 8, None, one), (one, one + 4, one), (one, None, one + 2)):
        assert L.dsgx_linear_prepare(a[0], a[1], _lib.FMT_INT4, 64, 512, a[2], None) == _lib.ERR_ARG
    assert L.dsgx_linear_bytes(17, 513, 0) == 2 * 2 * 4736 and L.dsgx_linear_bytes(17, 513, 1) == 3 * 2 * 4736


def test_refused_block_calls():
    """A whole layer in one launch: what is refused before anything is launched."""
    from dsgx10_b200 import moe
    L = _lib.lib()
    one = 1 << 20

    def call(M=1, x=one, out=one, res=None, lw=None, blk=None, **kw):
        shp = moe.shape(**{**dict(H=1024, I=512, E=16, topk=4, fmt=_lib.FMT_INT4), **kw})
        W = _lib.LayerW(pool=one, desc=one, fmt=shp.fmt)
        for k, v in (lw or {}).items():
            setattr(W if k in ("pool", "desc", "fmt") else W.sh, k, v)
        B = _lib.MoeBlock(one, None, one, one, one, None)
        for k, v in (blk or {}).items():
            setattr(B, k, v)
        return L.dsgx_moe_block_decode(C.byref(shp), C.byref(W), x, M, C.byref(B), res, out, None)

    for kw in (dict(M=0), dict(M=17), dict(x=None), dict(out=None), dict(x=one + 8), dict(out=one + 4), dict(res=one + 2), dict(lw=dict(pool=None)),
               dict(lw=dict(pool=one + 128)), dict(lw=dict(bg=one)), dict(lw=dict(bd=one)), dict(lw=dict(bgu=one, bu=one, bd=one)),
               dict(blk=dict(wr=None)), dict(blk=dict(ws=None)), dict(blk=dict(ws=one + 64)), dict(blk=dict(idx=None)), dict(blk=dict(w=None))):
        assert call(**kw) == _lib.ERR_ARG, kw
    for kw in (dict(fmt=_lib.FMT_FP8), dict(fmt=_lib.FMT_MXFP4), dict(fmt=_lib.FMT_NVFP4), dict(lw=dict(fmt=_lib.FMT_BF16)), dict(lw=dict(g=one))):
        assert call(**kw) == _lib.ERR_FORMAT, kw
    for kw in (dict(H=1000), dict(I=768), dict(topk=9), dict(E=513), dict(topk=5, E=4), dict(swiglu_limit=10.0), dict(H=1 << 20)):
        assert call(**kw) == _lib.ERR_SHAPE, kw
    for kw in (dict(e_lo=1), dict(e_hi=15)):
        assert call(**kw) == _lib.ERR_UNSUPPORTED, kw
    shp = moe.shape(1024, 512, 16, 4, fmt=_lib.FMT_FP8)
    assert L.dsgx_moe_block_ws_bytes(C.byref(shp)) == 0
    assert L.dsgx_moe_block_ws_bytes(C.byref(moe.shape(6144, 2048, 168, 8, fmt=_lib.FMT_INT4))) > 0


def test_product_in_place_is_refused():
    """The outputs of one CTA would be another's inputs: out = x is refused, out = res is not looked at."""
    L, x = _lib.lib(), 1 << 20
    W = _lib.LinearW(x, 512, 512, _lib.FMT_INT4, 0)
    assert L.dsgx_linear_decode(C.byref(W), x, 512, 1, None, 0, x, 512, 0, None, None) == _lib.ERR_ARG
