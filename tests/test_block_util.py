"""The checks of the whole-layer call see mistakes (on the CPU, planted in the 64-bit layer, never in a kernel)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def case():
    from dsgx10_b200 import synth
    from tests import block_util as U
    layer = synth.Int4Layer(1024, 1024, 12, 77)
    z = layer.pool.view(-1, 2368)[:, 2304:]
    z.copy_(torch.randint(0, 256, z.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(3)))
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 1024, generator=g).to(torch.bfloat16)
    idx = torch.stack([torch.randperm(12, generator=g)[:6] for _ in range(3)])
    w = torch.rand(3, 6, generator=g) * 0.2 + 0.1
    return layer, x, idx, w, *U.reference(layer, x, idx, w)


def _got(case, edit):
    from tests import block_util as U
    layer, x, idx, w = case[:4]
    return U.reference(layer, x, idx, w, edit=edit)[0].to(torch.float32).to(torch.bfloat16)


def _bits(h, n):
    """n significant bits, to nearest."""
    s = torch.exp2(n - 1 - torch.floor(torch.log2(h.abs().clamp_min(1e-300))))
    return torch.round(h * s) / s


def test_the_matrices_are_the_packed_ones(case):
    from dsgx10_b200 import synth
    from tests import block_util as U
    from tests.linear_util import unpack
    layer = case[0]
    N, K = layer.I, layer.H
    w, b = unpack(layer.pool[:N // 8 * (K // 512) * 2368].numpy(), N, K, bound=True)
    got = U.mats(layer, 0)[0]
    assert (got[0].numpy() == w).all() and (got[1].numpy() == b).all()
    sh = torch.from_numpy((layer.sh_bits[2].astype(np.uint32) << 16).view(np.float32)).double()
    assert torch.equal(U.mats(layer, None)[2][0], sh)


def test_the_contract_passes(case):
    from tests import block_util as U
    assert U.check_rows(_got(case, lambda e, m, h: U.as_operand(h.to(torch.float32), e is not None)), *case[4:]) <= 1
    assert U.check_rows(_got(case, None), *case[4:]) <= 1


def _drop(lo, hi, which, mul=0.0):
    def edit(e, m, h):
        if e in which:
            h = h.clone()
            h[:, lo:hi] *= mul
        return h
    return edit


@pytest.mark.parametrize("what", ["h in bf16", "h in five bits", "a unit of a pick", "a unit of the shared expert", "512 k of a pick", "a pick 4 % off"])
def test_a_mistake_does_not_pass(case, what):
    from tests import block_util as U
    e = int(case[2][1, 2])
    edit = {"h in bf16": lambda e, m, h: _bits(h, 8), "h in five bits": lambda e, m, h: _bits(h, 5),
            "a unit of a pick": _drop(512, 520, [e]), "a unit of the shared expert": _drop(1016, 1024, [None]),
            "512 k of a pick": _drop(512, 1024, [e]), "a pick 4 % off": _drop(0, 1024, [e], 1.04)}[what]
    assert U.check_rows(_got(case, edit), *case[4:]) > 1


@pytest.mark.parametrize("what", ["h", "y", "sum"])
def test_a_wrong_stage_is_found(case, what):
    from tests import block_util as U
    layer, x, idx, w = case[:4]
    h, y = torch.zeros(65, 8, layer.I), torch.zeros(65, 8, layer.H)
    out = torch.zeros(3, layer.H, dtype=torch.float64)
    for slot, e in enumerate(torch.unique(idx).tolist() + [None]):
        m = (idx == e).nonzero()[:, 0] if e is not None else torch.arange(3)
        gate, up, down = U.mats(layer, e)
        s = 64 if e is None else slot
        h[s, :len(m)] = U.hidden(x.double()[m], gate, up, False)[0].float()
        y[s, :len(m)] = (U.as_operand(h[s, :len(m)], e is not None) @ down[0].T).float()
        out[m] += y[s, :len(m)].double() * (w[idx == e].double()[:, None] if e is not None else 1.0)
    got = out.float().to(torch.bfloat16)
    U.check_stages(layer, x, idx, w, h, y, got)
    if what == "h":
        h[1, 0, 1023] *= 1.1
    elif what == "y":
        y[2, 0, 7] += 0.1 * y[2, 0].abs().mean()
    else:
        got[1, 5] *= 1.02
    with pytest.raises(AssertionError):
        U.check_stages(layer, x, idx, w, h, y, got)
