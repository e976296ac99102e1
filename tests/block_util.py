"""The layer of dsgx_moe_block_decode in 64 bits, stage by stage, on whatever device its layer is, and the two checks of a result.

`check_rows` bounds a row's error in the mean: the output's one rounding to bf16 and h's rounding to eleven bits are all that
a value may lose beside the last bits of f32 sums.  `check_stages` looks at every element of the kernel's own h and y (held in
its workspace) and at the sum made of them, so that a wrong unit of eight channels or of 512 k shows where it is."""
import numpy as np
import torch


def int4_matrix(blocks, N, K):
    """(W, (u + z) s) f64 [N][K] of INT4 blocks of 8 rows x 512 k (uint8), from the layout's address rule."""
    b, dev = blocks.reshape(-1), blocks.device
    n, k = torch.arange(N, device=dev)[:, None], torch.arange(K, device=dev)[None, :]
    r, g = k % 512, n % 8
    base = (n // 8 * (K // 512) + k // 512) * 2368
    jj, q, t, i = r // 128, r // 64 % 2, r // 16 % 4, r % 16
    u = (b[base + 512 * jj + 16 * (4 * g + t) + 8 * q + i // 2] >> (4 * (i % 2)) & 15).double()
    s = blocks.reshape(-1).view(torch.bfloat16)[(base + 2048 + 32 * g + 16 * (t // 2)) // 2 + 2 * jj + q].double()
    z = (b[base + 2304 + 8 * g + 4 * (t // 2) + jj] >> (4 * q) & 15).double()
    return (u - z) * s, (u + z) * s


def bf16_matrix(blocks, N, K):
    """(W, |W|) f64 [N][K] of bf16 blocks of 8 rows x 128 k: a lane's 16 bytes at 512 p + 16 (4 g + t)."""
    n, k = torch.arange(N, device=blocks.device)[:, None], torch.arange(K, device=blocks.device)[None, :]
    r, g = k % 128, n % 8
    p, t = 2 * (r // 64) + r // 8 % 2, r // 16 % 4
    w = blocks.reshape(-1).view(torch.bfloat16)[(n // 8 * (K // 128) + k // 128) * 1024 + 256 * p + 8 * (4 * g + t) + r % 8].double()
    return w, w.abs()


def mats(layer, e):
    """[(W, bound)] of expert e (None: the shared one): gate, up, down."""
    out = []
    for m, (N, K) in enumerate(((layer.I, layer.H), (layer.I, layer.H), (layer.H, layer.I))):
        if e is None:
            out.append(bf16_matrix(layer.sh_dev[m].reshape(-1).view(torch.uint8), N, K))
            continue
        off, size = layer.desc_host[e * 3 + m].off, N * K * 2 if layer.fmt == 3 else N // 8 * (K // 512) * 2368
        out.append((bf16_matrix if layer.fmt == 3 else int4_matrix)(layer.pool[off:off + size].clone(), N, K))
    return out


def gamma(K, b16):
    """Of a sum's bound.  INT4: the dense products' (80 + blocks).  bf16: a block's 64 MMAs at most (h: two for one) in one
    accumulator, 17 truncations each, then the blocks and tasks."""
    return ((64 * 17 + 8 if b16 else 80) + K // 512) * 2.0 ** -23


def small(x, bound):
    """What x loses as an f16 operand of INT4 products: values far below their 512-block's largest round by at most 2^-35 of it."""
    M, K = x.shape
    top = x.abs().reshape(M, -1, 512).amax(-1, keepdim=True).expand(M, K // 512, 512).reshape(M, K)
    return 2.0 ** -35 * (top @ bound.T)


def hidden(x, gate, up, b16):
    """h = silu(g) u and its bound: sums in f32, silu's slope below 1.1, the fast exponential and division within 2^-16 for |g| up to
    80; below -80 silu is less than 80 e^-80 < 2^-108, of which nothing need be left."""
    g, u = x @ gate[0].T, x @ up[0].T
    dg, du = (gamma(x.shape[1], b16) * (x.abs() @ m[1].T) + (0 if b16 else small(x, m[1])) for m in (gate, up))
    act = g * torch.sigmoid(g)
    return act * u, 1.1 * dg * (u.abs() + du) + act.abs() * du + (act * u).abs() * 2.0 ** -16 + 2.0 ** -108 * (u.abs() + du)


def as_operand(h, nib):
    """h as the down product's f16 operand: times the power of two that brings a 512-block's largest into [2^14, 2^15) (odd k of a
    nibble matrix 2^-4 of that), rounded once."""
    b = h.double().reshape(h.shape[0], -1, 512)
    top = b.abs().amax(-1, keepdim=True)
    E = torch.where(top >= 2.0 ** -126, (14 - torch.floor(torch.log2(top.clamp_min(2.0 ** -126)))).clamp_max(126), torch.full_like(top, 126.0))
    f = torch.exp2(E) * torch.ones(512, dtype=torch.float64, device=h.device)
    if nib:
        f[..., 1::2] *= 2.0 ** -4
    return ((b * f).to(torch.float32).to(torch.float16).double() / f).reshape(h.shape)


def reference(layer, x, idx, w, res=None, shared=True, edit=None):
    """out f64 [M][H] and the squares of what is added (picks times weight, shared expert).  edit(e, rows, h): another h (a mistake
    planted by a test of the checks)."""
    x, w = x.double(), w.double()
    out, parts = torch.zeros_like(x), torch.zeros_like(x)
    experts = torch.unique(idx).tolist() + ([None] if shared else [])
    for e in experts:
        gate, up, down = mats(layer, e)
        m, k = (idx == e).nonzero(as_tuple=True) if e is not None else (torch.arange(x.shape[0], device=x.device), None)
        h, _ = hidden(x[m], gate, up, False)
        if edit is not None:
            h = edit(e, m, h)
        y = (h @ down[0].T) * (w[m, k, None] if e is not None else 1.0)
        out[m] += y
        parts[m] += y * y
    return (out if res is None else out + res.double()), parts


def check_rows(got, out, parts):
    """The largest of the rows' squared errors over its limit (must be at most 1).  The limit: what rounding `out` to bf16 costs, and
    2^-11 of every part (h's rounding; its errors fall either way and add up like the products themselves).  A squared rounding
    error scatters by 0.9 of its mean, the mean over H of them by 0.9 / sqrt(H), the ratio of two such by 1.27 / sqrt(H): five of
    these are allowed."""
    err = (got.double() - out).pow(2).sum(1)
    rounding = (out.to(torch.float32).to(torch.bfloat16).double() - out).pow(2).sum(1)
    return float((err / (rounding * (1 + 6.4 / out.shape[1] ** 0.5) + 2.0 ** -22 * parts.sum(1) + 1e-60)).max())


def stages(block, H, I):
    """The kernel's h f32 [64 + 1][8][I] and y f32 [64 + 1][8][H], the last two regions of its workspace."""
    al = lambda v: -(-v // 256) * 256
    hb, yb = 65 * 8 * I * 4, 65 * 8 * H * 4
    end = block.ws.numel() - al(yb)
    return (block.ws[end - al(hb):end - al(hb) + hb].view(torch.float32).view(65, 8, I), block.ws[end:end + yb].view(torch.float32).view(65, 8, H))


def check_stages(layer, x, idx, w, h, y, got, res=None, shared=True):
    """Every element of h against x, of y against h, of got against y.  Slots are the picked experts in ascending id, a slot's rows the
    rows that picked it, in order; slot 64 is the shared expert."""
    x, w, b16 = x.double(), w.double(), layer.fmt == 3
    out, size = torch.zeros_like(x), torch.zeros_like(x)
    for slot, e in enumerate(torch.unique(idx).tolist() + ([None] if shared else [])):
        bf = b16 or e is None
        gate, up, down = mats(layer, e)
        m, k = (idx == e).nonzero(as_tuple=True) if e is not None else (torch.arange(x.shape[0], device=x.device), None)
        s, n = (64 if e is None else slot), len(m)
        want, tol = hidden(x[m], gate, up, bf)
        hk, yk = h[s, :n], y[s, :n].double()
        bad = (hk.double() - want).abs() > tol + 1e-37
        assert not bool(bad.any()), f"h of expert {e}: {bad.nonzero()[:4].tolist()}"
        op = as_operand(hk, not bf)
        bad = (yk - op @ down[0].T).abs() > gamma(layer.I, bf) * (op.abs() @ down[1].T) + 1e-37
        assert not bool(bad.any()), f"y of expert {e}: {bad.nonzero()[:4].tolist()}"
        c = yk * (w[m, k, None] if e is not None else 1.0)
        out[m] += c
        size[m] += c.abs()
    if res is not None:
        out, size = out + res.double(), size + res.double().abs()
    bad = (got.double() - out).abs() > 2.0 ** -8 * out.abs() + 2.0 ** -20 * size
    assert not bool(bad.any()), f"sum: {bad.nonzero()[:4].tolist()}"
