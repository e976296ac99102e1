"""INT4-g32 matrices for the tests of the dense products: random ones in the checkpoints' form, and a reader of the blocks
written from the layout's address rule, weight by weight (not from the packer)."""
import numpy as np


def random_int4(N, K, seed, zeros=True):
    """wp uint8 [N][ceil(K/2)], s bf16 bits [N][ceil(K/32)], zp uint32 [ceil(N/8)][ceil(K/32)] or None, W f64 [N][K], and its bound
    (u + z) s (what a sum of u x and one of z x are made of)."""
    rng = np.random.default_rng(seed)
    G = -(-K // 32)
    u = rng.integers(0, 16, (N, K + K % 2), dtype=np.uint8)
    wp = u[:, 0::2] | (u[:, 1::2] << 4)
    s = (0x3B00 + rng.integers(0, 256, (N, G))).astype(np.uint16)
    z = rng.integers(0, 16, (-(-N // 8) * 8, G)).astype(np.uint32) if zeros else np.full((-(-N // 8) * 8, G), 8, np.uint32)
    zp = (z.reshape(-1, 8, G) << (4 * np.arange(8, dtype=np.uint32))[None, :, None]).sum(1).astype(np.uint32)
    sf = (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    k = np.arange(K)
    uf, zf = u[:, :K].astype(np.float64), z[:N][:, k // 32].astype(np.float64)
    return wp, s, zp if zeros else None, (uf - zf) * sf[:, k // 32], (uf + zf) * sf[:, k // 32]


def unpack(blocks, N, K, bound=False):
    """W f64 [N][K] of blocks [N/8][K/512][2368], and (u + z) s with `bound`."""
    b = np.ascontiguousarray(blocks, np.uint8).reshape(-1)
    n, k = np.arange(N)[:, None], np.arange(K)[None, :]
    base = (n // 8 * (K // 512) + k // 512) * 2368
    r, g = k % 512, n % 8
    jj, q, t, i = r // 128, r // 64 % 2, r // 16 % 4, r % 16
    u = b[base + 512 * jj + 16 * (4 * g + t) + 8 * q + i // 2] >> (4 * (i % 2)) & 15
    at = base + 2048 + 32 * g + 16 * (t // 2) + 2 * (2 * jj + q)
    s = ((b[at].astype(np.uint32) | b[at + 1].astype(np.uint32) << 8) << 16).view(np.float32).astype(np.float64)
    z = b[base + 2304 + 8 * g + 4 * (t // 2) + jj] >> (4 * q) & 15
    w = (u.astype(np.float64) - z) * s
    return (w, (u.astype(np.float64) + z) * s) if bound else w
