"""Two 4-bit operators of the decode path, each in its plain form and as the library's calls.

linear  `linear.linear_decode`: y = x W^T for 1..16 rows over INT4-g32 weights, W[n][k] = (u[n][k] - z[n][k / 32]) s[n][k / 32]
        (u, z nibbles, s bf16), with the residual added (`res`) or, for two matrices, silu(x Wg^T) * (x Wu^T) (`swiglu`).
block   `moe.MoeBlock`: the whole MoE layer of an INT4-g32 model for 1..16 rows in one launch: router logits, selection, the
        picked experts' SwiGLU FFNs, the bf16 shared expert, the weighted sum, the residual.

The weights are held as a user's program holds them: the library's blocks of 8 rows x 512 k (2368 bytes) and, for the shared
expert, of 8 rows x 128 k in bf16 (2048 bytes).  `own` False computes with elementary torch operations, in 32 bits (the
router in 64: a selection must not hang on the last bits of a sum), rounded once at the end.
"""
import math

import torch

own = False

G = 32                      # weights a scale
BLK_K, BLK_BYTES = 512, 2368


def _up(v, m):
    return -(-v // m) * m


# ------------------------------------------------------------------------------------------------------------- cases

def listed():
    lin = dict(op="linear", res=False, swiglu=False, f32=False)
    blk = dict(op="block", score="softmax", groups=1, keep=1, shared=True, res=True, scale=1.0, bias=False)
    return [
        # a small projection of one token: launch and memory latency
        {**lin, "name": "linear 1 x 512 x 1024", "M": 1, "N": 512, "K": 1024},
        # the down matrix of one expert's size, residual added, a few tokens of speculative verification
        {**lin, "name": "linear 4 x 6144 x 2048 res", "M": 4, "N": 6144, "K": 2048, "res": True},
        # odd sizes: a ragged last strip of rows and a partial last group along K
        {**lin, "name": "linear 3 x 4099 x 5000", "M": 3, "N": 4099, "K": 5000},
        # a dense layer's gate and up matrices with their SwiGLU, one token
        {**lin, "name": "linear swiglu 1 x 12288 x 6144", "M": 1, "N": 12288, "K": 6144, "swiglu": True},
        # a long K and sixteen rows: the widest step
        {**lin, "name": "linear 16 x 6144 x 12288", "M": 16, "N": 6144, "K": 12288},
        # an output head: many rows, f32 logits of eight positions
        {**lin, "name": "linear 8 x 131072 x 4096 f32", "M": 8, "N": 131072, "K": 4096, "f32": True},
        # a small layer, one token: the chain of dependent steps counts
        {**blk, "name": "block 1: 1024 x 512, 16 experts", "M": 1, "H": 1024, "I": 512, "E": 16, "topk": 4, "score": "sigmoid"},
        # hidden 6144, 168 experts of 2048, top-8 softmax, shared expert: one and four tokens
        {**blk, "name": "block 1: 6144 x 2048, 168 experts", "M": 1, "H": 6144, "I": 2048, "E": 168, "topk": 8},
        {**blk, "name": "block 4: 6144 x 2048, 168 experts", "M": 4, "H": 6144, "I": 2048, "E": 168, "topk": 8},
        # hidden 4096, 256 experts of 2048, top-8 in groups, no shared expert: a full verification step
        {**blk, "name": "block 8: 4096 x 2048, 256 experts", "M": 8, "H": 4096, "I": 2048, "E": 256, "topk": 8, "score": "sigmoid",
         "groups": 8, "keep": 4, "shared": False, "scale": 2.5, "bias": True},
        # hidden 2048, 64 experts of 1024, top-6: sixteen rows
        {**blk, "name": "block 16: 2048 x 1024, 64 experts", "M": 16, "H": 2048, "I": 1024, "E": 64, "topk": 6, "score": "sqrtsoftplus"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    M = _log(rng, 1, 16)
    if rng.random() < 0.5:
        K = min(_log(rng, 40, 16384) | (rng.random() < 0.4), 16384)   # odd lengths among them
        N = _log(rng, 30, min(131072, 480_000_000 // K))
        swiglu = rng.random() < 0.3
        return dict(op="linear", M=M, N=max(1, N // 2) if swiglu else N, K=K, res=not swiglu and rng.random() < 0.4, swiglu=swiglu,
                    f32=rng.random() < 0.3)
    E = rng.choice([4, 7, 16, 32, 60, 64, 128, 168, 256, 384])
    groups = rng.choice([1, 4, 8]) if E % 8 == 0 and E >= 16 else 1
    keep = rng.randint((groups + 1) // 2, groups)
    topk = min(rng.randint(1, 8), E, keep * (E // groups))
    H = 512 * min(_log(rng, 1, 14), 12)
    I = 512 * min(_log(rng, 1, 5), 4)
    while E * H * I > 2_200_000_000:
        E, groups, keep = E // 2, 1, 1
        topk = min(topk, E)
    c = dict(op="block", M=M, H=H, I=I, E=E, topk=topk, score=rng.choice(["sigmoid", "softmax", "sqrtsoftplus"]), groups=groups,
             keep=keep, shared=rng.random() < 0.6, res=rng.random() < 0.5, scale=rng.choice([1.0, 1.5, 2.5]), bias=rng.random() < 0.3)
    while work(c)["bytes"] > 800_000_000:
        c["M"] //= 2
    return c


# ------------------------------------------------------------------------------------------------------------ inputs

def _int4_blocks(n, g):
    """n random blocks: uniform nibbles, bf16 scales in [2^-9, 2^-7), zero points around the middle of the range."""
    b = torch.empty(n, BLK_BYTES, dtype=torch.uint8, device="cuda")
    b[:, :2048] = torch.randint(0, 256, (n, 2048), generator=g, device="cuda", dtype=torch.uint8)
    sc = b[:, 2048:2304].view(n, 128, 2)
    sc[:, :, 0] = torch.randint(0, 256, (n, 128), generator=g, device="cuda", dtype=torch.uint8)
    sc[:, :, 1] = 0x3B
    z = torch.randint(6, 11, (n, 64, 2), generator=g, device="cuda", dtype=torch.uint8)
    b[:, 2304:] = z[:, :, 0] | (z[:, :, 1] << 4)
    return b


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    c, st = case, {}
    if c["op"] == "linear":
        n = _up(c["N"], 8) // 8 * (_up(c["K"], BLK_K) // BLK_K)
        st["w"] = _int4_blocks(n, g)
        if c["swiglu"]:
            st["w_up"] = _int4_blocks(n, g)
        st["x"] = randn(c["M"], c["K"]).to(torch.bfloat16)
        if c["res"]:
            st["res"] = randn(c["M"], c["N"]).to(torch.bfloat16)
        return st
    H, I, E, M = c["H"], c["I"], c["E"], c["M"]
    per = I * H // 4096                              # blocks a matrix
    st["pool"] = _int4_blocks(E * 3 * per, g)        # [E][gate, up, down]
    if c["shared"]:
        st["shared"] = [(randn(I * H) * 0.02).to(torch.bfloat16) for _ in range(3)]
    st["wr"] = randn(E, H) * 0.02
    if c["bias"]:
        st["bias"] = randn(E) * 0.1
    st["x"] = randn(M, H).to(torch.bfloat16)
    if c["res"]:
        st["res"] = randn(M, H).to(torch.bfloat16)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = dict(case)
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a user's program keeps of the library: the weights' handle and, for the layer, its workspace."""
    from dsgx10_b200 import _lib, linear, moe
    c = st["case"]
    if c["op"] == "linear":
        st["handle"] = linear.LinearW(c["N"], c["K"], st["w"], up=st.get("w_up"))
        return
    H, I, E = c["H"], c["I"], c["E"]
    score = {"sigmoid": _lib.SCORE_SIGMOID, "softmax": _lib.SCORE_SOFTMAX, "sqrtsoftplus": _lib.SCORE_SQRTSOFTPLUS}[c["score"]]
    shp = moe.shape(H, I, E, c["topk"], fmt=_lib.FMT_INT4, n_group=c["groups"], topk_group=c["keep"], score_fn=score,
                    route_scale=c["scale"])
    mat = I * H // 4096 * BLK_BYTES
    desc = (_lib.MatDesc * (E * 3))()
    for i in range(E * 3):
        desc[i].off, desc[i].s2, desc[i].fmt = i * mat, 1.0, _lib.FMT_INT4
    st["desc"] = torch.frombuffer(bytearray(bytes(desc)), dtype=torch.uint8).cuda()
    L = _lib.LayerW()
    L.pool, L.desc, L.fmt = st["pool"].data_ptr(), st["desc"].data_ptr(), _lib.FMT_INT4
    if c["shared"]:
        L.sh.bg, L.sh.bu, L.sh.bd = (t.data_ptr() for t in st["shared"])
    st["layer_w"] = L
    st["handle"] = moe.MoeBlock(shp, st["wr"], st.get("bias"))


# ------------------------------------------------------------------------------------------------------- the two forms

def _int4(b, N8, B):
    """Blocks [..., N8 * B * 2368 bytes] -> W f32 [..., 8 N8][512 B]: unit jj, row g, lane t, half q, byte of a lane's 16."""
    b = b.reshape(-1, N8, B, BLK_BYTES)
    L = b.shape[0]
    v = b[..., :2048].reshape(L, N8, B, 4, 8, 4, 2, 8)
    v = torch.stack((v & 15, v >> 4), -1).permute(0, 1, 4, 2, 3, 6, 5, 7, 8).reshape(L, N8 * 8, B * 16, G)
    s = b[..., 2048:2304].contiguous().view(torch.bfloat16).reshape(L, N8, B, 8, 2, 8)
    s = s.permute(0, 1, 3, 2, 5, 4).reshape(L, N8 * 8, B * 16, 1)
    z = b[..., 2304:].reshape(L, N8, B, 8, 2, 4)
    z = torch.stack((z & 15, z >> 4), -1).permute(0, 1, 3, 2, 5, 6, 4).reshape(L, N8 * 8, B * 16, 1)
    return ((v.float() - z.float()) * s.float()).reshape(L, N8 * 8, B * BLK_K)


def _bf16(t, N, K):
    """The shared expert's blocks of 8 rows x 128 k -> W f32 [N][K]."""
    return t.reshape(N // 8, K // 128, 2, 2, 8, 4, 8).permute(0, 4, 1, 2, 5, 3, 6).reshape(N, K).float()


def _silu(v):
    return v / (1 + torch.exp(-v))


def _scores(kind, logits):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    if kind == "softmax":
        e = torch.exp(logits - logits.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)
    return torch.sqrt(torch.log(1 + torch.exp(logits)))


def _route(c, st):
    """idx [M][topk] in descending key order, ties to the lower expert; w [M][topk]."""
    s = _scores(c["score"], st["x"].double() @ st["wr"].double().T)
    key = s + st["bias"].double() if c["bias"] else s
    if c["groups"] > 1:
        k3 = key.reshape(key.shape[0], c["groups"], -1)
        two = torch.sort(k3, dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.sort(two, dim=-1, descending=True, stable=True).indices[:, :c["keep"]]
        open_ = torch.zeros_like(two, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(open_[..., None], k3, -torch.inf).reshape(key.shape)
    idx = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :c["topk"]]
    w = s.gather(1, idx)
    return idx, w / (w.sum(-1, keepdim=True) + 1e-20) * c["scale"]


def _plain_linear(c, st):
    N8, B = _up(c["N"], 8) // 8, _up(c["K"], BLK_K) // BLK_K
    x = st["x"].float()
    y = x @ _int4(st["w"], N8, B)[0, :c["N"], :c["K"]].T
    if c["swiglu"]:
        y = _silu(y) * (x @ _int4(st["w_up"], N8, B)[0, :c["N"], :c["K"]].T)
    if c["res"]:
        y = y + st["res"].float()
    return y if c["f32"] else y.to(torch.bfloat16)


def _plain_block(c, st):
    H, I, E = c["H"], c["I"], c["E"]
    idx, w = _route(c, st)
    x = st["x"].float()
    picked, at = torch.unique(idx, return_inverse=True)      # the experts to run; every row through each, weight 0 where not picked
    mats = st["pool"].reshape(E, 3, -1)[picked]
    h = _silu(torch.einsum("mh,uih->umi", x, _int4(mats[:, 0], I // 8, H // BLK_K)))
    h = h * torch.einsum("mh,uih->umi", x, _int4(mats[:, 1], I // 8, H // BLK_K))
    y = torch.einsum("umi,uhi->umh", h, _int4(mats[:, 2], H // 8, I // BLK_K))
    mix = torch.zeros(x.shape[0], picked.numel(), device="cuda").scatter_(1, at, w.float())
    out = torch.einsum("mu,umh->mh", mix, y)
    if c["shared"]:
        g, u, d = st["shared"]
        out = out + (_silu(x @ _bf16(g, I, H).T) * (x @ _bf16(u, I, H).T)) @ _bf16(d, H, I).T
    if c["res"]:
        out = out + st["res"].float()
    return {"out": out.to(torch.bfloat16), "idx": idx.to(torch.int32), "w": w.float()}


def run(st):
    c = st["case"]
    if not own:
        return _plain_linear(c, st) if c["op"] == "linear" else _plain_block(c, st)
    if c["op"] == "linear":
        from dsgx10_b200 import linear
        return linear.linear_decode(st["handle"], st["x"], res=st.get("res"), out_dtype=torch.float32 if c["f32"] else torch.bfloat16)
    out, idx, w = st["handle"].run(st["layer_w"], st["x"], res=st.get("res"))
    return {"out": out, "idx": idx, "w": w}


# ---------------------------------------------------------------------------------------------------- floors and exact

def _int4_bytes(N, K):
    g = -(-K // G)
    return N * (-(-K // 2) + 2 * g + -(-g // 2))


def work(case):
    c, M = case, case["M"]
    if c["op"] == "linear":
        N, K, n = c["N"], c["K"], 2 if c["swiglu"] else 1
        return {"bytes": n * _int4_bytes(N, K) + M * (2 * K + (4 if c["f32"] else 2) * N + (2 * N if c["res"] else 0)),
                "flops": 2 * n * M * N * K}
    H, I, E, k = c["H"], c["I"], c["E"], c["topk"]
    union = E * (1 - (1 - k / E) ** M)               # distinct picks of M rows, on average
    b = union * (2 * _int4_bytes(I, H) + _int4_bytes(H, I)) + E * H * 4 + M * H * (6 if c["res"] else 4)
    f = M * k * 6 * H * I + 2 * M * E * H
    if c["shared"]:
        b, f = b + 6 * H * I, f + M * 6 * H * I
    return {"bytes": int(b), "flops": int(f)}


def _weight64(raw, n, K, Kp):
    """Rows n (a range) of an INT4 matrix from its bytes, weight by weight, by the layout's address rule."""
    k = torch.arange(K, device="cuda")
    b, r = k // 512, k % 512
    jj, q, t, i = r // 128, r // 64 % 2, r // 16 % 4, r % 16
    rows = torch.arange(n.start, n.stop, device="cuda")[:, None]
    base = (rows // 8 * (Kp // 512) + b) * BLK_BYTES
    g = rows % 8
    u = raw[base + 512 * jj + 16 * (4 * g + t) + 8 * q + i // 2].to(torch.int32) >> (4 * (i % 2)) & 15
    at = base + 2048 + 32 * g + 16 * (t // 2) + 2 * (2 * jj + q)
    s = (raw[at].to(torch.int32) | raw[at + 1].to(torch.int32) << 8) << 16
    z = raw[base + 2304 + 8 * g + 4 * (t // 2) + jj].to(torch.int32) >> (4 * q) & 15
    return (u - z).double() * s.view(torch.float32).double()


def _product64(x, raw, N, K):
    raw, Kp = raw.reshape(-1), _up(K, 512)
    step = max(8, (1 << 24) // K // 8 * 8)
    return torch.cat([x @ _weight64(raw, range(n, min(N, n + step)), K, Kp).T for n in range(0, N, step)], 1)


def _shared64(t, N, K):
    n, k = torch.arange(N, device="cuda")[:, None], torch.arange(K, device="cuda")
    r = k % 128
    return t.reshape(-1)[(n // 8 * (K // 128) + k // 128) * 1024 + (2 * (r // 64) + r // 8 % 2) * 256 + (4 * (n % 8) + r // 16 % 4) * 8 + r % 8].double()


def exact(case, seed):
    c, st = case, _inputs(case, seed)
    x = st["x"].double()
    act = lambda a, b: a * torch.sigmoid(a) * b
    if c["op"] == "linear":
        y = _product64(x, st["w"], c["N"], c["K"])
        if c["swiglu"]:
            y = act(y, _product64(x, st["w_up"], c["N"], c["K"]))
        return y + st["res"].double() if c["res"] else y
    H, I, E, M = c["H"], c["I"], c["E"], c["M"]
    logits = (x[:, None] * st["wr"].double()).sum(-1)
    s = {"sigmoid": torch.sigmoid, "softmax": lambda l: torch.softmax(l, -1),
         "sqrtsoftplus": lambda l: torch.nn.functional.softplus(l, threshold=50).sqrt()}[c["score"]](logits)
    key = (s + st["bias"].double() if c["bias"] else s).tolist()
    picks, size = [], E // c["groups"]
    for r in range(M):
        best = sorted(range(c["groups"]), key=lambda g: (-sum(sorted(key[r][g * size:(g + 1) * size])[-2:]), g))[:c["keep"]]
        ids = [e for e in range(E) if e // size in best]
        picks.append(sorted(ids, key=lambda e: (-key[r][e], e))[:c["topk"]])
    idx = torch.tensor(picks, device="cuda")
    w = s.gather(1, idx)
    w = w / (w.sum(-1, keepdim=True) + 1e-20) * c["scale"]
    out = st["res"].double() if c["res"] else torch.zeros_like(x)
    pool = st["pool"].reshape(E, 3, -1)
    for e in sorted(set(sum(picks, []))):
        rows = (idx == e).any(1).nonzero()[:, 0]
        h = act(_product64(x[rows], pool[e, 0], I, H), _product64(x[rows], pool[e, 1], I, H))
        out[rows] += _product64(h, pool[e, 2], H, I) * w[idx == e][:, None]
    if c["shared"]:
        g, u, d = st["shared"]
        out = out + act(x @ _shared64(g, I, H).T, x @ _shared64(u, I, H).T) @ _shared64(d, H, I).T
    return {"out": out, "idx": None, "w": w}
