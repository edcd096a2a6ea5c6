"""Work of the operators that pick rows of a hashed weight by an index: embedding lookup and its gradient, sorting rows by
the block they belong to, and matrix products grouped by expert.

Every weight here is virtual, as everywhere in this package: W[k, n] = hashed[off(k // BK, n // BN) + (k % BK) * BN + n % BN],
with `off` a hash of the tile's coordinates.  An embedding table is one such matrix with a row for each token; the matrices
of G experts are one such matrix with the experts' rows one below the other, each expert's rows starting at a new tile.

`run` computes each pass either from elementary torch operations in 32 bits (`own` false) or by the package's public calls
(`own` true); `exact` computes it in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
SMALL_PRIME = 45007          # the layers' default prime, with the two-level hash
LARGE_PRIME = 2038074743     # the single-level hash's
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    emb = dict(op="embed", bk=32, bn=64, two_level=True, compress=16)
    grp = dict(op="experts", bk=32, bn=64, two_level=True, compress=16, behind=0, bias=False, relu=False)
    return [
        # one step of decoding: a single new token
        dict(emb, name="embed: one token", tokens=1, vocab=32768, dim=4096, dtype="bf16", train=False, padded=0.0),
        # a prompt batch, lookup only
        dict(emb, name="embed: prompt", tokens=8192, vocab=32768, dim=4096, dtype="bf16", train=False, padded=0.0),
        # a training step of the table: lookup and gradient, right-padded sequences
        dict(emb, name="embed: training", tokens=16384, vocab=32768, dim=4096, dtype="bf16", train=True, padded=0.1),
        # a large vocabulary and a long batch, larger hash tiles
        dict(emb, name="embed: training, long", tokens=131072, vocab=131072, dim=1024, dtype="bf16", train=True, padded=0.0,
             bk=128, bn=128, two_level=False),
        # sizes that divide nothing, in 32 bits
        dict(emb, name="embed: training, odd", tokens=1777, vocab=50021, dim=1000, dtype="fp32", train=True, padded=0.05,
             bk=16, bn=24),
        # routing of a small decoding batch: 32 rows, two experts each
        dict(op="sort", name="sort: decoding", keys=64, bins=16, dropped=0.0),
        # routing of a long batch with capacity drops
        dict(op="sort", name="sort: long batch", keys=131072, bins=128, dropped=0.03),
        # decoding: few rows for each expert, the weights are what is read
        dict(grp, name="experts: decoding", rows=64, groups=16, k=2048, n=4096, dtype="bf16", train=False, skew=1.0,
             bias=True, relu=True),
        # a prompt batch through the first product of an expert layer
        dict(grp, name="experts: prompt", rows=8192, groups=32, k=2048, n=4096, dtype="bf16", train=False, skew=0.5, bias=True,
             relu=True, behind=100),
        # a training step: product, input gradient, weight gradient, bias gradient
        dict(grp, name="experts: training", rows=16384, groups=16, k=4096, n=4096, dtype="bf16", train=True, skew=0.5, bias=True,
             bk=64),
        # many small experts: the weight gradient adds far more than it multiplies
        dict(grp, name="experts: training, many", rows=4096, groups=64, k=1024, n=2048, dtype="bf16", train=True, skew=0.5),
        # 32-bit activations and ragged sizes
        dict(grp, name="experts: training, odd", rows=1003, groups=7, k=520, n=264, dtype="fp32", train=True, skew=1.0, bias=True,
             behind=13, bk=32, bn=32, two_level=False, compress=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["embed", "embed", "sort", "experts", "experts", "experts"])
    if kind == "sort":
        return dict(op="sort", keys=_log_int(rng, 1, 131072), bins=_log_int(rng, 1, 1024), dropped=rng.choice([0.0, 0.03]))
    if kind == "embed":
        c = dict(op="embed", tokens=_log_int(rng, 1, 100000), vocab=_log_int(rng, 1000, 131072),
                 dim=_log_int(rng, 64, 4096), dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.6,
                 padded=rng.choice([0.0, 0.1]), bk=rng.choice([16, 32, 64, 128]), bn=rng.choice([24, 32, 64, 128]),
                 two_level=rng.random() < 0.5, compress=rng.choice([4, 16]))
        if rng.random() < 0.6:
            c["dim"] = max(64, c["dim"] // 64 * 64)
        while c["tokens"] * c["dim"] > 2**26:
            c["tokens"] = c["tokens"] // 2 + 1
        while c["vocab"] * c["dim"] > 2**27:
            c["vocab"] = c["vocab"] // 2 + 1
        while c["vocab"] * c["dim"] // c["compress"] <= 2 * c["bk"] * c["bn"]:
            c["vocab"] *= 2
        return c
    c = dict(op="experts", rows=_log_int(rng, 1, 16384), groups=_log_int(rng, 1, 64), k=_log_int(rng, 128, 4096),
             n=_log_int(rng, 128, 4096), dtype=rng.choice(["bf16", "bf16", "bf16", "fp32"]), train=rng.random() < 0.6,
             skew=rng.choice([0.0, 0.5, 1.0]), bias=rng.random() < 0.5, relu=False, behind=0, bk=rng.choice([32, 64, 128]),
             bn=rng.choice([64, 128]), two_level=rng.random() < 0.5, compress=rng.choice([4, 16]))
    odd = rng.random()
    if odd < 0.85:                       # most layers have sides that are multiples of 8 at least
        step = 64 if odd < 0.5 else 8
        c["k"], c["n"] = c["k"] // step * step, c["n"] // step * step
    else:
        c["k"], c["n"] = c["k"] // 4 + 37, c["n"] // 4 + 37
    if not c["train"]:
        c["relu"] = rng.random() < 0.5
    if c["rows"] > 64 and rng.random() < 0.3:
        c["behind"] = rng.randrange(1, c["rows"] // 8)
    if c["dtype"] == "fp32":             # (three products in the place of one)
        c["rows"] = c["rows"] // 4 + 1
    while c["groups"] * c["k"] * c["n"] > 2**28 - 1:
        c["groups"] = c["groups"] // 2
    while c["groups"] * c["k"] * c["n"] // c["compress"] <= 2 * c["bk"] * c["bn"]:
        c["compress"], c["groups"] = 4, c["groups"] + 1
    return c


def work(c):
    if c["op"] == "sort":
        return {"bytes": c["keys"] * (8 + 4) + 4 * (c["bins"] + 1), "flops": 0}
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "embed":
        H, data = _hashed_size(c), c["tokens"] * c["dim"]
        b = 8 * c["tokens"] + 4 * min(H, data) + size * data
        if c["train"]:
            b += size * data + 4 * H
        return {"bytes": b, "flops": data * (2 if c["train"] else 1)}
    H, T, K, N, G = _hashed_size(c), c["rows"], c["k"], c["n"], c["groups"]
    bias = 4 * G * N if c["bias"] else 0
    b = size * T * (K + N) + 4 * H + 4 * (G + 1) + bias
    if c["train"]:
        b += size * T * (K + N) + 4 * H + bias
    return {"bytes": b, "flops": (6 if c["train"] else 2) * (T - c["behind"]) * K * N}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _hashed_size(c):
    rows, cols = (c["vocab"], c["dim"]) if c["op"] == "embed" else (c["groups"] * c["k"], c["n"])
    return max(rows * cols // c["compress"], 2 * c["bk"] * c["bn"])


def _random_numbers(c, seed):
    prime = SMALL_PRIME if c["two_level"] else LARGE_PRIME
    rng = random.Random(seed)
    return [prime] + [rng.randrange(1, prime) for _ in range(7)]


def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if c["op"] == "sort":
        p = torch.rand(c["bins"], generator=g, device=DEVICE).square() + 0.01      # some bins are wanted far more than others
        edges = (p.cumsum(0) / p.sum()).contiguous()
        u = torch.rand(c["keys"], generator=g, device=DEVICE)
        keys = torch.searchsorted(edges, u).clamp_(max=c["bins"] - 1)
        dropped = torch.rand(c["keys"], generator=g, device=DEVICE) < c["dropped"]
        return dict(c=c, keys=torch.where(dropped, -1, keys))
    dtype = DTYPES[c["dtype"]]
    s = dict(c=c, R=_random_numbers(c, seed))
    s["random_numbers"] = torch.tensor(s["R"], dtype=torch.int64)
    H = _hashed_size(c)
    if c["op"] == "embed":
        T, V, D = c["tokens"], c["vocab"], c["dim"]
        # the frequency of a token falls with its rank, as in text
        ids = (torch.rand(T, generator=g, device=DEVICE, dtype=torch.float64) * math.log(V)).exp().long().clamp_(0, V - 1)
        s["padding"] = V - 1
        ids[T - int(T * c["padded"]):] = s["padding"]
        s["ids"] = ids
        s["scale"] = math.sqrt(D)
        s["hashed"] = torch.randn(H, generator=g, device=DEVICE).mul_(D**-0.5).requires_grad_()
        if c["train"]:
            s["grad"] = torch.randn((T, D), generator=g, device=DEVICE).to(dtype)
        return s
    T, G, K, N = c["rows"], c["groups"], c["k"], c["n"]
    rng = np.random.RandomState(seed % 2**31)
    p = np.exp(c["skew"] * rng.randn(G))
    if G >= 4:
        p[rng.randint(G)] = 0.0                                                    # an expert that no row chose
    sizes = rng.multinomial(T - c["behind"], p / p.sum())
    s["sizes"], s["largest"] = [int(v) for v in sizes], max(1, int(sizes.max()))
    s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).to(DEVICE)
    s["scale"] = 1.0
    s["x"] = torch.randn((T, K), generator=g, device=DEVICE).to(dtype).requires_grad_(c["train"])
    s["hashed"] = torch.rand(H, generator=g, device=DEVICE).mul_(2).sub_(1).mul_(K**-0.5).requires_grad_(c["train"])
    s["bias"] = torch.randn((G, N), generator=g, device=DEVICE).mul_(0.1).requires_grad_(c["train"]) if c["bias"] else None
    if c["train"]:
        s["grad"] = torch.randn((T, N), generator=g, device=DEVICE).to(dtype)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(s):
    op = s["c"]["op"]
    if own:
        return {"sort": _own_sort, "embed": _own_embed, "experts": _own_experts}[op](s)
    return {"sort": _plain_sort, "embed": _plain_embed, "experts": _plain_experts}[op](s)


def _own_config(c):
    from rzlinear_b200 import RzConfig
    return RzConfig(block_size_k=c["bk"], block_size_n=c["bn"], hash_mode=1 if c["two_level"] else 0, relu=bool(c.get("relu")))


def _own_sort(s):
    from rzlinear_b200 import sort_rows
    order, offsets = sort_rows(s["keys"], s["c"]["bins"])
    return {"order": order, "offsets": offsets}


def _own_embed(s):
    from rzlinear_b200 import RzEmbeddingFunction
    c = s["c"]
    if not c["train"]:
        with torch.no_grad():
            return {"out": RzEmbeddingFunction.apply(s["ids"], s["hashed"], s["random_numbers"], c["vocab"], c["dim"], s["scale"],
                                                     _own_config(c), s["padding"], DTYPES[c["dtype"]])}
    out = RzEmbeddingFunction.apply(s["ids"], s["hashed"], s["random_numbers"], c["vocab"], c["dim"], s["scale"], _own_config(c),
                                    s["padding"], DTYPES[c["dtype"]])
    (dh,) = torch.autograd.grad(out, s["hashed"], s["grad"])
    return {"out": out.detach(), "hashed_grad": dh}


def _own_experts(s):
    from rzlinear_b200 import RzGroupedLinearFunction
    c = s["c"]
    if not c["train"]:
        with torch.no_grad():
            return {"out": RzGroupedLinearFunction.apply(s["x"], s["hashed"], s["random_numbers"], s["offsets"], c["n"], s["scale"],
                                                         _own_config(c), s["bias"])}
    out = RzGroupedLinearFunction.apply(s["x"], s["hashed"], s["random_numbers"], s["offsets"], c["n"], s["scale"], _own_config(c),
                                        s["bias"])
    wanted = [s["x"], s["hashed"]] + ([s["bias"]] if c["bias"] else [])
    grads = torch.autograd.grad(out, wanted, s["grad"])
    return {"out": out.detach(), "input_grad": grads[0], "hashed_grad": grads[1], "bias_grad": grads[2] if c["bias"] else None}


def _plain_offset(c, R, H, pk, pn):
    """Start of tile (pk, pn) in the hashed array."""
    v = (pk * R[3] + pn * R[2] + R[1]) % R[0]
    if c["two_level"]:
        v = v * R[0] + (pk * R[7] + pn * R[5] + R[4]) % R[0]
    return v % (H - c["bk"] * c["bn"])


def _plain_index(c, R, H, pk, k_in, cols):
    """Where the rows (tile row pk, row k_in of it) of the virtual matrix are in the hashed array: [rows, cols]."""
    n = torch.arange(cols, device=DEVICE)
    pn = torch.arange(-(-cols // c["bn"]), device=DEVICE)
    off = _plain_offset(c, R, H, pk[:, None], pn[None, :])
    return off[:, n // c["bn"]] + k_in[:, None] * c["bn"] + n % c["bn"]


def _plain_sort(s):
    keys, bins = s["keys"], s["c"]["bins"]
    inside = (keys >= 0) & (keys < bins)
    key = torch.where(inside, keys, bins)
    ranked, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ranked, torch.arange(bins + 1, device=DEVICE))
    return {"order": order.int(), "offsets": offsets.int()}


def _plain_embed(s):
    c, ids, H = s["c"], s["ids"], s["hashed"].numel()
    index = _plain_index(c, s["R"], H, ids // c["bk"], ids % c["bk"], c["dim"])
    used = ((ids >= 0) & (ids < c["vocab"]) & (ids != s["padding"]))[:, None]
    out = torch.where(used, s["hashed"].detach()[index] * s["scale"], 0.0).to(DTYPES[c["dtype"]])
    if not c["train"]:
        return {"out": out}
    part = torch.where(used, s["grad"].float() * s["scale"], 0.0)
    dh = torch.zeros(H, device=DEVICE).index_add_(0, index.flatten(), part.flatten())
    return {"out": out, "hashed_grad": dh}


def _plain_experts(s):
    c, H, off = s["c"], s["hashed"].numel(), s["offsets"].long()
    T, G, K, N, C = c["rows"], c["groups"], c["k"], c["n"], s["largest"]
    k, nk = torch.arange(K, device=DEVICE), -(-K // c["bk"])
    pk = (torch.arange(G, device=DEVICE)[:, None] * nk + k // c["bk"]).flatten()
    index = _plain_index(c, s["R"], H, pk, (k % c["bk"]).repeat(G), N)
    W = s["hashed"].detach()[index].view(G, K, N)
    # every group's rows, filled up to the largest group's
    row = off[:-1, None] + torch.arange(C, device=DEVICE)
    there = (row < off[1:, None])[..., None]
    row = row.clamp(max=T - 1)
    xs = torch.where(there, s["x"].detach().float()[row], 0.0)
    t = torch.arange(T, device=DEVICE)
    group = torch.searchsorted(off[1:], t, right=True)
    held, group = (group < G)[:, None], group.clamp(max=G - 1)
    place = (t - off[group]).clamp(0, C - 1)
    y = torch.bmm(xs, W) * s["scale"]
    if c["bias"]:
        y = y + s["bias"].detach()[:, None, :]
    if c["relu"]:
        y = y.clamp(min=0)
    dtype = DTYPES[c["dtype"]]
    out = torch.where(held, y[group, place], 0.0).to(dtype)
    if not c["train"]:
        return {"out": out}
    gs = torch.where(there, s["grad"].float()[row], 0.0)
    dx = torch.where(held, (torch.bmm(gs, W.transpose(1, 2)) * s["scale"])[group, place], 0.0).to(dtype)
    dw = torch.bmm(xs.transpose(1, 2), gs) * s["scale"]
    dh = torch.zeros(H, device=DEVICE).index_add_(0, index.flatten(), dw.flatten())
    return {"out": out, "input_grad": dx, "hashed_grad": dh, "bias_grad": gs.sum(1) if c["bias"] else None}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------
def _exact_starts(c, R, H, tile_rows, cols):
    """[tile rows, tile columns] table of slice starts, from the definition, on the host."""
    pk = np.asarray(tile_rows, dtype=object)[:, None]
    pn = np.arange(-(-cols // c["bn"]), dtype=object)[None, :]
    first = (pk * R[3] + pn * R[2] + R[1]) % R[0]
    if c["two_level"]:
        first = first * R[0] + (pk * R[7] + pn * R[5] + R[4]) % R[0]
    return torch.from_numpy((first % (H - c["bk"] * c["bn"])).astype(np.int64)).to(DEVICE)


def _exact_rows(c, R, H, rows, tile_row, in_tile, cols):
    """Words of the hashed array that make up the given rows of the virtual matrix, [len(rows), cols]."""
    table = _exact_starts(c, R, H, np.arange(int(tile_row.max()) + 1), cols)
    begin = table[tile_row] + in_tile[:, None] * c["bn"]                       # [rows, tile columns]: one segment each
    words = begin[:, :, None] + torch.arange(c["bn"], device=DEVICE)
    return words.reshape(len(rows), -1)[:, :cols]


def _exact_scatter(words, values, H):
    return torch.bincount(words.reshape(-1), weights=values.reshape(-1), minlength=H)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "sort":
        keys = s["keys"].cpu().numpy()
        key = np.where((keys < 0) | (keys >= c["bins"]), c["bins"], keys)
        count = np.bincount(key, minlength=c["bins"] + 1)
        return {"order": np.lexsort((np.arange(len(key)), key)).astype(np.int32),
                "offsets": (np.cumsum(count) - count).astype(np.int32)}
    h, R = s["hashed"].detach().double(), s["R"]
    H = h.numel()
    if c["op"] == "embed":
        ids, D = s["ids"], c["dim"]
        live = (ids != s["padding"]).nonzero()[:, 0]
        out = torch.zeros((len(ids), D), dtype=torch.float64, device=DEVICE)
        dh = torch.zeros(H, dtype=torch.float64, device=DEVICE)
        if len(live):
            v = ids[live]
            words = _exact_rows(c, R, H, v, v.div(c["bk"], rounding_mode="floor"), v.remainder(c["bk"]), D)
            out[live] = h[words] * s["scale"]
            if c["train"]:
                dh = _exact_scatter(words, s["grad"][live].double(), H) * s["scale"]
        return {"out": out, "hashed_grad": dh} if c["train"] else {"out": out}
    K, N, nk = c["k"], c["n"], -(-c["k"] // c["bk"])
    k = torch.arange(K, device=DEVICE)
    out = torch.zeros((c["rows"], N), dtype=torch.float64, device=DEVICE)
    dx = torch.zeros((c["rows"], K), dtype=torch.float64, device=DEVICE)
    dh = torch.zeros(H, dtype=torch.float64, device=DEVICE)
    db = torch.zeros((c["groups"], N), dtype=torch.float64, device=DEVICE)
    table = _exact_starts(c, R, H, np.arange(c["groups"] * nk), N)
    begin = 0
    for g, size in enumerate(s["sizes"]):
        rows = slice(begin, begin + size)
        begin += size
        if not size:
            continue
        words = (table[g * nk + k.div(c["bk"], rounding_mode="floor")] + (k.remainder(c["bk"]) * c["bn"])[:, None])[:, :, None] \
            + torch.arange(c["bn"], device=DEVICE)
        words = words.reshape(K, -1)[:, :N]
        w, x = h[words] * s["scale"], s["x"].detach()[rows].double()
        y = x @ w
        if c["bias"]:
            y += s["bias"].detach()[g].double()
        out[rows] = y.relu() if c["relu"] else y
        if c["train"]:
            gy = s["grad"][rows].double()
            dx[rows] = gy @ w.T
            dh += _exact_scatter(words, (x.T @ gy) * s["scale"], H)
            db[g] = gy.sum(0)
    if not c["train"]:
        return {"out": out}
    return {"out": out, "input_grad": dx, "hashed_grad": dh, "bias_grad": db if c["bias"] else None}
