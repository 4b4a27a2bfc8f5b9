"""Learned type vectors: the operators between type indices and the vector-typed grids.

``embed``    y[n] = s_n W[t_n], a zero row where t_n names no row of W; its gradients dW and ds
``norm``     layer norm over the channels, with the gradients of its input, weight and bias
``dropout``  y = x keep / (1 - p), keep from a counter-based generator; its gradient is the same map
``encode``   dropout(norm(s W[t])), the three in one, with the gradients of W and of norm's parameters

The random numbers are a function of (seed, offset, position): element e of the flattened array takes
the 16-bit half e % 8 of the four 32-bit words (low half first) that Philox4x32 with ten rounds gives
for the counter (e / 8, offset) and the key seed; it is kept where that half is at least
T = round(65536 p), and kept elements are scaled by 65536 / (65536 - T).
"""
import math

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"
EPS = 1e-5


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def listed():
    return [
        # one atom looked up: what a call costs when there is nothing to do
        {"name": "embed one", "op": "embed", "back": False, "batch": 1, "length": 1, "rows": 28,
         "channels": 32, "type": F32, "index": "float32", "per_token": False},
        # a padded batch of 50 complexes of 1,015 to 4,080 atoms (float indices, padded with type 0
        # whose gradient is zero), soft-typed by a weight per atom; one training step
        {"name": "embed atoms", "op": "embed", "back": True, "batch": 50, "length": 4080, "rows": 28,
         "channels": 28, "type": F32, "index": "float32", "per_token": True},
        # a vocabulary of words: few frequent rows, many rare ones, an odd number of rows
        {"name": "embed words", "op": "embed", "back": True, "batch": 16, "length": 1024,
         "rows": 50257, "channels": 1024, "type": BF16, "index": "int64", "per_token": False},
        # a large table: the gradient's own rows are most of the traffic
        {"name": "embed large", "op": "embed", "back": True, "batch": 16, "length": 4096,
         "rows": 131072, "channels": 4096, "type": BF16, "index": "int64", "per_token": False},
        # one token while serving
        {"name": "norm one", "op": "norm", "back": False, "tokens": 1, "channels": 4096, "type": BF16,
         "params": F32},
        # the 121,231 atoms of a batch of 50 complexes, 28 channels each
        {"name": "norm atoms", "op": "norm", "back": True, "tokens": 121231, "channels": 28,
         "type": F32, "params": F32},
        # odd sizes: rows that start at every alignment
        {"name": "norm odd", "op": "norm", "back": True, "tokens": 4099, "channels": 1001, "type": F16,
         "params": F16},
        # a training step of a wide model
        {"name": "norm large", "op": "norm", "back": True, "tokens": 32768, "channels": 8192,
         "type": BF16, "params": F32},
        # a small activation, odd length
        {"name": "dropout small", "op": "dropout", "tokens": 5, "channels": 1001, "type": F32, "p": 0.1},
        # a training step's activation and its gradient
        {"name": "dropout large", "op": "dropout", "tokens": 32768, "channels": 8192, "type": BF16,
         "p": 0.1},
        # the whole way from the atoms of a batch of 50 complexes to their type vectors
        {"name": "encode atoms", "op": "encode", "back": True, "batch": 50, "length": 2425, "rows": 28,
         "channels": 32, "type": F32, "index": "float32", "params": F32, "p": 0.1},
        # the same for words
        {"name": "encode words", "op": "encode", "back": True, "batch": 32, "length": 1024,
         "rows": 32000, "channels": 2048, "type": BF16, "index": "int64", "params": F32, "p": 0.1},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["embed", "norm", "dropout", "encode"])
    dtype = rng.choice([F32, F16, BF16])
    channels = _log(rng, 3, 8192)
    if rng.random() < 0.5:                       # half of the widths are multiples of eight
        channels = max(8, channels // 8 * 8)
    most = min(1 << 18, (1 << 27) // channels)   # at most half of the largest listed array
    params = rng.choice([F32, dtype])
    if kind in ("norm", "dropout"):
        c = {"op": kind, "tokens": _log(rng, 1, most), "channels": channels, "type": dtype}
        c.update({"back": rng.random() < 0.7, "params": params} if kind == "norm"
                 else {"p": rng.choice([0.0, 0.05, 0.1, 0.3, 0.5, 0.9])})
        return c
    batch = rng.choice([1, 1, 4, 16, 50])
    c = {"op": kind, "back": rng.random() < 0.7, "batch": batch,
         "length": _log(rng, 1, max(2, most // batch)),
         "rows": _log(rng, 2, max(3, min(1 << 18, (1 << 28) // channels))), "channels": channels,
         "type": dtype, "index": rng.choice(["float32", "int32", "int64"])}
    c.update({"per_token": rng.random() < 0.5} if kind == "embed"
             else {"params": params, "p": rng.choice([0.0, 0.1, 0.5])})
    return c


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gradient_like(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _tokens(case, g):
    """Indices of a padded batch and which of them are padding: atoms (up to 64 rows) are spread
    evenly over the types and padded with type 0; words fall off with their rank and are padded
    with -1, which names no row."""
    b, n, rows = case["batch"], case["length"], case["rows"]
    u = torch.rand((b, n), generator=g, device="cuda", dtype=torch.float64)
    if rows <= 64:
        t = (u * rows).long().clamp_(max=rows - 1)
        pad = 0
    else:
        rank = torch.exp(u * math.log(rows)).long().clamp_(1, rows) - 1
        t = torch.randperm(rows, generator=g, device="cuda")[rank]
        pad = -1
    length = torch.randint(max(1, n // 4), n + 1, (b, 1), generator=g, device="cuda")
    length[0] = n
    padding = torch.arange(n, device="cuda")[None, :] >= length
    t = torch.where(padding, torch.full_like(t, pad), t)
    return t.to(getattr(torch, case["index"])), padding


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = getattr(torch, case["type"])
    s = dict(case)
    if case["op"] in ("norm", "dropout"):
        shape = (case["tokens"], case["channels"])
        # activations: channels of different widths and offsets, a few of them large
        width = torch.exp(0.7 * torch.randn(shape[1], generator=g, device="cuda"))
        shift = 0.5 * torch.randn(shape[1], generator=g, device="cuda")
        x = torch.randn(shape, generator=g, device="cuda")
        s["x"] = x.mul_(width).add_(shift).to(dtype)
        s["grad"] = _gradient_like(shape, dtype, g)
    else:
        s["tokens_in"], padding = _tokens(case, g)
        c = case["channels"]
        table = torch.randn((case["rows"], c), generator=g, device="cuda")
        s["table"] = table.mul_(0.02 if case["rows"] > 64 else 1.0).to(dtype)
        grad = _gradient_like(tuple(s["tokens_in"].shape) + (c,), dtype, g)
        s["grad"] = grad.masked_fill_(padding[..., None], 0)
        s["scale"] = math.sqrt(c)
        if case.get("per_token"):
            s["scale"] = 0.5 + torch.rand(s["tokens_in"].shape, generator=g, device="cuda")
    if case["op"] in ("norm", "encode"):
        params = getattr(torch, case["params"])
        c = case["channels"]
        s["weight"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(params)
        s["bias"] = (0.1 * torch.randn(c, generator=g, device="cuda")).to(params)
    if "p" in case:
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ seed, seed % 1000
    return s


# ---------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------
MASK = 0xFFFFFFFF


def _round_of(c, key):
    """One round of Philox4x32 on 64-bit integers that hold 32-bit words (a product of two of them
    wraps around 2^64; its bits are the wanted ones)."""
    a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
    return [((b >> 32) & MASK) ^ c[1] ^ key[0], b & MASK, ((a >> 32) & MASK) ^ c[3] ^ key[1], a & MASK]


def _keep(n, p, seed, offset):
    """(which of the first n elements are kept, the factor of the kept ones)"""
    limit = int(math.floor(p * 65536 + 0.5))
    group = torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64)
    zero = torch.zeros_like(group)
    c = [group & MASK, group >> 32, zero + (offset & MASK), zero + ((offset >> 32) & MASK)]
    k0, k1 = seed & MASK, (seed >> 32) & MASK
    for r in range(10):
        c = _round_of(c, ((k0 + r * 0x9E3779B9) & MASK, (k1 + r * 0xBB67AE85) & MASK))
    halves = torch.stack([h for w in c for h in (w & 0xFFFF, w >> 16)], dim=1).reshape(-1)[:n]
    return halves >= limit, 65536.0 / (65536 - limit) if limit < 65536 else 0.0


def _dropped(x, p, seed, offset):
    keep, factor = _keep(x.numel(), p, seed, offset)
    return torch.where(keep.view(x.shape), x * factor, torch.zeros_like(x))


def _rows_of(s):
    """(flat row numbers, which of them name a row, the scale as a column or a number)"""
    t = torch.floor(s["tokens_in"]).long() if s["tokens_in"].is_floating_point() else s["tokens_in"].long()
    t = t.reshape(-1)
    named = (t >= 0) & (t < s["rows"])
    scale = s["scale"]
    return torch.where(named, t, torch.zeros_like(t)), named, scale.reshape(-1, 1) if torch.is_tensor(scale) else scale


def _normed(x):
    d = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS)
    return d * r, r


def _norm_gradient(g, h, r, weight):
    q = g * weight
    dx = r * (q - q.mean(-1, keepdim=True) - h * (q * h).mean(-1, keepdim=True))
    return dx, (g * h).sum(0), g.sum(0)


def _embed(s):
    t, named, scale = _rows_of(s)
    dtype = s["table"].dtype
    rows = s["table"].float()[t] * named[:, None]
    out = [(rows * scale).to(dtype).view(s["grad"].shape)]
    if s["back"]:
        g = s["grad"].float().view(rows.shape)
        dw = torch.zeros(s["table"].shape, device="cuda").index_add_(0, t, g * named[:, None] * scale)
        out.append(dw.to(dtype))
        if s["per_token"]:
            out.append((g * rows).sum(-1).view(s["tokens_in"].shape))
    return out


def _norm(s):
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    h, r = _normed(x)
    out = [(h * w + b).to(s["x"].dtype)]
    if s["back"]:
        dx, dw, db = _norm_gradient(s["grad"].float(), h, r, w)
        out += [dx.to(s["x"].dtype), dw.to(s["weight"].dtype), db.to(s["weight"].dtype)]
    return out


def _dropout(s):
    return [_dropped(x.float(), s["p"], s["seed"], s["offset"]).to(x.dtype) for x in (s["x"], s["grad"])]


def _encode(s):
    t, named, scale = _rows_of(s)
    dtype, w, b = s["table"].dtype, s["weight"].float(), s["bias"].float()
    h, r = _normed(s["table"].float()[t] * scale)
    y = (h * w + b) * named[:, None]
    out = [_dropped(y, s["p"], s["seed"], s["offset"]).to(dtype).view(s["grad"].shape)]
    if s["back"]:
        g = _dropped(s["grad"].float().view(y.shape), s["p"], s["seed"], s["offset"]) * named[:, None]
        dx, dw, db = _norm_gradient(g, h, r, w)
        table = torch.zeros(s["table"].shape, device="cuda").index_add_(0, t, dx * scale)
        out += [table.to(dtype), dw.to(s["weight"].dtype), db.to(s["weight"].dtype)]
    return out


# ---------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------
def _framework(s):
    import libmolgrid_amd as molgrid
    if s["op"] == "embed":
        out = [molgrid.embed_types(s["tokens_in"], s["table"], s["scale"])]
        if s["back"]:
            grads = molgrid.embed_types_backward(s["grad"], s["tokens_in"], s["table"], s["scale"])
            out += [x for x in grads if x is not None]
        return out
    if s["op"] == "norm":
        y, mean, rstd = molgrid.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if not s["back"]:
            return [y]
        return [y] + list(molgrid.layer_norm_backward(s["grad"], s["x"], mean, rstd, s["weight"]))
    if s["op"] == "dropout":
        return [molgrid.dropout(x, s["p"], s["seed"], s["offset"]) for x in (s["x"], s["grad"])]
    how = dict(scale=s["scale"], eps=EPS, p=s["p"], seed=s["seed"], offset=s["offset"])
    out = [molgrid.encode_types(s["tokens_in"], s["table"], s["weight"], s["bias"], **how)]
    if s["back"]:
        out += list(molgrid.encode_types_backward(s["grad"], s["tokens_in"], s["table"], s["weight"], **how))
    return out


def run(state):
    if own:
        return _framework(state)
    return {"embed": _embed, "norm": _norm, "dropout": _dropout, "encode": _encode}[state["op"]](state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["type"] == F32 else 2
    c = case["channels"]
    if case["op"] in ("norm", "dropout"):
        n = case["tokens"] * c
        if case["op"] == "dropout":
            return {"bytes": 4 * n * size, "flops": 2 * n}
        params = (4 if case["params"] == F32 else 2) * c
        if not case["back"]:
            return {"bytes": 2 * n * size + 2 * params, "flops": 8 * n}
        return {"bytes": 4 * n * size + 4 * params, "flops": 22 * n}      # x, grad -> y, dx
    tokens = case["batch"] * case["length"]
    n, table = tokens * c, case["rows"] * c
    index = (8 if case["index"] == "int64" else 4) * tokens
    used = min(table, n) * size                  # rows that can be read at all
    total = {"bytes": index + used + n * size, "flops": n}
    if case["op"] == "encode":
        params = (4 if case["params"] == F32 else 2) * c
        total["bytes"] += 2 * params
        total["flops"] += 8 * n
    if case["back"]:
        total["bytes"] += n * size + table * size
        total["flops"] += 2 * n
        if case.get("per_token"):
            total["bytes"] += 8 * tokens
            total["flops"] += 2 * n
        if case["op"] == "encode":
            total["bytes"] += 2 * params
            total["flops"] += 14 * min(n, table)
    return total


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def _times_32(m, x):
    """(high, low) 32-bit words of m x, by 16-bit pieces"""
    m1, m0 = m >> 16, m & 0xFFFF
    x1, x0 = x >> 16, x & 0xFFFF
    low, mid1, mid2, high = m0 * x0, m1 * x0, m0 * x1, m1 * x1
    mid = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
    return high + (mid1 >> 16) + (mid2 >> 16) + (mid >> 16), (low & 0xFFFF) + ((mid & 0xFFFF) << 16)


def _factors(start, n, p, seed, offset):
    """What elements start .. start + n - 1 (start a multiple of eight) are multiplied by."""
    word = torch.arange(start // 8, (start + n + 7) // 8, device="cuda")
    x0, x1 = word % (1 << 32), word // (1 << 32)
    x2, x3 = torch.full_like(word, offset % (1 << 32)), torch.full_like(word, offset // (1 << 32))
    key = [seed % (1 << 32), seed // (1 << 32)]
    for _ in range(10):
        h0, l0 = _times_32(0xD2511F53, x0)
        h1, l1 = _times_32(0xCD9E8D57, x2)
        x0, x1, x2, x3 = h1 ^ x1 ^ key[0], l1, h0 ^ x3 ^ key[1], l0
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    draws = torch.empty((word.numel(), 4, 2), device="cuda", dtype=torch.int64)
    for i, x in enumerate((x0, x1, x2, x3)):
        draws[:, i, 0], draws[:, i, 1] = x % 65536, x // 65536
    limit = int(round(p * 65536))
    return (draws.reshape(-1)[:n] >= limit).double() * (65536.0 / max(1, 65536 - limit))


def _exact_normed(x):
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + EPS)
    return (x - mean) / sd, sd


def _exact_norm_gradient(g, h, sd, w):
    q = g * w
    c = q.shape[1]
    return (q - (q.sum(1, keepdim=True) + h * (q * h).sum(1, keepdim=True)) / c) / sd


def exact(case, seed):
    s = prepare(case, seed)
    c = case["channels"]
    step = max(8, (1 << 24) // c // 8 * 8)       # rows taken at a time
    if case["op"] == "dropout":
        out = []
        for x in (s["x"], s["grad"]):
            y = torch.empty(x.numel(), device="cuda", dtype=torch.float64)
            for at in range(0, x.numel(), 1 << 24):
                part = x.reshape(-1)[at:at + (1 << 24)].double()
                y[at:at + (1 << 24)] = part * _factors(at, part.numel(), s["p"], s["seed"], s["offset"])
            out.append(y.view(x.shape))
        return out
    if case["op"] == "norm":
        w, b = s["weight"].double(), s["bias"].double()
        y, dx = (torch.empty(s["x"].shape, device="cuda", dtype=torch.float64) for _ in range(2))
        dw, db = torch.zeros_like(w), torch.zeros_like(b)
        for at in range(0, case["tokens"], step):
            h, sd = _exact_normed(s["x"][at:at + step].double())
            g = s["grad"][at:at + step].double()
            y[at:at + step] = torch.addcmul(b, h, w)
            dx[at:at + step] = _exact_norm_gradient(g, h, sd, w)
            dw += (g * h).sum(0)
            db += g.sum(0)
        return [y, dx, dw, db] if case["back"] else [y]
    encode = case["op"] == "encode"
    table = s["table"].double()
    at_row = torch.floor(s["tokens_in"].double().reshape(-1)).long()
    at_row = torch.where((at_row < 0) | (at_row >= case["rows"]), case["rows"], at_row)
    scale = s["scale"].double().reshape(-1) if torch.is_tensor(s["scale"]) else torch.full(
        at_row.shape, s["scale"], device="cuda", dtype=torch.float64)
    if encode:                                   # every token of a row has the same vector
        w, b = s["weight"].double(), s["bias"].double()
        h, sd = _exact_normed(table * s["scale"])
        table = torch.addcmul(b, h, w)
    table = torch.cat([table, torch.zeros_like(table[:1])])
    tokens = at_row.numel()
    grad = s["grad"].reshape(tokens, c)
    y = torch.empty((tokens, c), device="cuda", dtype=torch.float64)
    sums = torch.zeros_like(table)
    ds = torch.empty(tokens, device="cuda", dtype=torch.float64)
    for at in range(0, tokens, step):
        rows = at_row[at:at + step]
        g = grad[at:at + step].double()
        f = _factors(at * c, rows.numel() * c, s["p"], s["seed"], s["offset"]).view(g.shape) if encode \
            else scale[at:at + step, None]
        y[at:at + step] = table[rows] * f
        ds[at:at + step] = (g * table[rows]).sum(1)
        sums.index_add_(0, rows, g * f)
    out = [y.view(s["grad"].shape)]
    if not case["back"]:
        return out
    sums = sums[:-1]
    if encode:
        dx = _exact_norm_gradient(sums, h, sd, w)
        return out + [dx * s["scale"], (sums * h).sum(0), sums.sum(0)]
    return out + [sums] + ([ds.view(s["tokens_in"].shape)] if case["per_token"] else [])
