"""Plain 64-bit forms of the learned type vectors' operators in numpy, and how far a computation in
32 bits with one rounding at the end may be from them.

Bounds: u = 2^-24 is half a step of float32 at 1.  A sum of k terms in 32 bits, in whatever order,
is off by at most k u times the sum of the terms' magnitudes (first order; 2 % are added for the
higher ones); a row's sums run over several lanes, at most `depth(channels)` additions behind one
another.  Errors of one step go into the next one with that step's derivative.  What is stored is
rounded to its type once more: half a step of it, or half of its smallest subnormal step."""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half of the smallest step: float16 has subnormals of 2^-24, the others reach far below what the
# tests compare
SMALLEST = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def depth(channels):
    """Additions behind one another in a sum over a row's channels: at least four lanes share a row
    of more than 16 channels."""
    return min(channels, channels // 4 + 16) + 1


def f64(t):
    return t.detach().cpu().double().numpy()


def check(got, ref, bound, dtype, what=""):
    """got (tensor of dtype) against the 64-bit values and the bound of what was rounded to it."""
    assert got.dtype == dtype and tuple(got.shape) == ref.shape, (what, got.dtype, got.shape, ref.shape)
    g = f64(got)
    allowed = 1.02 * bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * np.abs(ref) + SMALLEST[dtype]
    off = np.abs(g - ref)
    bad = ~(off <= allowed)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, off / allowed, 0)), ref.shape)
        raise AssertionError("%s: %d of %d values beyond their bound; at %s: got %r, expected %r +- %g"
                             % (what, int(bad.sum()), ref.size, at, g[at], ref[at], allowed[at]))


def rows_of(type_index, nrows):
    """Row of every index, -1 where it names none."""
    t = f64(type_index).reshape(-1) if type_index.is_floating_point() else \
        type_index.cpu().numpy().reshape(-1).astype(object)
    out = np.full(t.shape, -1, np.int64)
    for i, v in enumerate(t):
        if v == v and 0 <= v < nrows:
            out[i] = int(np.floor(v)) if isinstance(v, float) else int(v)
    return out


def take(table, rows):
    picked = np.zeros((len(rows), table.shape[1]))
    named = rows >= 0
    picked[named] = table[rows[named]]
    return picked


def embed(rows, table, scale):
    """scale: a number or one per token. (values, bound)"""
    y = take(table, rows) * np.reshape(np.broadcast_to(scale, rows.shape), (-1, 1))
    return y, U * np.abs(y)                      # one product


def sum_by_row(rows, terms, magnitudes, nrows, roundings):
    """Sums of the tokens' terms by row, of which each went through `roundings` roundings before."""
    out = np.zeros((nrows, terms.shape[1]))
    size = np.zeros_like(out)
    named = rows >= 0
    np.add.at(out, rows[named], terms[named])
    np.add.at(size, rows[named], magnitudes[named])
    count = np.bincount(rows[named], minlength=nrows)[:, None]
    return out, U * (count + roundings) * size


def embed_backward(rows, grad, table, scale):
    """((gradient of the table, bound), (gradient of a per-token scale, bound))"""
    terms = grad * np.reshape(np.broadcast_to(scale, rows.shape), (-1, 1))
    to_table = sum_by_row(rows, terms, np.abs(terms), table.shape[0], 2)
    products = grad * take(table, rows)
    c = table.shape[1]
    return to_table, (products.sum(1), U * (depth(c) + 1) * np.abs(products).sum(1))


class Norm(object):
    """Statistics of the rows of x (n, c) and their bounds; `given` is the error that x itself has."""

    def __init__(self, x, eps, given=0.0):
        c = x.shape[1]
        k = depth(c)
        self.eps = float(np.float32(eps))
        self.mean = x.mean(1, keepdims=True)
        self.d_mean = U * (k + 1) * np.abs(x).mean(1, keepdims=True) + np.mean(given + 0 * x, 1, keepdims=True)
        d = x - self.mean
        d_d = given + self.d_mean + U * np.abs(d)
        var = (d * d).mean(1, keepdims=True)
        # the differences of a row are off by d_mean alike (and by their own rounding), the squares'
        # mean by twice their product and its square
        d_var = (2 * np.abs(d) * d_d + d_d * d_d).mean(1, keepdims=True) + U * (k + 2) * var
        self.rstd = 1 / np.sqrt(var + self.eps)
        # sqrt falls by at most what the derivative at the lower end says
        low = np.maximum(var + self.eps - d_var, (var + self.eps) / 4)
        self.d_rstd = self.rstd * (0.5 * d_var / low + 4 * U)
        self.h = d * self.rstd
        self.d_h = d_d * self.rstd + np.abs(d) * self.d_rstd + d_d * self.d_rstd + U * np.abs(self.h)
        self.k, self.c = k, c

    def forward(self, weight, bias):
        y = self.h * weight + bias
        return y, self.d_h * np.abs(weight) + 2 * U * (np.abs(self.h * weight) + np.abs(bias))

    def backward(self, grad, weight, d_grad=0.0):
        """(of x, of weight, of bias), each with its bound; d_grad: the error of the gradient."""
        grad_size = np.abs(grad)
        q = grad * weight
        d_q = d_grad * np.abs(weight) + U * np.abs(q)
        mean_q = q.mean(1, keepdims=True)
        d_mean_q = d_q.mean(1, keepdims=True) + U * (self.k + 1) * np.abs(q).mean(1, keepdims=True)
        qh = q * self.h
        mean_qh = qh.mean(1, keepdims=True)
        d_mean_qh = ((d_q * (np.abs(self.h) + self.d_h) + np.abs(q) * self.d_h).mean(1, keepdims=True) +
                     U * (self.k + 2) * np.abs(qh).mean(1, keepdims=True))
        inner = q - mean_q - self.h * mean_qh
        d_inner = (d_q + d_mean_q + np.abs(self.h) * d_mean_qh + self.d_h * (np.abs(mean_qh) + d_mean_qh) +
                   3 * U * (np.abs(q) + np.abs(mean_q) + np.abs(self.h * mean_qh)))
        dx = self.rstd * inner
        d_dx = self.rstd * d_inner + self.d_rstd * (np.abs(inner) + d_inner) + 2 * U * np.abs(dx)
        n = grad.shape[0]
        gh = grad * self.h
        dw, db = gh.sum(0), grad.sum(0)
        d_gh = d_grad * (np.abs(self.h) + self.d_h) + grad_size * self.d_h
        d_dw = d_gh.sum(0) + U * (n + 2) * np.abs(gh).sum(0)
        d_db = (d_grad + 0 * grad_size).sum(0) + U * (n + 1) * grad_size.sum(0)
        return (dx, d_dx), (dw, d_dw), (db, d_db)


def philox(counters, offset, seed):
    """The four words of Philox4x32-10 for counters (low, high 64 bits) = (counters, offset)."""
    m32 = np.uint64(0xFFFFFFFF)
    low = np.asarray(counters, np.uint64)
    c = [low & m32, low >> np.uint64(32), np.full_like(low, offset & 0xFFFFFFFF),
         np.full_like(low, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & m32,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def kept(n, p, seed, offset):
    """(which of n elements are kept, the factor of the kept ones)"""
    limit = int(np.floor(p * 65536 + 0.5))
    words = philox(np.arange((n + 7) // 8), offset, seed)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[:n]
    return halves >= limit, 65536.0 / (65536 - limit) if limit < 65536 else 0.0


def dropout(x, p, seed, offset):
    """(values, bound): the factor is rounded and multiplied with; what is dropped is zero"""
    keep, factor = kept(x.size, p, seed, offset)
    y = np.where(keep.reshape(x.shape), x * factor, 0.0)
    return y, np.where(keep.reshape(x.shape), 2 * U * np.abs(y), 0.0)


def encode(rows, table, scale, weight, bias, eps, p, seed, offset):
    scale = float(np.float32(scale))
    x = take(table, rows) * scale
    norm = Norm(x, eps, U * np.abs(x))
    y, d = norm.forward(weight, bias)
    y, d = y * (rows >= 0)[:, None], d * (rows >= 0)[:, None]
    keep, factor = kept(y.size, p, seed, offset)
    keep = keep.reshape(y.shape)
    y = np.where(keep, y * factor, 0.0)
    return y, np.where(keep, d * factor + 2 * U * np.abs(y), 0.0)


def encode_backward(rows, grad, table, scale, weight, eps, p, seed, offset):
    """(of the table, of weight, of bias) with their bounds"""
    scale = float(np.float32(scale))
    g, _ = dropout(grad, p, seed, offset)
    sums, d_sums = sum_by_row(rows, g, np.abs(g), table.shape[0], 3)
    x = table * scale
    norm = Norm(x, eps, U * np.abs(x))
    (dx, d_dx), dw, db = norm.backward(sums, weight, d_sums)
    return (dx * scale, abs(scale) * (d_dx + 2 * U * np.abs(dx))), dw, db
