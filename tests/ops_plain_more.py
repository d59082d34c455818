"""The operators of a model with matrices as its states from their definitions, in 64 bits on the CPU, with bounds of what 32-bit
arithmetic may be off by before the outputs' rounding. The GPU tests compare with these."""
import numpy as np
import torch

from tests.ops_plain import U


def words(counter, key):
    """The generator's four words of a counter of four (arrays of) 32-bit words under a key of two, as uint64."""
    m = np.uint64(0xFFFFFFFF)
    a, b, c, d = (np.asarray(x, dtype=np.uint64) & m for x in counter)
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    for _ in range(10):
        x, y = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (y >> np.uint64(32)) ^ b ^ k0, y & m, (x >> np.uint64(32)) ^ d ^ k1, x & m
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & m, (k1 + np.uint64(0xBB67AE85)) & m
    return a, b, c, d


def kept(n, p, seed, site=0, first=0):
    """(bool [n]: which of the elements from index `first` on are kept, the factor of those)"""
    seed %= 1 << 64
    index = np.arange(first, first + n, dtype=np.uint64)
    block = index >> np.uint64(3)
    w = np.stack(words((block, block >> np.uint64(32), np.full_like(block, site), np.zeros_like(block)), (seed & 0xFFFFFFFF, seed >> 32)))
    half = w[(index >> np.uint64(1)) & np.uint64(3), np.arange(n)] >> (np.uint64(16) * (index & np.uint64(1))) & np.uint64(0xFFFF)
    least = int(p * 65536 + 0.5)
    return torch.from_numpy(half >= np.uint64(least)), 65536 / (65536 - least) if least < 65536 else 0.0


def layer(stream, weight, bias, eps, d_y=None, d_stream=None):
    """{name: (value, bound)} of the layer norm of the stored stream [N, D] and its gradients. Sums over D are taken as good to
    D / 64 + 16 last places (lanes sum side by side): that is c. The first mean is off by c mean|s| at most; what the third sum
    leaves of that is c of the distances' own size."""
    s, w = stream.double(), weight.double()
    b = bias.double() if bias is not None else torch.zeros_like(w)
    D = s.shape[1]
    c = (D / 64 + 16) * U
    mean = s.mean(-1, keepdim=True)
    d = s - mean
    var = d.square().mean(-1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    off = c * s.abs().mean(-1, keepdim=True)                     # of the first mean
    e_d = 3 * U * d.abs() + U * off + c * (d.abs().mean(-1, keepdim=True) + off)
    rel = 0.5 * c * (var + 2 * off.square()) / (var + eps) + 4 * U     # of r
    u = d * r
    e_u = r * e_d + u.abs() * rel
    y = u * w + b
    out = {"y": (y, w.abs() * (e_u + 2 * U * u.abs()) + U * y.abs())}
    if d_y is None:
        return out
    d_y, ds = d_y.double(), d_stream.double() if d_stream is not None else torch.zeros_like(s)
    g = d_y * w
    mean_of = lambda x: x.mean(-1, keepdim=True)  # noqa: E731
    inner = g - mean_of(g) - u * mean_of(g * u)
    d = ds + r * inner
    size = g.abs() + mean_of(g.abs()) + u.abs() * mean_of((g * u).abs())
    e = U * (ds.abs() + d.abs()) + r * ((2 * c + rel) * size + e_u * mean_of((g * u).abs()) + u.abs() * mean_of(g.abs() * e_u))
    N = s.shape[0]
    return out | {"d": (d, e), "d_weight": ((d_y * u).sum(0), (N + 16) * U * (d_y * u).abs().sum(0) + (d_y.abs() * e_u).sum(0) + 1e-37),
                  "d_bias": (d_y.sum(0), (N + 16) * U * d_y.abs().sum(0))}
