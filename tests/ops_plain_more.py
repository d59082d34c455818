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


def delta(query, key, value, gate, write, state=None, reset=None, eps=1e-6):
    """(out, last) of the gated delta rule step by step, in the tensors' own precision; autograd gives its gradients."""
    B, T, H, K = query.shape
    G, V = value.shape[2:]
    unit = lambda x: (x / torch.sqrt(x.square().sum(-1, keepdim=True) + eps)).repeat_interleave(G // H, 2)  # noqa: E731
    q, k = unit(query), unit(key)
    keep, rate = torch.sigmoid(-gate), torch.sigmoid(write)
    S = state if state is not None else query.new_zeros(B, G, K, V)
    outs = []
    for t in range(T):
        S = keep[:, t, :, None, None] * S
        if reset is not None:
            S = torch.where(reset[:, t, None, None, None].bool(), torch.zeros_like(S), S)
        u = rate[:, t, :, None] * (value[:, t] - (k[:, t, :, None] @ S)[:, :, 0])
        S = S + k[:, t, :, :, None] * u[:, :, None]
        outs.append((q[:, t, :, None] @ S)[:, :, 0])
    return torch.stack(outs, 1), S


def delta_off(name, dtype):
    """How far, in the 2-norm and relative to it, a result of the gated delta rule may be off, without its own rounding. What is
    made in 32 bits is a chain of four sums of 256 terms at most (over a key, and over the steps of a chunk twice), each good to
    as many last places, and four of them more backwards. For tensors of 16 bits its operands have 22 bits, or 11 where they
    reach 16-bit outputs only: four such roundings each way, of half a unit of 2^-22 or 2^-11."""
    sums = (8 if name.startswith("d_") else 4) * 256 * U
    if dtype == torch.float32:
        return sums
    wide = 8 * 2.0 ** -23
    return sums + wide + (0.0 if name in ("last", "d_state", "d_value") else 8 * 2.0 ** -12)


def near(got, want, off, dtype):
    """Asserts that `got` is within `off` and half a step of `dtype` of `want` in the 2-norm, and no element off by over 32 times that
    of its own size or of the tensor's typical one (of terms that cancel to its size, about 1,000 as large)."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    off = off + {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    norm, size = float(want.norm()), want.numel()
    if not norm:
        assert float(got.abs().max()) == 0.0 if size else True
        return
    d = (got - want).abs()
    # (what lies below float32's smallest numbers, 2^-126, as after a step that keeps e^-120 = 2^-173, is 0 there)
    assert float(d.norm()) <= off * norm + 2.0 ** -126 * size ** 0.5, f"{float(d.norm()) / norm} off, {off} allowed"
    over = d - 2.0 ** -126 - 32 * off * torch.maximum(want.abs(), torch.full_like(want, norm / size ** 0.5))
    assert float(over.max()) <= 0, f"{float(d.max())} off at {int(over.argmax())}, typical {norm / size ** 0.5}"
