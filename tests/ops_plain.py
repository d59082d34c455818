"""The operators of panvram_amd.ops from their definitions, in 64 bits on the CPU, with bounds of what 32-bit arithmetic and
the outputs' rounding may be off by. The GPU tests compare with these."""
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # 2 ** -p of p significant bits
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}   # where rounding stops being relative
U = 2.0 ** -24


def inside(got, want, bound):
    """Asserts |got - want| <= bound everywhere, NaN and infinities at the same places."""
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN at other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    over = (got - want).abs() - (bound if isinstance(bound, torch.Tensor) else torch.full_like(want, bound))
    over = over[fine]
    assert not over.numel() or float(over.max()) <= 0, f"{float(over.max())} over the bound, at {int(over.argmax())} of {over.numel()}"


def rounded(want, dtype):
    """What storing `want` in dtype may add."""
    return want.abs() * UNIT[dtype] + TINY[dtype]


def scan(gate, value, state=None, reset=None, d_out=None, d_last=None):
    """{name: (value, bound before the output's rounding)} of the gated recurrence and its gradients. The bounds follow the
    rounding errors through the recurrence: sigmoid(g) and 1 - sigmoid(g) are taken as good to (8 + 2 |g|) last places (the
    exponential's argument is rounded after the scaling by log2(e)), each product and sum to one; a chunk's product of
    (1 - z) times its start is the same sum of relative errors as the steps one by one."""
    g, v = gate.double(), value.double()
    B, T, D = g.shape
    z, k = torch.sigmoid(g), torch.sigmoid(-g)
    c = (8 + 2 * g.abs().clamp(max=1e4)) * U
    first = state.double() if state is not None else g.new_zeros(B, D)
    cut = torch.zeros(B, T, dtype=torch.bool) if reset is None else reset.bool()
    h, e = first, torch.zeros_like(first)
    hs, es, before, eb = [], [], [], []
    for t in range(T):
        r = cut[:, t, None]
        h0, e0 = torch.where(r, torch.zeros_like(h), h), torch.where(r, torch.zeros_like(e), e)
        before.append(h0)
        eb.append(e0)
        x = z[:, t] * v[:, t]
        h = torch.where(r, x, k[:, t] * h0 + x)
        e = k[:, t] * e0 + c[:, t] * ((k[:, t] * h0).abs() + x.abs()) + 1e-37
        hs.append(h)
        es.append(e)
    out = {"out": (torch.stack(hs, 1), torch.stack(es, 1)), "last": (h, e)}
    if d_out is None:
        return out
    before, eb = torch.stack(before, 1), torch.stack(eb, 1)
    C = d_last.double() if d_last is not None else g.new_zeros(B, D)
    eC = torch.zeros_like(C)
    dv, dg, edv, edg = (torch.empty_like(g) for _ in range(4))
    for t in range(T - 1, -1, -1):
        G = d_out[:, t].double() + C
        eG = eC + U * G.abs()
        dv[:, t] = z[:, t] * G
        edv[:, t] = z[:, t] * eG + c[:, t] * dv[:, t].abs() + 1e-37
        diff = v[:, t] - before[:, t]
        ediff = eb[:, t] + U * diff.abs()
        dg[:, t] = z[:, t] * k[:, t] * G * diff
        edg[:, t] = z[:, t] * k[:, t] * (eG * diff.abs() + G.abs() * ediff) + 2 * c[:, t] * dg[:, t].abs() + 1e-37
        r = cut[:, t, None]
        flow = k[:, t] * G
        C = torch.where(r, torch.zeros_like(C), flow)
        eC = torch.where(r, torch.zeros_like(C), k[:, t] * eG + c[:, t] * flow.abs() + 1e-37)
    return out | {"d_gate": (dg, edg), "d_value": (dv, edv), "d_state": (C, eC)}


def norm(stream, weight, eps, d_y=None, d_stream=None):
    """{name: (value, bound)} of the norm of the stored stream [N, D] and its gradients. Sums of D squares are taken as good to
    D / 64 + 16 last places: 64 lanes, or more, sum side by side."""
    s, w = stream.double(), weight.double()
    D = s.shape[1]
    c = (D / 64 + 16) * U
    r = 1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps)
    u = s * r
    y = u * w
    out = {"y": (y, c * y.abs())}
    if d_y is None:
        return out
    d_y, ds = d_y.double(), d_stream.double() if d_stream is not None else torch.zeros_like(s)
    g = d_y * w
    m = (g * u).mean(-1, keepdim=True)
    d = ds + r * (g - u * m)
    e = U * (ds.abs() + d.abs()) + 3 * c * r * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    each = (d_y * u)
    return out | {"d": (d, e), "d_weight": (each.sum(0), ((s.shape[0] + 16) * U + c) * each.abs().sum(0) + 1e-37)}


def loss(hidden, weight, tokens, ignore, factor=None, scale=1.0):
    """{name: (value, bound)} of the next token's cross-entropy and its gradients: `each`, `loss`, and of scale * loss, or of
    sum factor * each, `d_hidden`, `d_weight`. Products over D are taken as good to D / 16 + 16 last places of the sum of
    absolute values; where weight has 16 bits, the gradients of the logits as held to 16 bits in the products after them."""
    B, T, D = hidden.shape
    V = weight.shape[0]
    w = weight.double()
    t = torch.full((B, T), -1, dtype=torch.int64)
    t[:, :-1] = tokens[:, 1:].long()
    counts = (t >= 0) & (t < V) & (t != (-1 if ignore is None else ignore))
    h = torch.where(counts[..., None], hidden.double(), torch.zeros(()).double())
    logits = h @ w.T
    off = (D / 16 + 16) * U * (h.abs() @ w.abs().T).amax(-1)                 # of any logit
    lse = torch.logsumexp(logits, -1)
    own = logits.gather(-1, torch.where(counts, t, 0)[..., None])[..., 0]
    zero = torch.zeros_like(lse)
    each = torch.where(counts, lse - own, zero)
    e_each = torch.where(counts, 2 * off + (V + 8) * U * (1 + lse.abs() + own.abs()), zero)
    n = max(1, int(counts.sum()))
    out = {"each": (each, e_each), "loss": (each.sum() / n, e_each.sum() / n + 4 * U * each.sum() / n)}
    f = factor.double() if factor is not None else torch.full((B, T), scale / n, dtype=torch.float64)
    f = torch.where(counts, f, zero)[..., None]
    p = torch.softmax(logits, -1)
    hot = torch.nn.functional.one_hot(torch.where(counts, t, 0), V).double()
    dl = (p - hot) * f
    e_dl = f.abs() * (p * (2 * off[..., None] + (V + 16) * U) + 4 * U * (p - hot).abs()) + 1e-37 * (f != 0)
    half = 2.0 ** -16 if weight.dtype != torch.float32 else 0.0
    d_hidden = dl @ w
    e_dh = e_dl @ w.abs() + ((V + 8) * U + half) * (dl.abs() @ w.abs())
    flat = lambda x: x.reshape(B * T, -1)  # noqa: E731
    d_weight = flat(dl).T @ flat(h)
    e_dw = flat(e_dl).T @ flat(h).abs() + ((n + 64) * U + half) * (flat(dl).abs().T @ flat(h).abs())
    return out | {"d_hidden": (d_hidden, e_dh), "d_weight": (d_weight, e_dw)}
