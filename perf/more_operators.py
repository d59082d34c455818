"""The operators of a model with matrices as its states, in their plain forms and as the package's calls.

  delta    panvram_amd.ops.gated_delta: a state S [K, V] for each head, S[t] = a S[t-1] + k u^T with a = 1 - sigmoid(gate),
           u = sigmoid(write) (v - a S[t-1]^T k), and out = S[t]^T q, of keys and queries divided by their length; from a state
           or from zero; a reset at t drops S[t-1]; several value heads may share a query and key head; its gradients
  layer    panvram_amd.ops.add_layer_norm: the residual stream s = residual + dropout(x), stored in its type, and
           (s - mean) / sqrt(var + eps) * weight + bias; its gradients
  dropout  panvram_amd.ops.dropout: each element by its own 16 bits of a counter-based generator; its gradient

They are a block of such a model with what stands around it; the forms of one token are generation's.
"""
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_UNIT_EPS = 1e-6
_NORM_EPS = 1e-5
_CHUNK = 64


def listed():
    return [
        # generation: one base for each of 64 sequences, the states carried from call to call
        {"name": "delta_step_64x8x128", "op": "delta", "B": 64, "T": 1, "H": 8, "G": 8, "K": 128, "V": 128, "dtype": "bfloat16", "state": True},
        # a training step's layer on a batch of the headline's window length, read from one projection
        {"name": "delta_train_8x8192x8x128", "op": "delta", "B": 8, "T": 8192, "H": 8, "G": 8, "K": 128, "V": 128, "dtype": "bfloat16", "train": True, "joined": True},
        # a small model in full precision: odd sizes, two value heads to a key head, packed windows, a carried state
        {"name": "delta_train_3x1025x3x48", "op": "delta", "B": 3, "T": 1025, "H": 3, "G": 6, "K": 48, "V": 80, "dtype": "float32", "train": True, "state": True, "reset": True},
        # a slice of 2^17 bases of one haplotype through a layer at inference: few heads, a long sequence
        {"name": "delta_1x131072x4x128", "op": "delta", "B": 1, "T": 1 << 17, "H": 4, "G": 4, "K": 128, "V": 128, "dtype": "bfloat16", "state": True},
        # generation: the norm of 16 rows, where only latency counts
        {"name": "layer_16x1024", "op": "layer", "N": 16, "D": 1024, "dtype": "bfloat16"},
        # the norm of the training step above with its branch's dropout, forward and backward
        {"name": "layer_train_65536x1024", "op": "layer", "N": 65536, "D": 1024, "dtype": "bfloat16", "train": True, "p": 0.1},
        # the small model's, in full precision and without dropout
        {"name": "layer_train_10245x500", "op": "layer", "N": 10245, "D": 500, "dtype": "float32", "train": True},
        # long windows of a wide model, scored
        {"name": "layer_32768x4096", "op": "layer", "N": 32768, "D": 4096, "dtype": "float16"},
        # dropout of the training step's embeddings, forward and backward
        {"name": "dropout_train_65536x1024", "op": "dropout", "N": 65536, "D": 1024, "dtype": "bfloat16", "p": 0.1, "train": True},
        # the small model's
        {"name": "dropout_train_10245x500", "op": "dropout", "N": 10245, "D": 500, "dtype": "float32", "p": 0.25, "train": True},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["delta", "delta", "layer", "dropout"])
    case = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if op == "delta":
        train = rng.random() < 0.5
        case["T"] = 1 if rng.random() < 0.2 else _log(rng, 2, 8192 if train else 1 << 17)
        case |= {"K": _log(rng, 16, 128), "V": _log(rng, 16, 128), "H": _log(rng, 1, 16)}
        case["G"] = case["H"] * rng.choice([1, 1, 2, 3])
        most = (1 << (26 if train else 27)) // (case["T"] * case["G"] * (case["K"] + case["V"]))
        if case["T"] == 1:
            most = (1 << 24) // (case["G"] * case["K"] * case["V"])
        case["B"] = _log(rng, 1, max(1, min(64, most)))
        for flag in ("state", "reset", "joined"):
            if rng.random() < 0.4:
                case[flag] = True
        if train:
            case["train"] = True
        return case
    case["D"] = _log(rng, 64, 8192)
    case["N"] = _log(rng, 1, (1 << 26) // case["D"])
    if op == "dropout" or rng.random() < 0.5:
        case["p"] = round(rng.uniform(0.02, 0.5), 3)
    if rng.random() < 0.6:
        case["train"] = True
    return case


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = dict(case)

    def normal(*shape, mean=0.0, std=1.0, kind=dtype):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(std).add_(mean).to(kind)

    if case["op"] == "delta":
        B, T, H, G, K, V = (case[k] for k in "BTHGKV")
        # keys and queries of one sign more often than not, as an activation leaves them: neighbouring keys are alike
        if case.get("joined"):
            both = normal(B, T, 2 * H * K + G * V, mean=0.3)
            q, k, v = both.split([H * K, H * K, G * V], -1)
            s["query"], s["key"], s["value"] = q.unflatten(-1, (H, K)).detach(), k.unflatten(-1, (H, K)).detach(), v.unflatten(-1, (G, V)).detach()
        else:
            s["query"], s["key"], s["value"] = normal(B, T, H, K, mean=0.3), normal(B, T, H, K, mean=0.3), normal(B, T, G, V)
        # gates that keep most of the state from base to base
        s["gate"], s["write"] = normal(B, T, G, mean=-4.0, std=1.5), normal(B, T, G)
        s["state"] = normal(B, G, K, V, std=0.3, kind=torch.float32) if case.get("state") else None
        s["reset"] = None
        if case.get("reset"):
            s["reset"] = torch.rand(B, T, generator=gen, device=dev) < 2.0 / T
        if case.get("train"):
            s["d_out"] = normal(B, T, G, V, std=0.01)
            s["wanted"] = [t.requires_grad_() for t in (s["query"], s["key"], s["value"], s["gate"], s["write"], s["state"]) if t is not None]
        return s
    N, D = case["N"], case["D"]
    s["seed"] = torch.randint(1 << 62, (1,), generator=gen, device=dev)
    s["x"] = normal(N, D, std=0.5)
    if case["op"] == "layer":
        s["residual"] = normal(N, D, mean=0.2, std=2.0)
        s["weight"], s["bias"] = normal(D, mean=1.0, std=0.2, kind=torch.float32), normal(D, std=0.2, kind=torch.float32)
        if case.get("train"):
            s["d_y"], s["d_stream"] = normal(N, D, std=0.01), normal(N, D, std=0.01)
            s["wanted"] = [t.requires_grad_() for t in (s["x"], s["residual"], s["weight"], s["bias"])]
    elif case.get("train"):
        s["d_y"] = normal(N, D, std=0.01)
        s["x"].requires_grad_()
    return s


# ---- the plain forms: elementary torch operations in 32 bits, rounded once


def _unit(x):
    """(x over its length, 1 over its length)"""
    r = torch.rsqrt((x * x).sum(-1, keepdim=True) + _UNIT_EPS)
    return x * r, r


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular A [..., C, C], C a power of two: blocks of two inverted ones, doubling."""
    C = A.shape[-1]
    inv = torch.eye(C, device=A.device).expand(A.shape).clone()
    n = 1
    while n < C:
        # the diagonal's blocks of 2 n: [..., blocks, 2 n, 2 n]
        a, t = (X.unflatten(-1, (-1, 2 * n)).unflatten(-3, (-1, 2 * n)).diagonal(dim1=-4, dim2=-2).movedim(-1, -3) for X in (A, inv))
        t[..., n:, :n] = -(t[..., n:, n:] @ a[..., n:, :n] @ t[..., :n, :n])
        n *= 2
    return inv


def _chunks(x, T, C):
    """[B, T, G, ...] -> [chunks, B, G, C, ...] in 32 bits, zeros behind the last step"""
    pad = -T % C
    x = x.movedim(2, 1).float()
    if pad:
        x = torch.cat([x, x.new_zeros(*x.shape[:2], pad, *x.shape[3:])], 2)
    return x.unflatten(2, (-1, C)).movedim(2, 0)


@torch.no_grad()
def _delta_plain(s):
    """Chunks of 64 steps, or of the few that there are, as matrix products. With c(i) the sum of the logarithms of a in a chunk, M[i, j] = exp(c(i) - c(j)),
    g(i) = exp(c(i)) and l(i) = exp(c(last) - c(i)), each zero across a reset, and S the state before the chunk:
    D = v - g k S; (I + b M k k^T) U = b D; out = g q S + (M q k^T) U; the state after it: g(last) S + (l k)^T U."""
    dtype = s["query"].dtype
    B, T, H, G, K, V = (s[k] for k in "BTHGKV")
    C, share, dev = min(_CHUNK, 1 << (T - 1).bit_length()), G // H, s["query"].device
    q_raw, k_raw = s["query"].float(), s["key"].float()
    (q1, rq), (k1, rk) = _unit(q_raw), _unit(k_raw)
    q, k, v = _chunks(q1.repeat_interleave(share, 2), T, C), _chunks(k1.repeat_interleave(share, 2), T, C), _chunks(s["value"], T, C)
    n = q.shape[0]
    b = _chunks(torch.sigmoid(s["write"].float()), T, C)
    log_a = -torch.nn.functional.softplus(s["gate"].double())
    log_a = torch.cat([log_a, log_a.new_zeros(B, n * C - T, G)], 1)
    cut = torch.zeros(B, n * C, dtype=torch.bool, device=dev)
    if s["reset"] is not None:
        cut[:, :T] = s["reset"]
    log_a = log_a.masked_fill(cut[..., None], 0.0).movedim(2, 1).unflatten(2, (n, C)).movedim(2, 0)        # [n, B, G, C]
    segment = cut.unflatten(1, (n, C)).movedim(1, 0).cumsum(-1)[:, :, None]                                    # [n, B, 1, C]
    c = log_a.cumsum(-1)
    lower = torch.ones(C, C, dtype=torch.bool, device=dev).tril()
    M = (c[..., :, None] - c[..., None, :]).masked_fill(~(lower & (segment[..., :, None] == segment[..., None, :])), -torch.inf).exp().float()
    g = c.masked_fill(segment != 0, -torch.inf).exp().float()
    l = (c[..., -1:] - c).masked_fill(segment != segment[..., -1:], -torch.inf).exp().float()
    kk = k @ k.mT
    P = (q @ k.mT) * M
    inv = _inverse((b[..., None] * M * kk).tril(-1))
    end = g[..., -1, None, None]
    S = s["state"].clone() if s["state"] is not None else torch.zeros(B, G, K, V, device=dev)
    starts, rests = [], []
    for i in range(n):
        rest = v[i] - g[i, ..., None] * (k[i] @ S)
        U = inv[i] @ (b[i, ..., None] * rest)
        starts.append(S)
        rests.append(rest)
        S = end[i] * S + (l[i, ..., None] * k[i]).mT @ U
    starts, rests = torch.stack(starts), torch.stack(rests)
    U = inv @ (b[..., None] * rests)
    out = g[..., None] * (q @ starts) + P @ U
    back = lambda x, shape: x.movedim(0, 2).flatten(2, 3)[:, :, :T].movedim(1, 2).reshape(shape)  # noqa: E731
    result = {"out": back(out, (B, T, G, V)).to(dtype), "last": S}
    if not s.get("train"):
        return result
    dO = _chunks(s["d_out"], T, C)
    straight = P.mT @ dO
    dS = torch.zeros_like(S)
    ends, d_rests = [None] * n, [None] * n
    for i in range(n - 1, -1, -1):
        ends[i] = dS
        d_rests[i] = inv[i].mT @ (straight[i] + l[i, ..., None] * (k[i] @ dS))
        dS = end[i] * dS + (g[i, ..., None] * q[i]).mT @ dO[i] - ((b[i] * g[i])[..., None] * k[i]).mT @ d_rests[i]
    ends, dR = torch.stack(ends), torch.stack(d_rests)
    E = (dO @ U.mT) * M
    F = -(dR @ U.mT) * (M.tril(-1))
    Fb = F * b[..., None]
    from_q, from_k, to_k = dO @ starts.mT, dR @ starts.mT, U @ ends.mT
    dq = g[..., None] * from_q + E @ k
    dk = l[..., None] * to_k - (b * g)[..., None] * from_k + E.mT @ q + (Fb + Fb.mT) @ k
    db = (dR * rests).sum(-1) + (F * kk).sum(-1)
    # the logarithm of a at t: pairs j < t <= i, what reaches i >= t from the state, what j < t leaves behind, and the state itself
    pairs = E * (q @ k.mT) + Fb * kk
    rows = pairs.sum(-1) + g * ((q * from_q).sum(-1) - b * (k * from_k).sum(-1))
    left = l * (k * to_k).sum(-1)
    one = segment[..., None, :] == segment[..., :, None]
    # sums over the steps of t's own piece between resets: from t on for rows, before t for columns and what is left behind
    after = (lower.T & one).float()
    before = (lower.tril(-1) & one).float()
    d_log = (after @ rows[..., None])[..., 0] - (after @ pairs.sum(-2)[..., None])[..., 0] + (before @ (left * (segment == segment[..., -1:]))[..., None])[..., 0]
    whole = (end * ends * starts).sum((-2, -1))
    d_log = d_log + whole[..., None] * (segment == 0)
    d_log = back(d_log, (B, T, G))
    z, keep = torch.sigmoid(s["gate"].float()), torch.sigmoid(-s["gate"].float())
    d_gate = -z * d_log
    if s["reset"] is not None:
        d_gate = d_gate.masked_fill(s["reset"][..., None], 0.0)
    w = s["write"].float()
    shared = lambda x: back(x, (B, T, H, share, K)).sum(3)  # noqa: E731
    dq, dk = shared(dq), shared(dk)
    result["d_query"] = (rq * (dq - q1 * (q1 * dq).sum(-1, keepdim=True))).to(dtype)
    result["d_key"] = (rk * (dk - k1 * (k1 * dk).sum(-1, keepdim=True))).to(dtype)
    result["d_value"] = back(b[..., None] * dR, (B, T, G, V)).to(dtype)
    result["d_gate"] = d_gate.to(dtype)
    result["d_write"] = (back(db, (B, T, G)) * torch.sigmoid(w) * torch.sigmoid(-w)).to(dtype)
    if s["state"] is not None:
        result["d_state"] = dS
    return result


def _kept(seed, n, p, site=0):
    """(truth values of n elements, the factor of those kept): element i is dropped where its 16 bits are below p 2^16. The bits
    are those of the ten-round generator of four 32-bit words by Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as
    easy as 1, 2, 3", 2011), of key `seed` and counter (i / 8, site): eight elements to a counter, low half of a word first."""
    low = 0xFFFFFFFF
    at = torch.arange(-(-n // 8), device=seed.device, dtype=torch.int64)
    w = [at & low, at >> 32, torch.full_like(at, site), torch.zeros_like(at)]
    key = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        a, b = w[0] * 0xD2511F53, w[2] * 0xCD9E8D57        # (products of 64 bits, wrapped as such)
        w = [((b >> 32) & low) ^ w[1] ^ key[0], b & low, ((a >> 32) & low) ^ w[3] ^ key[1], a & low]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    bits = torch.stack([h for x in w for h in (x & 0xFFFF, x >> 16)], -1).flatten()[:n]
    least = int(p * 65536 + 0.5)
    return bits >= least, 65536 / (65536 - least)


@torch.no_grad()
def _layer_plain(s):
    dtype, w = s["x"].dtype, s["weight"]
    x = s["x"].float()
    kept = None
    if s.get("p"):
        kept, up = _kept(s["seed"], x.numel(), s["p"])
        kept = kept.view(x.shape)
        x = torch.where(kept, x * up, torch.zeros_like(x))
    stream = (x + s["residual"].float()).to(dtype)                # the stream as the next layer reads it
    f = stream.float()
    f = f - f.mean(-1, keepdim=True)
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + _NORM_EPS)
    unit = f * r
    out = {"y": (unit * w + s["bias"]).to(dtype), "stream": stream}
    if s.get("train"):
        d_y = s["d_y"].float()
        g = d_y * w
        d = s["d_stream"].float() + r * (g - g.mean(-1, keepdim=True) - unit * (g * unit).mean(-1, keepdim=True))
        out["d_x"] = (d if kept is None else torch.where(kept, d * up, torch.zeros_like(d))).to(dtype)
        out["d_residual"] = d.to(dtype)
        out["d_weight"] = (d_y * unit).sum(0)
        out["d_bias"] = d_y.sum(0)
    return out


@torch.no_grad()
def _dropout_plain(s):
    dtype = s["x"].dtype
    kept, up = _kept(s["seed"], s["x"].numel(), s["p"])
    kept = kept.view(s["x"].shape)
    drop = lambda t: torch.where(kept, t.float() * up, torch.zeros((), device=t.device)).to(dtype)  # noqa: E731
    out = {"y": drop(s["x"])}
    if s.get("train"):
        out["d_x"] = drop(s["d_y"])
    return out


# ---- the package's calls


def _delta_own(s):
    from panvram_amd import ops
    out, last = ops.gated_delta(s["query"], s["key"], s["value"], s["gate"], s["write"], state=s["state"], reset=s["reset"], eps=_UNIT_EPS)
    result = {"out": out, "last": last}
    if s.get("train"):
        d = torch.autograd.grad(out, s["wanted"], s["d_out"])
        result |= zip(("d_query", "d_key", "d_value", "d_gate", "d_write", "d_state"), d)
    return result


def _layer_own(s):
    from panvram_amd import ops
    y, stream = ops.add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], eps=_NORM_EPS, dropout=s.get("p", 0.0), seed=s["seed"] if s.get("p") else None)
    out = {"y": y, "stream": stream}
    if s.get("train"):
        out |= zip(("d_x", "d_residual", "d_weight", "d_bias"), torch.autograd.grad((y, stream), s["wanted"], (s["d_y"], s["d_stream"])))
    return out


def _dropout_own(s):
    from panvram_amd import ops
    y = ops.dropout(s["x"], s["p"], s["seed"])
    out = {"y": y}
    if s.get("train"):
        (out["d_x"],) = torch.autograd.grad(y, (s["x"],), s["d_y"])
    return out


_PLAIN = {"delta": _delta_plain, "layer": _layer_plain, "dropout": _dropout_plain}
_OWN = {"delta": _delta_own, "layer": _layer_own, "dropout": _dropout_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def work(case):
    """Each input read once, each output written once. Operations of the delta rule: its recurrence's three products a step."""
    e = torch.empty(0, dtype=_TYPES[case["dtype"]]).element_size()
    train = case.get("train", False)
    if case["op"] == "delta":
        B, T, H, G, K, V = (case[k] for k in "BTHGKV")
        inputs = B * T * (2 * H * K + G * V + 2 * G) * e + B * G * K * V * 4 * case.get("state", False)
        moved = inputs + B * T * G * V * e + B * G * K * V * 4 + B * T * case.get("reset", False)
        return {"bytes": moved + (inputs + B * T * G * V * e if train else 0), "flops": 6.0 * B * T * G * K * V * (3 if train else 1)}
    N, D = case["N"], case["D"]
    if case["op"] == "layer":
        return {"bytes": N * D * e * (8 if train else 4) + 8 * D * (1 + train), "flops": N * D * (20.0 if train else 8.0)}
    return {"bytes": N * D * e * (4 if train else 2), "flops": N * D * (2.0 if train else 1.0)}


# ---- the same from the definitions in 64 bits


@torch.no_grad()
def _delta_exact(s):
    """Step by step; backwards through the states of 128 steps at a time, made again from the one before them."""
    q0, k0, v = (s[k].double().movedim(1, 0) for k in ("query", "key", "value"))       # [T, B, heads, ...]
    T, B, H, K = q0.shape
    G, V = v.shape[2:]
    to_v = lambda x: x.repeat_interleave(G // H, 2)  # noqa: E731
    q_len, k_len = torch.sqrt(q0.square().sum(-1, keepdim=True) + _UNIT_EPS), torch.sqrt(k0.square().sum(-1, keepdim=True) + _UNIT_EPS)
    q, k = to_v(q0 / q_len), to_v(k0 / k_len)
    a = 1 / (1 + torch.exp(s["gate"].double())).movedim(1, 0)
    b = 1 / (1 + torch.exp(-s["write"].double())).movedim(1, 0)
    keep = a
    if s["reset"] is not None:
        keep = a * (~s["reset"]).double().T[..., None]
    S = s["state"].double() if s["state"] is not None else q.new_zeros(B, G, K, V)
    out = torch.empty(T, B, G, V, device=q.device, dtype=torch.float64)
    piece, starts = 128, []

    def step(S, t):
        kept = keep[t][..., None, None] * S
        u = b[t][..., None] * (v[t] - (k[t][..., None, :] @ kept)[..., 0, :])
        return kept + k[t][..., :, None] * u[..., None, :]

    for t in range(T):
        if t % piece == 0:
            starts.append(S)
        S = step(S, t)
        out[t] = (q[t][..., None, :] @ S)[..., 0, :]
    result = {"out": out.movedim(0, 1), "last": S}
    if not s.get("train"):
        return result
    d_out = s["d_out"].double().movedim(1, 0)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    d_keep, db = torch.empty_like(keep), torch.empty_like(b)
    dS = torch.zeros_like(S)
    for p in range(len(starts) - 1, -1, -1):
        states = [starts[p]]
        for t in range(p * piece, min(T, p * piece + piece)):
            states.append(step(states[-1], t))
        for t in range(min(T, p * piece + piece) - 1, p * piece - 1, -1):
            S, after = states[t - p * piece], states[t - p * piece + 1]
            told = (k[t][..., None, :] @ S)[..., 0, :]
            rest = v[t] - keep[t][..., None] * told
            dS = dS + q[t][..., :, None] * d_out[t][..., None, :]
            dq[t] = (after @ d_out[t][..., None])[..., 0]
            du = (k[t][..., None, :] @ dS)[..., 0, :]
            db[t] = (du * rest).sum(-1)
            dv[t] = b[t][..., None] * du
            dk[t] = (dS @ (b[t][..., None] * rest)[..., None] - keep[t][..., None, None] * (S @ dv[t][..., None]))[..., 0]
            d_kept = dS - k[t][..., :, None] * dv[t][..., None, :]
            d_keep[t] = (d_kept * S).sum((-2, -1))
            dS = keep[t][..., None, None] * d_kept
    fold = lambda x: x.unflatten(2, (H, G // H)).sum(3)  # noqa: E731
    for name, d, x, length in (("d_query", fold(dq), q0, q_len), ("d_key", fold(dk), k0, k_len)):
        result[name] = (d / length - x * (x * d).sum(-1, keepdim=True) / length ** 3).movedim(0, 1)
    result["d_value"] = dv.movedim(0, 1)
    result["d_gate"] = (-d_keep * keep * (1 - a)).movedim(0, 1)
    result["d_write"] = (db * b * (1 - b)).movedim(0, 1)
    if s["state"] is not None:
        result["d_state"] = dS
    return result


def _dropped(seed, shape, p):
    """Truth values of the elements that are dropped, by products of 16-bit halves"""
    n = 1
    for d in shape:
        n *= d
    at = torch.arange(n, device=seed.device, dtype=torch.int64)
    block, lane = at // 8, at % 8
    block = block[::8]

    def times(x, m):
        """The high and the low 32 bits of x m"""
        xl, xh, ml, mh = x % 65536, x // 65536, m % 65536, m // 65536
        middle = xh * ml + (xl * ml) // 65536
        cross = middle % 65536 + xl * mh
        return xh * mh + middle // 65536 + cross // 65536, (cross % 65536) * 65536 + (xl * ml) % 65536

    value = int(seed.item())
    k0, k1 = value % 2 ** 32, value // 2 ** 32 % 2 ** 32
    x0, x1, x2, x3 = block % 2 ** 32, block // 2 ** 32, torch.zeros_like(block), torch.zeros_like(block)
    for turn in range(10):
        (h0, l0), (h1, l1) = times(x0, 0xD2511F53), times(x2, 0xCD9E8D57)
        x0, x1, x2, x3 = h1 ^ x1 ^ ((k0 + turn * 0x9E3779B9) % 2 ** 32), l1, h0 ^ x3 ^ ((k1 + turn * 0xBB67AE85) % 2 ** 32), l0
    words = torch.stack([x0, x1, x2, x3], 1)[at // 8, lane // 2]
    half = torch.where(lane % 2 == 0, words % 65536, words // 65536)
    return (half < round(p * 65536)).view(shape)


@torch.no_grad()
def _layer_exact(s):
    x = s["x"].double()
    factor = torch.ones_like(x)
    if s.get("p"):
        factor = (~_dropped(s["seed"], x.shape, s["p"])).double() / (1 - round(s["p"] * 65536) / 65536)
    stream = (x * factor + s["residual"].double()).to(s["x"].dtype).double()        # the stream is stored in its type
    w = s["weight"].double()
    D = stream.shape[1]
    var, mean = torch.var_mean(stream, -1, correction=0, keepdim=True)
    std = torch.sqrt(var + _NORM_EPS)
    unit = (stream - mean) / std
    out = {"y": unit * w + s["bias"].double(), "stream": stream}
    if s.get("train"):
        d_y = s["d_y"].double()
        g = d_y * w
        d = s["d_stream"].double() + (g - g.sum(-1, keepdim=True) / D - unit * (g * unit).sum(-1, keepdim=True) / D) / std
        out |= {"d_x": d * factor, "d_residual": d, "d_weight": (d_y * unit).sum(0), "d_bias": d_y.sum(0)}
    return out


@torch.no_grad()
def _dropout_exact(s):
    factor = (~_dropped(s["seed"], s["x"].shape, s["p"])).double() / (1 - round(s["p"] * 65536) / 65536)
    out = {"y": s["x"].double() * factor}
    if s.get("train"):
        out["d_x"] = s["d_y"].double() * factor
    return out


def exact(case, seed):
    return {"delta": _delta_exact, "layer": _layer_exact, "dropout": _dropout_exact}[case["op"]](prepare(case, seed))
