"""The operators of a recurrent language model over the cohort's windows, in their plain forms and as the package's calls.

  scan    panvram_amd.ops.gated_scan: z = sigmoid(gate), h[t] = (1 - z[t]) h[t-1] + z[t] value[t] over [B, T, D], from a
          state or from zero; a reset at t drops h[t-1] (windows packed back to back); its gradients
  norm    panvram_amd.ops.add_rms_norm / add_rms_norm_8bit: the residual stream s = x + residual, stored in its type, and
          s / sqrt(mean(s^2) + eps) * weight; in 8 bits with one scale per row; its gradients
  loss    panvram_amd.ops.next_base_loss / next_base_loss_grad: the head's logits over the alphabet, the mean cross-entropy
          of the next token over the places whose next token counts; its gradients; or each place's own loss
  clip    panvram_amd.ops.clip_gradients: the norm over all gradients, and the gradients scaled to at most max_norm

A training step strings them together on what Cohort.sample(tokens=True) returns; the forms of one token are generation's.
"""
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPS = 1e-6
_E4M3_MAX = 448.0
_IGNORE = 4          # the window token of every byte other than A, C, G, T


def listed():
    return [
        # generation: one base for each of 16 sequences, the state carried from call to call
        {"name": "scan_step_16x1024", "op": "scan", "B": 16, "T": 1, "D": 1024, "dtype": "bfloat16", "state": True},
        # a training step's layer on a batch of the headline's window length, gate and value halves of one projection
        {"name": "scan_train_8x8192x1024", "op": "scan", "B": 8, "T": 8192, "D": 1024, "dtype": "bfloat16", "train": True, "joined": True},
        # a small model in full precision on the loader's odd context length, two windows packed in each row, a carried state
        {"name": "scan_train_5x2049x500", "op": "scan", "B": 5, "T": 2049, "D": 500, "dtype": "float32", "train": True, "state": True, "reset": True},
        # a whole 2^20-base slice of one haplotype through a layer at inference
        {"name": "scan_1x1048576x512", "op": "scan", "B": 1, "T": 1 << 20, "D": 512, "dtype": "bfloat16", "state": True},
        # generation: the norm of 16 rows, where only latency counts
        {"name": "norm_16x1024", "op": "norm", "N": 16, "D": 1024, "dtype": "bfloat16"},
        # the norm of the training step above, forward and backward
        {"name": "norm_train_65536x1024", "op": "norm", "N": 65536, "D": 1024, "dtype": "bfloat16", "train": True},
        # a long context scored with 8-bit projections
        {"name": "norm_8bit_32768x4096", "op": "norm", "N": 32768, "D": 4096, "dtype": "bfloat16", "bits8": True},
        # the loss of the training step above with its gradients: four bases, and one more id
        {"name": "loss_train_8x8192x1024", "op": "loss", "B": 8, "T": 8192, "D": 1024, "V": 5, "dtype": "bfloat16", "train": True},
        # the small model's loss in full precision, odd sizes, a few ids for special tokens
        {"name": "loss_train_5x2049x500", "op": "loss", "B": 5, "T": 2049, "D": 500, "V": 12, "dtype": "float32", "train": True},
        # held-out windows of 32 KiB scored base by base, no gradients
        {"name": "loss_16x32768x512", "op": "loss", "B": 16, "T": 32768, "D": 512, "V": 5, "dtype": "bfloat16"},
        # the gradients of a small model: many tensors, odd sizes, most of them short
        {"name": "clip_2M_in_150", "op": "clip", "tensors": 150, "total": 2_000_000, "dtype": "float32"},
        # those of a model of half a billion parameters
        {"name": "clip_500M_in_300", "op": "clip", "tensors": 300, "total": 500_000_000, "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["scan", "scan", "norm", "norm", "loss", "clip"])
    case = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}
    if op == "scan":
        train = rng.random() < 0.5
        most = 1 << (26 if train else 28)
        case |= {"T": 1 if rng.random() < 0.2 else _log(rng, 2, 1 << (15 if train else 20)), "D": _log(rng, 16, 2048)}
        case["B"] = _log(rng, 1, max(1, min(64, most // (case["T"] * case["D"]))))
        for flag in ("state", "reset", "joined"):
            if rng.random() < 0.4:
                case[flag] = True
        if train:
            case["train"] = True
    elif op == "norm":
        case["D"] = _log(rng, 64, 8192)
        case["N"] = _log(rng, 1, (1 << 26) // case["D"])
        form = rng.choice(["plain", "train", "bits8"])
        if form != "plain":
            case[form] = True
    elif op == "loss":
        case |= {"D": _log(rng, 32, 2048), "T": _log(rng, 16, 32768), "V": rng.randint(4, 16)}
        case["B"] = _log(rng, 1, max(1, min(64, (1 << 26) // (case["T"] * case["D"]))))
        if rng.random() < 0.6:
            case["train"] = True
    else:
        case |= {"tensors": rng.randint(1, 300), "total": _log(rng, 20_000, 1 << 27)}
    return case


def _sizes(case):
    """The tensors' sizes: a few large matrices, many short vectors, odd ones among them, `total` elements about."""
    k, total = case["tensors"], case["total"]
    weights = [1.0 / (1 + (i * 7) % 13) ** 4 for i in range(k)]
    scale = total / sum(weights)
    return [max(1, int(scale * w)) for w in weights]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    s = dict(case)

    def normal(*shape, mean=0.0, std=1.0, kind=dtype):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).mul_(std).add_(mean).to(kind)

    if case["op"] == "scan":
        B, T, D = case["B"], case["T"], case["D"]
        # gates that keep most of the state from base to base, as trained ones over long windows do
        if case.get("joined"):
            both = torch.empty(B, T, 2 * D, device=dev, dtype=dtype)
            both[..., :D] = normal(B, T, D, mean=-2.0, std=1.5)
            both[..., D:] = normal(B, T, D)
            s["gate"], s["value"] = (half.detach() for half in both.chunk(2, -1))
        else:
            s["gate"], s["value"] = normal(B, T, D, mean=-2.0, std=1.5), normal(B, T, D)
        s["state"] = normal(B, D, kind=torch.float32) if case.get("state") else None
        s["reset"] = None
        if case.get("reset"):
            s["reset"] = torch.rand(B, T, generator=gen, device=dev) < 2.0 / T
        if case.get("train"):
            s["d_out"] = normal(B, T, D, std=0.01)
            s["wanted"] = [t.requires_grad_() for t in (s["gate"], s["value"], s["state"]) if t is not None]
    elif case["op"] == "norm":
        N, D = case["N"], case["D"]
        s["x"], s["residual"] = normal(N, D, std=0.5), normal(N, D, std=2.0)
        s["weight"] = normal(D, mean=1.0, std=0.2, kind=torch.float32)
        if case.get("train"):
            s["d_y"], s["d_stream"] = normal(N, D, std=0.01), normal(N, D, std=0.01)
            s["wanted"] = [t.requires_grad_() for t in (s["x"], s["residual"], s["weight"])]
    elif case["op"] == "loss":
        B, T, D, V = case["B"], case["T"], case["D"], case["V"]
        s["hidden"] = normal(B, T, D)
        s["weight"] = normal(V, D, std=D ** -0.5)
        bases = torch.randint(4, (B, T), generator=gen, device=dev, dtype=torch.uint8)
        unknown = torch.rand(B, T, generator=gen, device=dev) < 0.01
        s["tokens"] = torch.where(unknown, torch.full_like(bases, _IGNORE), bases)
    else:
        sizes = _sizes(case)
        s["grads"] = [normal(n, std=1e-2) for n in sizes]
        # the clipped gradients go into one flat buffer, each at a multiple of 64 elements, as a sharded optimizer keeps them
        step = [-(-n // 64) * 64 for n in sizes]
        s["flat"] = torch.zeros(sum(step), device=dev, dtype=dtype)
        s["out"] = [piece[:n] for piece, n in zip(s["flat"].split(step), sizes)]
        s["max_norm"] = 1.0
    return s


# ---- the plain forms: elementary torch operations in 32 bits, rounded once


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] from h[-1] = 0 along dim 1, by doubling: after each step every place has summed up twice as
    many of those before it. (A loop of log2(T) steps: elementary operations have no scan of products and sums.)"""
    d, T = 1, a.shape[1]
    while d < T:
        b = torch.cat([b[:, :d], torch.addcmul(b[:, d:], a[:, d:], b[:, :-d])], 1)
        if 2 * d < T:
            a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


@torch.no_grad()
def _scan_plain(s):
    dtype = s["gate"].dtype
    gate, value, state = s["gate"].float(), s["value"].float(), s["state"]
    z, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    if s["reset"] is not None:
        keep = keep.masked_fill(s["reset"][..., None], 0.0)
    add = z * value
    if state is not None:
        add[:, 0] += keep[:, 0] * state
    h = _recurrence(keep, add)
    out = {"out": h.to(dtype), "last": h[:, -1].clone()}
    if s.get("train"):
        before = torch.zeros_like(h)
        before[:, 1:] = h[:, :-1]
        if state is not None:
            before[:, 0] = state
        if s["reset"] is not None:
            before = before.masked_fill(s["reset"][..., None], 0.0)
        # the gradient of h[t], from the end: G[t] = d_out[t] + keep[t+1] G[t+1]
        after = torch.zeros_like(keep)
        after[:, :-1] = keep[:, 1:]
        G = _recurrence(after.flip(1), s["d_out"].float().flip(1)).flip(1)
        out["d_gate"] = (z * torch.sigmoid(-gate) * G * (value - before)).to(dtype)
        out["d_value"] = (z * G).to(dtype)
        if state is not None:
            out["d_state"] = keep[:, 0] * G[:, 0]
    return out


@torch.no_grad()
def _norm_plain(s):
    dtype, w = s["x"].dtype, s["weight"]
    stream = (s["x"].float() + s["residual"].float()).to(dtype)      # the stream as the next layer reads it
    f = stream.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + _EPS)
    y = f * r * w
    if s.get("bits8"):
        scale = y.abs().amax(-1, keepdim=True) / _E4M3_MAX
        return {"q": (y / scale).to(torch.float8_e4m3fn), "scale": scale[:, 0], "stream": stream}
    out = {"y": y.to(dtype), "stream": stream}
    if s.get("train"):
        d_y = s["d_y"].float()
        unit, g = f * r, d_y * w
        d = s["d_stream"].float() + r * (g - unit * (g * unit).mean(-1, keepdim=True))
        out["d_x"] = d.to(dtype)
        out["d_residual"] = out["d_x"]
        out["d_weight"] = (d_y * unit).sum(0)
    return out


@torch.no_grad()
def _loss_plain(s):
    dtype, V = s["hidden"].dtype, s["V"]
    B, T, D = s["hidden"].shape
    hidden, weight = s["hidden"].reshape(B * T, D).float(), s["weight"].float()
    target = torch.full((B, T), _IGNORE, device=hidden.device, dtype=torch.int64)
    target[:, :-1] = s["tokens"][:, 1:]
    target = target.reshape(B * T)
    counts = target != _IGNORE
    count = counts.sum().clamp(min=1)
    logits = hidden @ weight.T
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    at = torch.where(counts, target, torch.zeros_like(target))[:, None]
    each = (torch.log(total) + top - logits.gather(1, at))[:, 0]
    each = torch.where(counts, each, torch.zeros_like(each))
    if not s.get("train"):
        return {"loss": each.view(B, T)}
    loss = each.sum() / count
    hot = (at == torch.arange(V, device=hidden.device)).float()
    d_logits = (e / total - hot) * (counts[:, None] / count)
    return {"loss": loss, "d_hidden": (d_logits @ weight).to(dtype).view(B, T, D), "d_weight": (d_logits.T @ hidden).to(dtype)}


@torch.no_grad()
def _clip_plain(s):
    norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * factor)
    return {"norm": norm, "out": s["flat"]}


# ---- the package's calls


def _scan_own(s):
    from panvram_amd import ops
    h, last = ops.gated_scan(s["gate"], s["value"], state=s["state"], reset=s["reset"])
    out = {"out": h, "last": last}
    if s.get("train"):
        d = torch.autograd.grad(h, s["wanted"], s["d_out"])
        out["d_gate"], out["d_value"] = d[:2]
        if s["state"] is not None:
            out["d_state"] = d[2]
    return out


def _norm_own(s):
    from panvram_amd import ops
    if s.get("bits8"):
        q, scale, stream = ops.add_rms_norm_8bit(s["x"], s["residual"], s["weight"], eps=_EPS)
        return {"q": q, "scale": scale, "stream": stream}
    y, stream = ops.add_rms_norm(s["x"], s["residual"], s["weight"], eps=_EPS)
    out = {"y": y, "stream": stream}
    if s.get("train"):
        out["d_x"], out["d_residual"], out["d_weight"] = torch.autograd.grad((y, stream), s["wanted"], (s["d_y"], s["d_stream"]))
    return out


def _loss_own(s):
    from panvram_amd import ops
    if not s.get("train"):
        return {"loss": ops.next_base_loss(s["hidden"], s["weight"], s["tokens"], ignore=_IGNORE, reduction="none")}
    loss, d_hidden, d_weight = ops.next_base_loss_grad(s["hidden"], s["weight"], s["tokens"], ignore=_IGNORE)
    return {"loss": loss, "d_hidden": d_hidden, "d_weight": d_weight}


def _clip_own(s):
    from panvram_amd import ops
    return {"norm": ops.clip_gradients(s["grads"], s["max_norm"], out=s["out"]), "out": s["flat"]}


_PLAIN = {"scan": _scan_plain, "norm": _norm_plain, "loss": _loss_plain, "clip": _clip_plain}
_OWN = {"scan": _scan_own, "norm": _norm_own, "loss": _loss_own, "clip": _clip_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


def work(case):
    """Each input read once, each output written once. The products of the loss are counted with the alphabet as it is."""
    e = torch.empty(0, dtype=_TYPES[case["dtype"]]).element_size()
    op = case["op"]
    if op == "scan":
        B, T, D = case["B"], case["T"], case["D"]
        n, train, state = B * T * D, case.get("train", False), case.get("state", False)
        moved = 3 * n * e + B * D * 4 * (1 + state) + (B * T if case.get("reset") else 0)
        return {"bytes": moved + (3 * n * e + B * D * 4 * state if train else 0), "flops": n * (20.0 if train else 8.0)}
    if op == "norm":
        N, D = case["N"], case["D"]
        if case.get("bits8"):
            return {"bytes": N * D * (3 * e + 1) + 4 * (N + D), "flops": 7.0 * N * D}
        train = case.get("train", False)
        return {"bytes": N * D * e * (7 if train else 4) + 4 * D * (1 + train), "flops": N * D * (16.0 if train else 5.0)}
    if op == "loss":
        n, D, V, train = case["B"] * case["T"], case["D"], case["V"], case.get("train", False)
        return {"bytes": (n * D + V * D) * e * (1 + train) + n * (1 if train else 5), "flops": 2.0 * n * D * V * (3 if train else 1)}
    n = sum(_sizes(case))
    return {"bytes": 2 * n * e, "flops": 3.0 * n}


# ---- the same from the definitions in 64 bits


def _walk(keep, add, first):
    """Every h[t] = keep[t] h[t-1] + add[t] from h[-1] = first, step by step: the steps of all pieces of about sqrt(T) places
    at once, then each piece's true start, then the steps again from it."""
    B, T, D = keep.shape
    piece = max(1, int(T ** 0.5))
    pieces = -(-T // piece)
    pad = pieces * piece - T
    if pad:
        keep = torch.cat([keep, keep.new_ones(B, pad, D)], 1)
        add = torch.cat([add, add.new_zeros(B, pad, D)], 1)
    keep, add = keep.view(B, pieces, piece, D), add.view(B, pieces, piece, D)
    h, through = add.new_zeros(B, pieces, D), add.new_ones(B, pieces, D)
    for t in range(piece):
        h = keep[:, :, t] * h + add[:, :, t]
        through = through * keep[:, :, t]
    starts, now = [], first
    for p in range(pieces):
        starts.append(now)
        now = through[:, p] * now + h[:, p]
    h = torch.stack(starts, 1)
    out = torch.empty_like(add)
    for t in range(piece):
        h = keep[:, :, t] * h + add[:, :, t]
        out[:, :, t] = h
    return out.view(B, pieces * piece, D)[:, :T]


@torch.no_grad()
def _scan_exact(s):
    gate, value = s["gate"].double(), s["value"].double()
    B, T, D = gate.shape
    first = s["state"].double() if s["state"] is not None else gate.new_zeros(B, D)
    z = 1 / (1 + torch.exp(-gate))
    rest = 1 / (1 + torch.exp(gate))
    goes_on = torch.ones(B, T, 1, device=gate.device, dtype=torch.float64) if s["reset"] is None else (~s["reset"]).double()[..., None]
    h = _walk(rest * goes_on, z * value, first)
    out = {"out": h, "last": h[:, -1].clone()}
    if s.get("train"):
        before = torch.cat([first[:, None], h[:, :-1]], 1) * goes_on
        keep = rest * goes_on
        back = torch.cat([keep[:, 1:], keep.new_zeros(B, 1, D)], 1).flip(1)
        G = _walk(back, s["d_out"].double().flip(1), gate.new_zeros(B, D)).flip(1)
        out["d_gate"] = G * (value - before) * z * rest
        out["d_value"] = G * z
        if s["state"] is not None:
            out["d_state"] = G[:, 0] * keep[:, 0]
    return out


@torch.no_grad()
def _norm_exact(s):
    stream = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()      # the stream is stored in its type
    w = s["weight"].double()
    length = torch.sqrt(stream.square().sum(-1) / stream.shape[1] + _EPS)[:, None]
    y = stream / length * w
    if s.get("bits8"):
        scale = y.abs().max(-1).values / _E4M3_MAX
        return {"q": (y / scale[:, None]).to(torch.float8_e4m3fn).double(), "scale": scale, "stream": stream}
    out = {"y": y, "stream": stream}
    if s.get("train"):
        d_y, d_stream = s["d_y"].double(), s["d_stream"].double()
        inner = (d_y * w * stream).sum(-1, keepdim=True) / stream.shape[1]
        d = d_stream + d_y * w / length - stream * inner / length ** 3
        out["d_x"] = out["d_residual"] = d
        out["d_weight"] = (d_y * stream / length).sum(0)
    return out


@torch.no_grad()
def _loss_exact(s):
    hidden, weight = s["hidden"].double(), s["weight"].double()
    B, T, D = hidden.shape
    target = s["tokens"][:, 1:].long().reshape(-1)
    rows = hidden[:, :-1].reshape(-1, D)
    p = torch.log_softmax(rows @ weight.T, -1)
    used = (target != _IGNORE).nonzero()[:, 0]
    n = max(1, len(used))
    if not s.get("train"):
        each = p.new_zeros(p.shape[0])
        each[used] = -p[used, target[used]]
        return {"loss": torch.cat([each.view(B, T - 1), each.new_zeros(B, 1)], 1)}
    loss = -p[used, target[used]].sum() / n
    d = torch.zeros_like(p)
    d[used] = torch.exp(p[used]) / n
    d[used, target[used]] -= 1.0 / n
    d_hidden = torch.zeros_like(hidden)
    d_hidden[:, :-1] = (d @ weight).view(B, T - 1, D)
    return {"loss": loss, "d_hidden": d_hidden, "d_weight": d.T @ rows}


@torch.no_grad()
def _clip_exact(s):
    squares = sum((g.double() * g.double()).sum() for g in s["grads"])
    norm = torch.sqrt(squares)
    factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    flat = torch.zeros(s["flat"].shape, device=s["flat"].device, dtype=torch.float64)
    at = 0
    for g in s["grads"]:
        flat[at:at + g.numel()] = g.double() * factor
        at += -(-g.numel() // 64) * 64
    return {"norm": norm, "out": flat}


def exact(case, seed):
    return {"scan": _scan_exact, "norm": _norm_exact, "loss": _loss_exact, "clip": _clip_exact}[case["op"]](prepare(case, seed))
