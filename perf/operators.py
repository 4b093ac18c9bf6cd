"""Cases of the sequence and matrix-update operators: what a pass computes, in plain form and through the framework.

Two operators and the optimizer step built on the second:

* `gated_scan`: h_t = g_t * h_{t-1} + x_t along packed or batched sequences, forward alone and with its backward pass;
* `orthogonalize`: an update matrix brought near its orthogonal factor by Newton-Schulz products;
* `muon_step`: momentum, orthogonalisation and the weight update of one matrix parameter.

`run` computes them from elementary torch operations in 32 bits, or, with `own` set, by the package's calls. `exact`
computes them from their definitions in 64 bits.
"""
import importlib
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gs():
    return importlib.import_module("3dgs_from_scratch_b200")


# ---- cases ---------------------------------------------------------------------------------------------------------


def _scan(name, **kw):
    """rows: rows of all sequences together; sequences: their number; even: a (sequences, T, C) batch, otherwise packed
    with offsets; tail: rows behind the last sequence; gates: per row (channels for one each); type, gate_type; train:
    with the backward pass; reverse; near: how near 1 the gates lie (the memory is about 1 / near rows)."""
    case = {"op": "scan", "name": name, "even": True, "tail": 0, "type": "f32", "gate_type": "f32", "train": True,
            "reverse": False, "near": 0.05}
    case.update(kw)
    return case


def _ortho(name, **kw):
    case = {"op": "ortho", "name": name, "batch": 1, "type": "f32"}
    case.update(kw)
    return case


def listed():
    return [
        # One frame of a running session: 64 states of 512 channels advance by a row. Latency.
        _scan("scan_frame", rows=64, sequences=64, channels=512, gates=512, train=False),
        # Inference over four sequences of a recurrent layer, half precision in and out.
        _scan("scan_layer_forward", rows=4 * 2048, sequences=4, channels=1024, gates=1024, type="bf16", gate_type="bf16",
              train=False, near=0.02),
        # A training step of the same layer, gates kept in 32 bits.
        _scan("scan_layer_train", rows=8 * 2048, sequences=8, channels=1024, gates=1024, type="bf16", near=0.02),
        # A state of 16 channels for each of 65,536 Gaussians over 30 frames: many short sequences.
        _scan("scan_gaussians_train", rows=65536 * 30, sequences=65536, channels=16, gates=16, near=0.1),
        # Back-to-front compositing of 35 channels (colour and features) over the sorted lists of 16,384 rays, one gate
        # (1 - alpha) a sample, ragged with empty rays.
        _scan("scan_composite_train", rows=524288, sequences=16384, channels=35, gates=1, even=False, reverse=True,
              near=0.2),
        # One very long sequence with few channels: only the time axis can be split.
        _scan("scan_long_train", rows=262144, sequences=1, channels=64, gates=64, near=0.001),
        # Ragged sequences in a padded buffer, odd sizes, 8 gates each shared by 25 channels.
        _scan("scan_heads_train", rows=30011, sequences=37, channels=200, gates=8, even=False, tail=77, type="f16",
              gate_type="f16", near=0.03),
        # The update of a small projection. Latency.
        _ortho("ortho_small", rows=64, cols=64),
        # The updates of the equal projections of a stack of layers, in half precision.
        _ortho("ortho_stack", rows=256, cols=512, batch=12, type="bf16"),
        # An odd, tall matrix in 32 bits.
        _ortho("ortho_odd", rows=1333, cols=1000),
        # A whole optimizer step of a projection of a wide layer.
        _ortho("muon_step", op="muon", rows=1024, cols=2048),
        # The largest square projection of the range.
        _ortho("ortho_large", rows=4096, cols=4096, type="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.6:
        train = rng.random() < 0.7
        channels = _log_int(rng, 3, 1500)
        rows = _log_int(rng, 40, min(1 << 20, (1 << 24) // channels))
        sequences = _log_int(rng, 1, rows)
        even = rng.random() < 0.4
        if even:
            rows = max(1, rows // sequences) * sequences
        divisors = [g for g in range(1, channels + 1) if channels % g == 0]
        gates = rng.choice([channels, channels, 1, rng.choice(divisors)])
        kind = rng.choice(["f32", "f32", "bf16", "f16"])
        case = _scan("", rows=rows, sequences=sequences, channels=channels, gates=gates, even=even, train=train,
                     type=kind, gate_type=rng.choice([kind, "f32"]), reverse=rng.random() < 0.3,
                     tail=0 if even else rng.choice([0, rng.randint(1, 100)]),
                     near=math.exp(rng.uniform(math.log(0.001), math.log(0.3))))
    else:
        rows, cols = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        batch = max(1, min(_log_int(rng, 1, 32), (1 << 24) // (rows * cols)))
        if rng.random() < 0.3:
            case = _ortho("", op="muon", rows=rows, cols=cols, batch=batch)
        else:
            case = _ortho("", rows=rows, cols=cols, batch=batch, type=rng.choice(["f32", "bf16", "f16"]))
    del case["name"]
    return case


def work(case):
    if case["op"] == "scan":
        n, s = case["rows"] * case["channels"], case["sequences"] * case["channels"]
        e, ge = torch.finfo(TYPES[case["type"]]).bits // 8, torch.finfo(TYPES[case["gate_type"]]).bits // 8
        gates = case["rows"] * case["gates"] * ge
        # forward: x and the gates in, h out, a state in and out for each sequence
        moved, flops = 2 * n * e + gates + 8 * s, 2 * n
        if case["train"]:
            # backward: dh and the final states' gradient in, dx, the gates' and the initial states' gradient out
            moved, flops = moved + 2 * n * e + gates + 8 * s, flops + 8 * n
        return {"bytes": moved, "flops": flops}
    m, n = sorted((case["rows"], case["cols"]))
    size = case["batch"] * m * n
    # A A and X X^T are symmetric: half of each product suffices
    flops = STEPS * case["batch"] * (m * m * n + m ** 3 + 2 * m * m * n)
    if case["op"] == "muon":
        return {"bytes": 5 * 4 * size, "flops": flops}
    return {"bytes": 2 * size * torch.finfo(TYPES[case["type"]]).bits // 8, "flops": flops}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _lengths(case, gen):
    """Ragged lengths that add up to the rows: cut points at random places, some twice, so that sequences may be empty."""
    rows, count = case["rows"], case["sequences"]
    cuts = torch.randint(0, rows + 1, (count - 1,), generator=gen, device="cuda")
    cuts = torch.cat([cuts.new_zeros(1), cuts.sort().values, cuts.new_full((1,), rows)])
    return cuts.to(torch.int32)


def _update(gen, batch, rows, cols, kind):
    """A gradient's look: a few strong directions over a broad floor, at a gradient's small scale."""
    rank = max(1, min(rows, cols) // 16)
    strong = torch.randn(batch, rows, rank, generator=gen, device="cuda") @ torch.randn(
        batch, rank, cols, generator=gen, device="cuda")
    noise = torch.randn(batch, rows, cols, generator=gen, device="cuda")
    return ((0.5 / math.sqrt(rank)) * strong + noise).mul_(1e-3).to(TYPES[kind])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": dict(case)}
    if case["op"] == "scan":
        total, c, s = case["rows"] + case["tail"], case["channels"], case["sequences"]
        kind, gate_kind = TYPES[case["type"]], TYPES[case["gate_type"]]

        def normal(*shape):
            return torch.randn(*shape, generator=gen, device="cuda")

        # Gates between 1 - 2 near and 1, an exact reset here and there; compositing weights lie in the same range.
        gate = 1.0 - 2.0 * case["near"] * torch.rand(total, case["gates"], generator=gen, device="cuda")
        gate = torch.where(torch.rand(total, case["gates"], generator=gen, device="cuda") < 1e-4, 0.0, gate)
        shape = (s, total // s) if case["even"] else (total,)
        state["x"] = (normal(total, c) * math.sqrt(case["near"])).to(kind).reshape(*shape, c)
        state["gate"] = gate.to(gate_kind).reshape(*shape, case["gates"])
        state["initial"] = normal(s, c)
        state["offsets"] = None
        state["longest"] = total // s
        if not case["even"]:
            state["offsets"] = _lengths(case, gen)
            state["longest"] = int((state["offsets"][1:] - state["offsets"][:-1]).max())
        if case["train"]:
            state["dh"] = normal(total, c).to(kind).reshape(*shape, c)
            state["dfinal"] = normal(s, c)
            for k in ("x", "gate", "initial"):
                state[k].requires_grad_(True)
        return state
    b, m, n = case["batch"], case["rows"], case["cols"]
    if case["op"] == "muon":
        state["weight"] = torch.randn(b, m, n, generator=gen, device="cuda") / math.sqrt(n)
        state["grad"] = _update(gen, b, m, n, "f32")
        state["momentum"] = _update(gen, b, m, n, "f32")
    else:
        state["update"] = _update(gen, b, m, n, case["type"])
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------


def _places(state):
    """For every row of the packed axis: its sequence, whether it is inside one, whether it is its sequence's first and
    last; and whether each sequence is empty."""
    case, offsets = state["case"], state["offsets"]
    total, s = case["rows"] + case["tail"], case["sequences"]
    row = torch.arange(total, device="cuda")
    if offsets is None:
        offsets = torch.arange(s + 1, device="cuda", dtype=torch.int32) * (total // s)
    seq = torch.searchsorted(offsets[1:], row.to(torch.int32), right=True)
    inside = seq < s
    seq = seq.clamp(max=s - 1)
    first = inside & (row == offsets[seq])
    last = inside & (row + 1 == offsets[seq + 1])
    return seq, inside, first, last, offsets[1:] == offsets[:-1]


def _doubling(mult, add, longest):
    """h_t = mult_t h_{t-1} + add_t from h_{-1} = 0 over the first axis, in log2(longest) passes over all rows."""
    step = 1
    while step < longest:
        add = torch.cat([add[:step], add[step:] + mult[step:] * add[:-step]])
        mult = torch.cat([mult[:step], mult[step:] * mult[:-step]])
        step *= 2
    return add


def _plain_scan(state):
    case = state["case"]
    total, c, g, s = case["rows"] + case["tail"], case["channels"], case["gates"], case["sequences"]
    with torch.no_grad():
        x = state["x"].reshape(total, g, c // g).float()
        gate = state["gate"].reshape(total, g, 1).float()
        initial = state["initial"].reshape(s, g, c // g).float()
        seq, inside, first, last, empty = _places(state)
        if case["reverse"]:
            first, last = last, first
        i, f, e = (v[:, None, None] for v in (inside, first, last))

        def along(t):
            return t.flip(0) if case["reverse"] else t

        def against(t):
            return t if case["reverse"] else t.flip(0)

        # the initial state enters at a sequence's first row, where the chain from the row before ends
        started = torch.where(f, gate * initial[seq], 0.0)
        h = _doubling(along(torch.where(i & ~f, gate, 0.0)), along(torch.where(i, x + started, 0.0)), state["longest"])
        h = along(h)
        final = torch.empty_like(initial)
        final[empty] = initial[empty]
        final[seq[last]] = h[last]
        out = {"h": h.reshape(state["x"].shape).to(state["x"].dtype), "final": final.reshape(s, c)}
        if not case["train"]:
            return out
        dh = torch.where(i, state["dh"].reshape(total, g, c // g).float(), 0.0)
        dfinal = state["dfinal"].reshape(s, g, c // g).float()
        dh = dh + torch.where(e, dfinal[seq], 0.0)
        v = _doubling(against(torch.where(i & ~e, gate, 0.0)), against(gate * dh), state["longest"])
        v = torch.where(i, against(v), 0.0)
        # what flows to a row from the one after it, and the state that it was computed from
        later, before = (v[:-1], h[1:]) if case["reverse"] else (v[1:], h[:-1])
        nothing = torch.zeros_like(v[:1])
        later = torch.cat([nothing, later] if case["reverse"] else [later, nothing])
        before = torch.cat([before, nothing] if case["reverse"] else [nothing, before])
        dx = torch.where(i, dh + torch.where(e, 0.0, later), 0.0)
        dgate = (dx * torch.where(f, initial[seq], before)).sum(2)
        dinitial = torch.where(empty[:, None, None], dfinal, 0.0)
        dinitial[seq[first]] = v[first]
        out["dx"] = dx.reshape(state["x"].shape).to(state["x"].dtype)
        out["dgate"] = dgate.reshape(state["gate"].shape).to(state["gate"].dtype)
        out["dinitial"] = dinitial.reshape(s, c)
        return out


def _plain_orthogonalize(update):
    a, b, c = COEFFICIENTS
    x = update.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / norm.clamp(min=1e-7).float()
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if tall else x).to(update.dtype)


MUON = {"lr": 0.02, "beta": 0.95, "weight_decay": 0.01}


def _plain_muon(state):
    weight, momentum, grad = state["weight"], state["momentum"], state["grad"]
    lr, beta, decay = MUON["lr"], MUON["beta"], MUON["weight_decay"]
    momentum.mul_(beta).add_(grad, alpha=1 - beta)
    update = _plain_orthogonalize(beta * momentum + (1 - beta) * grad)
    scale = math.sqrt(max(1.0, weight.shape[-2] / weight.shape[-1]))
    weight.mul_(1 - lr * decay).add_(update, alpha=-lr * scale)
    return {"weight": weight, "momentum": momentum}


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if case["op"] == "scan":
        if not own:
            return _plain_scan(state)
        h, final = _gs().gated_scan(state["x"], state["gate"], initial=state["initial"], offsets=state["offsets"],
                                    reverse=case["reverse"])
        if not case["train"]:
            return {"h": h, "final": final}
        dx, dgate, dinitial = torch.autograd.grad((h, final), (state["x"], state["gate"], state["initial"]),
                                                  (state["dh"], state["dfinal"]))
        return {"h": h, "final": final, "dx": dx, "dgate": dgate, "dinitial": dinitial}
    if case["op"] == "muon":
        if not own:
            return _plain_muon(state)
        _gs().muon_step(state["weight"], state["grad"], state["momentum"], steps=STEPS, coefficients=COEFFICIENTS, **MUON)
        return {"weight": state["weight"], "momentum": state["momentum"]}
    if not own:
        return _plain_orthogonalize(state["update"])
    return _gs().orthogonalize(state["update"], steps=STEPS, coefficients=COEFFICIENTS)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------


def _walk(gate, add, begin, count, start, backward):
    """One row of every piece at a time: piece p holds `count[p]` rows from row `begin[p]` on (from the last of them back,
    where `backward`), its state starts at start[p]. Returns all rows' states and each piece's product of gates and end."""
    order = torch.argsort(count, descending=True)
    begin, count, state = begin[order], count[order], start[order].clone()
    product = torch.ones(state.shape[0], *gate.shape[1:], dtype=torch.float64, device=state.device)
    out = torch.zeros_like(add)
    lens = count.cpu()
    for t in range(int(lens[0]) if len(lens) else 0):
        n = int((lens > t).sum())
        rows = begin[:n] + (count[:n] - 1 - t if backward else t)
        product[:n] *= gate[rows]
        state[:n] = gate[rows] * state[:n] + add[rows]
        out[rows] = state[:n]
    back = torch.argsort(order)
    return out, product[back], state[back]


def _recur(gate, add, offsets, start, backward):
    """h = gate h + add over every sequence from its start state: each sequence in pieces of 512 rows, the pieces first
    from zero for their products and ends, then again from the state that these give. Returns the rows and the ends."""
    piece, device = 512, add.device
    lens = (offsets[1:] - offsets[:-1]).tolist()
    begin, count, owner = [], [], []
    for s, (o, n) in enumerate(zip(offsets[:-1].tolist(), lens)):
        cuts = list(range(o, o + n, piece))
        for p in reversed(cuts) if backward else cuts:
            begin.append(p)
            count.append(min(piece, o + n - p))
            owner.append(s)
    if not begin:
        return torch.zeros_like(add), start.clone()
    begin, count = (torch.tensor(v, dtype=torch.int64, device=device) for v in (begin, count))
    owners = torch.tensor(owner, device=device)
    states = start[owners].clone()
    many = [k for k in range(1, len(owner)) if owner[k] == owner[k - 1]]
    if many:
        _, product, end = _walk(gate, add, begin, count, torch.zeros_like(states), backward)
        for k in many:
            states[k] = product[k - 1] * states[k - 1] + end[k - 1]
    out, _, end = _walk(gate, add, begin, count, states, backward)
    ends = start.clone()
    final = torch.tensor([k for k in range(len(owner)) if k + 1 == len(owner) or owner[k + 1] != owner[k]], device=device)
    ends[owners[final]] = end[final]
    return out, ends


def _exact_scan(case, state):
    total, c, g, s = case["rows"] + case["tail"], case["channels"], case["gates"], case["sequences"]
    x = state["x"].detach().double().reshape(total, g, c // g)
    gate = state["gate"].detach().double().reshape(total, g, 1)
    initial = state["initial"].detach().double().reshape(s, g, c // g)
    offsets = state["offsets"]
    offsets = torch.arange(s + 1, device="cuda") * (total // s) if offsets is None else offsets.long()
    h, final = _recur(gate, x, offsets, initial, case["reverse"])
    out = {"h": h.reshape(state["x"].shape), "final": final.reshape(s, c)}
    if not case["train"]:
        return out
    # u_t = dh_t + gate_{t+1} u_{t+1} from the far end, in terms of w_t = gate_t u_t
    dh = state["dh"].double().reshape(total, g, c // g)
    dh[int(offsets[-1]):] = 0
    w, dinitial = _recur(gate, gate * dh, offsets, state["dfinal"].double().reshape(s, g, c // g), not case["reverse"])
    dx, before = dh.clone(), torch.zeros_like(h)
    begin, end = offsets[:-1], offsets[1:]
    full = end > begin
    begin, end = begin[full], end[full]
    dfinal = state["dfinal"].double().reshape(s, g, c // g)[full]
    edge = torch.zeros(total + 1, dtype=torch.bool, device="cuda")
    edge[begin] = True
    edge[offsets[-1]:] = True
    inner = (~edge[1:-1]).nonzero().squeeze(1)  # rows whose next row belongs to the same sequence
    if case["reverse"]:
        dx[inner + 1] += w[inner]
        dx[begin] += dfinal
        before[inner] = h[inner + 1]
        before[end - 1] = initial[full]
    else:
        dx[inner] += w[inner + 1]
        dx[end - 1] += dfinal
        before[inner + 1] = h[inner]
        before[begin] = initial[full]
    out["dx"] = dx.reshape(state["x"].shape)
    out["dgate"] = (dx * before).sum(2).reshape(state["gate"].shape)
    out["dinitial"] = dinitial.reshape(s, c)
    return out


def _exact_orthogonalize(update):
    """The same polynomials on the other side, X (a + b X^T X + c (X^T X)^2), with X^T X the smaller product."""
    a, b, c = COEFFICIENTS
    wide = update.shape[-1] > update.shape[-2]
    x = (update.mT if wide else update).double()
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp(min=1e-7)
    unit = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = x.mT @ x
        x = x @ (a * unit + gram @ (b * unit + c * gram))
    return x.mT.contiguous() if wide else x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "scan":
        return _exact_scan(case, state)
    if case["op"] == "ortho":
        return _exact_orthogonalize(state["update"])
    lr, beta, decay = MUON["lr"], MUON["beta"], MUON["weight_decay"]
    grad = state["grad"].double()
    momentum = beta * state["momentum"].double() + (1 - beta) * grad
    update = _exact_orthogonalize(beta * momentum + (1 - beta) * grad)
    scale = math.sqrt(max(1.0, case["rows"] / case["cols"]))
    return {"weight": (1 - lr * decay) * state["weight"].double() - lr * scale * update, "momentum": momentum}
