"""Operators on the samples along a ray and on quantised leaf records, each as a user calls it.

* ``gated_scan``: the gated linear recurrence that emission and absorption along a ray follow,
  ``h[t] = a[t] h[t-1] + (1 - a[t]) x[t]`` with ``a = exp(-thickness)`` (``premultiplied``: ``+ x[t]``),
  all its states and the last one, and its backward pass;
* ``composite``: the last state alone, front to back: samples of rays of any length to colours, and
  its backward pass;
* ``RecordCache``: leaf records held in 8 bits, quantised as they are written (``set`` by point,
  ``write`` by leaf id) and read back (by point, ``read`` by leaf id).

``own`` chooses between the package's calls and the same in elementary tensor operations.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
# shell of the refined part of a tree: occupied space is a thin surface
SHELL = (0.30, 0.35)
# elements of `values` that a drawn case has at most
MOST = 1 << 26


def _scan(name, B, T, C, H, dtype, gates, grad, reverse=False, premultiplied=False):
    case = {"kind": "scan", "B": B, "T": T, "C": C, "H": H, "dtype": dtype, "gates": gates,
            "grad": grad, "reverse": reverse, "premultiplied": premultiplied}
    return case if name is None else {**case, "name": name}


def _rays(name, B, mean, C, dtype, grad, packed=True):
    case = {"kind": "rays", "B": B, "mean": mean, "C": C, "dtype": dtype, "grad": grad,
            "packed": packed}
    return case if name is None else {**case, "name": name}


def _records(name, kind, basis, code, Q, refine, extra, by, out):
    case = {"kind": kind, "basis": basis, "code": code, "Q": Q, "refine": refine, "extra": extra,
            "by": by, "out": out}
    return case if name is None else {**case, "name": name}


def listed():
    return [
        # one more step of a running recurrence, a gate for each channel: latency counts
        _scan("scan_token", 64, 1, 1024, 1024, "bf16", "fp32", False),
        # a training step over sequences of odd length and width, 32-bit, back to front
        _scan("scan_train_odd", 7, 1001, 333, 333, "fp32", "fp32", True, reverse=True),
        # heads of 64 channels that share a gate, inputs weighted beforehand
        _scan("scan_train_heads", 4, 2048, 512, 8, "bf16", "fp32", True, premultiplied=True),
        # one long sequence, far more steps than channels
        _scan("scan_long", 1, 131072, 64, 64, "fp32", "fp32", False),
        # a training step of a large batch: bound by memory
        _scan("scan_train_large", 8, 4096, 2048, 2048, "bf16", "bf16", True),
        # the rays of the toy scene, a few samples each: latency counts
        _rays("rays_toy", 4096, 21, 3, "fp32", False),
        # a stochastic training step: ragged rays, many without any sample
        _rays("rays_train", 65536, 84, 3, "fp32", True),
        # the benchmark's 2^20 rays, one step
        _rays("rays_train_large", 1 << 20, 42, 3, "fp32", True),
        # feature vectors instead of colours, as many samples on each ray
        _rays("rays_features", 16384, 64, 32, "bf16", True, packed=False),
        # a few records changed in a small tree and looked at: latency counts
        _records("records_edit", "write", 4, "int8", 1000, 3, 0, "ids", "fp32"),
        # records of 2^20 points written to a sparse tree and read back
        _records("records_write", "write", 9, "int8", 1 << 20, 5, 2, "points", "fp32"),
        # reading the benchmark's largest records along many rays
        _records("records_read", "read", 16, "e4m3", (1 << 22) + 1, 5, 3, "points", "fp32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "rays", "rays", "write", "read"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "scan":
        H, D = rng.choice([(_spread(rng, 1, 1024), 1), (_spread(rng, 1, 16), _spread(rng, 2, 96)),
                           (1, _spread(rng, 2, 512))])
        T = _spread(rng, 1, 16384)
        B = _spread(rng, 1, max(1, min(4096, MOST // (T * H * D))))
        return _scan(None, B, T, H * D, H, dtype, rng.choice(["fp32", dtype]),
                     rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.3)
    if kind == "rays":
        C, mean = rng.choice([1, 3, 3, 3, 4, _spread(rng, 2, 64)]), _spread(rng, 4, 256)
        B = _spread(rng, 16, max(16, min(1 << 20, MOST // (mean * C))))
        return _rays(None, B, mean, C, dtype, rng.random() < 0.6, rng.random() < 0.7)
    basis, extra = rng.choice([1, 4, 9, 16, 25]), rng.randrange(3)
    Q = _spread(rng, 1, (1 << 22) // (1 + basis // 9))
    return _records(None, kind, basis, rng.choice(["int8", "e4m3"]), Q, rng.randrange(2, 6), extra,
                    rng.choice(["points", "ids"]), dtype)


# ---------------------------------------------------------------------------
# Inputs

def _gates_shape(case):
    return (case["B"], case["T"], case["H"]) if case["H"] > 1 else (case["B"], case["T"])


def _thickness(shape, gen):
    """What the samples of a ray absorb: nothing in empty space, little in haze, all at a surface."""
    kind = torch.rand(shape, device=DEVICE, generator=gen)
    soft = torch.rand(shape, device=DEVICE, generator=gen)
    g = torch.where(kind < 0.9, 0.1 * soft, 8.0 * soft)
    return torch.where(kind < 0.5, torch.zeros_like(g), g)


def _offsets(B, mean, gen):
    """Where the samples of each ray begin: B * mean samples cut at random places, and an eighth of
    the rays miss the scene."""
    hits = torch.randperm(B, device=DEVICE, generator=gen)[:B - B // 8]
    cuts = torch.randint(0, B * mean + 1, (hits.numel() - 1,), device=DEVICE, generator=gen)
    ends = torch.tensor([0, B * mean], device=DEVICE)
    n = torch.zeros(B, dtype=torch.int64, device=DEVICE)
    n[hits] = torch.cat([ends[:1], cuts.sort()[0], ends[1:]]).diff()
    return torch.cat([ends[:1], n.cumsum(0)])


def _prepare_scan(case, gen):
    B, T, C = case["B"], case["T"], case["C"]
    dt, gd = DTYPES[case["dtype"]], DTYPES[case["gates"]]

    def normal(*shape):
        return torch.randn(shape, device=DEVICE, generator=gen)

    s = {"values": normal(B, T, C).to(dt),
         # between forgetting at once and remembering for a hundred steps
         "thickness": torch.exp(1.5 * normal(*_gates_shape(case)) - 2.0).to(gd),
         "initial": normal(B, C)}
    if case["grad"]:
        s["d_states"] = normal(B, T, C).to(dt)
        s["d_last"] = normal(B, C)
    return s


def _prepare_rays(case, gen):
    B, C, dt = case["B"], case["C"], DTYPES[case["dtype"]]
    s = {"offsets": None}
    if case["packed"]:
        s["offsets"] = _offsets(B, case["mean"], gen)
        lead = (B * case["mean"],)
    else:
        lead = (B, case["mean"])
    s["values"] = torch.rand((*lead, C), device=DEVICE, generator=gen).to(dt)
    s["thickness"] = _thickness(lead, gen)
    s["initial"] = torch.rand((B, C), device=DEVICE, generator=gen)
    if case["grad"]:
        s["d_last"] = torch.randn((B, C), device=DEVICE, generator=gen)
    return s


def _octree(refine, extra):
    """child (M, 8) int32 of a tree of (2^(refine + 1))^3 leaves, those of them whose centre lies in
    SHELL split `extra` times more; the ids of the leaves split first."""
    levels = refine + 1
    start = [(8 ** i - 1) // 7 for i in range(levels + 1)]
    M = start[levels]
    child = torch.zeros((M, 8), dtype=torch.int32, device=DEVICE)
    corner = torch.zeros((1, 3), device=DEVICE)
    cells = torch.stack(torch.meshgrid(*[torch.arange(2, device=DEVICE)] * 3, indexing="ij"),
                        -1).reshape(1, 8, 3)
    for i in range(levels):
        below = (corner[:, None] + cells * 0.5 ** (i + 1)).reshape(-1, 3)
        if i + 1 < levels:
            node = torch.arange(start[i], start[i + 1], device=DEVICE)[:, None]
            slots = torch.arange(8 ** (i + 1), device=DEVICE).reshape(-1, 8)
            child[start[i]:start[i + 1]] = (start[i + 1] + slots - node).to(torch.int32)
        corner = below
    dist = (corner + 0.5 ** (levels + 1) - 0.5).norm(dim=1)
    split = torch.nonzero((dist >= SHELL[0]) & (dist <= SHELL[1])).flatten() + 8 * start[levels - 1]
    first = split
    for _ in range(extra if split.numel() else 0):
        n = split.numel()
        new = torch.arange(M, M + n, device=DEVICE)
        child.view(-1)[split] = (new - split // 8).to(torch.int32)
        child = torch.cat([child, torch.zeros((n, 8), dtype=torch.int32, device=DEVICE)])
        split = (new[:, None] * 8 + torch.arange(8, device=DEVICE)).flatten()
        M += n
    return child, first


def _prepare_records(case, gen):
    basis, Q, extra = case["basis"], case["Q"], case["extra"]
    K = 3 * basis + 1
    child, split = _octree(case["refine"], extra)

    def rows(n):
        v = torch.randn((n, K), device=DEVICE, generator=gen)
        v[:, -1] = torch.rand(n, device=DEVICE, generator=gen) * 50.0
        return v

    levels = case["refine"] + 1 + extra
    s = {"out": DTYPES[case["out"]]}
    near = torch.randn((Q, 3), device=DEVICE, generator=gen)
    near = 0.5 + near / near.norm(dim=1, keepdim=True) * (
        SHELL[0] + (SHELL[1] - SHELL[0]) * torch.rand((Q, 1), device=DEVICE, generator=gen))
    points = torch.rand((Q, 3), device=DEVICE, generator=gen)
    points = torch.where(torch.rand((Q, 1), device=DEVICE, generator=gen) < 0.5, points, near)
    if case["by"] == "points":
        s["points"] = points
    else:
        s["ids"] = _leaf_of(child, points, levels)
    data = rows(child.numel())
    if own:
        import svox_b200 as svox
        tree = svox.N3Tree(data_format="SH%d" % basis, init_refine=case["refine"], device=DEVICE)
        if extra and split.numel():
            tree.refine(extra, sel=(split // 8, split // 4 % 2, split // 2 % 2, split % 2))
        tree.data.data.view(-1, K)[:child.numel()] = data
        s["cache"] = svox.RecordCache(tree, dtype=CODES[case["code"]])
    else:
        s["child"], s["levels"], s["data"] = child, levels, data
        s["cache"] = _encode(data, basis, case["code"])
    if case["kind"] == "write":
        s["values"] = rows(Q)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"scan": _prepare_scan, "rays": _prepare_rays, "write": _prepare_records,
         "read": _prepare_records}[case["kind"]](case, gen)
    s["case"] = case
    if case.get("grad"):
        for name in ("values", "thickness", "initial"):
            s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# The package's calls

def _run_own(s):
    import svox_b200 as svox
    case = s["case"]
    if case["kind"] == "write":
        if "points" in s:
            s["cache"].set(s["points"], s["values"])
        else:
            s["cache"].write(s["ids"], s["values"])
    if case["kind"] in ("write", "read"):
        if "points" in s:
            return s["cache"](s["points"], dtype=s["out"])
        return s["cache"].read(s["ids"], dtype=s["out"])
    leaves = [s["values"], s["thickness"], s["initial"]]
    if case["kind"] == "scan":
        states, last = svox.gated_scan(s["values"], s["thickness"], initial=s["initial"],
                                       reverse=case["reverse"],
                                       premultiplied=case["premultiplied"])
        if not case["grad"]:
            return {"states": states, "last": last}
        grads = torch.autograd.grad([states, last], leaves, [s["d_states"], s["d_last"]])
        out = {"states": states, "last": last}
    else:
        last = svox.composite(s["values"], s["thickness"], background=s["initial"],
                              offsets=s["offsets"])
        if not case["grad"]:
            return {"last": last}
        grads = torch.autograd.grad([last], leaves, [s["d_last"]])
        out = {"last": last}
    return {**out, "d_values": grads[0], "d_thickness": grads[1], "d_initial": grads[2]}


# ---------------------------------------------------------------------------
# The plain forms

def _prefix(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1 from h = 0, and the products of a up to t: each round
    joins every step with what ends `step` before it."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


def _plain_scan(s):
    case = s["case"]
    B, T, C, H = (case[k] for k in "BTCH")
    x, g = s["values"].float(), s["thickness"].float().reshape(B, T, H, 1)
    # (a gate is repeated over the channels of its head)
    g = g.expand(B, T, H, C // H).reshape(B, T, C)
    if case["reverse"]:
        x, g = x.flip(1), g.flip(1)
    a = torch.exp(-g)
    w = torch.ones_like(a) if case["premultiplied"] else -torch.expm1(-g)
    h0 = s["initial"][:, None]
    decay, h = _prefix(a, w * x)
    h = h + decay * h0

    def order(v):
        return v.flip(1) if case["reverse"] else v

    out = {"states": order(h).to(s["values"].dtype), "last": h[:, -1].clone()}
    if not case["grad"]:
        return out
    # G[t] = d[t] + a[t+1] G[t+1]: the same from the other end, the gates one step on
    d = order(s["d_states"].float())
    d = torch.cat([d[:, :-1], d[:, -1:] + s["d_last"][:, None]], 1).flip(1)
    ahead = torch.cat([torch.zeros_like(a[:, :1]), a[:, 1:].flip(1)], 1)
    G = _prefix(ahead, d)[1].flip(1)
    before = torch.cat([h0, h[:, :-1]], 1)
    dg = a * G * (-before if case["premultiplied"] else x - before)
    return {**out, "d_values": order(w * G).to(s["values"].dtype),
            "d_thickness": order(dg).reshape(B, T, H, C // H).sum(-1).to(
                s["thickness"].dtype).reshape(s["thickness"].shape),
            "d_initial": a[:, 0] * G[:, 0]}


def _sums(v):
    """Sums of all rows before each, and of all: (n, C) -> (n + 1, C)."""
    upto = v.T.contiguous().cumsum(1).T
    return torch.cat([upto.new_zeros(1, v.shape[1]), upto])


def _plain_rays(s):
    case = s["case"]
    B, C = case["B"], case["C"]
    x = s["values"].reshape(-1, C)
    g = s["thickness"].reshape(-1).double()     # sums over all samples: 64 bits
    o = s["offsets"]
    if o is None:
        o = torch.arange(B + 1, device=DEVICE) * case["mean"]
    ray = torch.repeat_interleave(torch.arange(B, device=DEVICE), o.diff(),
                                  output_size=g.numel())
    upto = _sums(g[:, None])[:, 0]
    through = torch.exp(upto[o[:-1]][ray] - upto[:-1])       # what reaches each sample
    end = torch.exp(upto[o[:-1]] - upto[o[1:]])              # what reaches the background
    w = through * -torch.expm1(-g)
    total = _sums(w[:, None] * x)
    last = total[o[1:]] - total[o[:-1]] + end[:, None] * s["initial"]
    out = {"last": last.float()}
    if not case["grad"]:
        return out
    d = s["d_last"].double()
    c = (d[ray] * x).sum(-1)
    upto_c = _sums((w * c)[:, None])[:, 0]
    behind = upto_c[o[1:]][ray] - upto_c[1:] + (end * (d * s["initial"]).sum(-1))[ray]
    dg = through * torch.exp(-g) * c - behind
    return {**out, "d_values": (w[:, None] * d[ray]).to(x.dtype).reshape(s["values"].shape),
            "d_thickness": dg.float().reshape(s["thickness"].shape),
            "d_initial": (end[:, None] * d).float()}


def _exponent(most, code):
    """The power of two by which a group whose largest magnitude is `most` is divided: the smallest
    one after which that rounds to no more than 127 (int8), or is at most 448 (e4m3)."""
    m, e = torch.frexp(most)
    m, e = 2.0 * m, e - 1
    e = e - 6 + (m >= 127.5 / 64) if code == "int8" else e - 8 + (m > 1.75)
    return torch.where(most > 0, e, -126).clamp(min=-126).to(torch.int32)


def _two_to(e):
    """2^e as a float, from its bits."""
    return ((e + 127) << 23).view(torch.float32)


def _encode(values, basis, code):
    """Records in 8 bits: codes (n, 3, basis), the exponent of each colour channel's scale, the
    density in 16 bits."""
    colour = values[:, :-1].float().reshape(-1, 3, basis)
    e = _exponent(colour.abs().amax(-1), code)
    y = colour * _two_to(-e)[..., None]
    codes = torch.round(y).to(torch.int8) if code == "int8" else y.to(torch.float8_e4m3fn)
    return {"codes": codes, "e": e, "density": values[:, -1].half()}


def _leaf_of(child, points, levels):
    """Ids of the leaves that hold the points, of a tree at most `levels` deep."""
    flat, pos = child.view(-1), points.clamp(0.0, 1.0 - 1e-6)
    node = torch.zeros(points.shape[0], dtype=torch.int64, device=points.device)
    leaf = torch.full_like(node, -1)
    for _ in range(levels):
        pos = pos * 2
        cell = pos.floor()
        pos = pos - cell
        cell = cell.long()
        slot = node * 8 + cell[:, 0] * 4 + cell[:, 1] * 2 + cell[:, 2]
        step = flat[slot].long()
        leaf = torch.where((leaf < 0) & (step == 0), slot, leaf)
        node = node + step          # (stays where it is once a leaf is found)
    return leaf


def _plain_records(s):
    ids = s["ids"] if "ids" in s else _leaf_of(s["child"], s["points"], s["levels"])
    cache = s["cache"]
    if s["case"]["kind"] == "write":
        new = _encode(s["values"], s["case"]["basis"], s["case"]["code"])
        # of several rows for one leaf the last counts
        row = torch.arange(ids.numel(), device=DEVICE)
        owner = torch.full((cache["e"].shape[0],), -1, dtype=torch.int64, device=DEVICE)
        owner = owner.scatter_reduce(0, ids, row, "amax")
        rows = owner[ids]
        for name in cache:
            cache[name].view(torch.int8 if name == "codes" else cache[name].dtype)[ids] = \
                new[name].view(torch.int8 if name == "codes" else new[name].dtype)[rows]
    codes = cache["codes"].view(torch.int8)[ids].view(cache["codes"].dtype)
    colour = codes.float() * _two_to(cache["e"][ids])[..., None]
    return torch.cat([colour.reshape(ids.numel(), -1), cache["density"][ids].float()[:, None]],
                     1).to(s["out"])


@torch.no_grad()
def _run_plain(s):
    return {"scan": _plain_scan, "rays": _plain_rays, "write": _plain_records,
            "read": _plain_records}[s["case"]["kind"]](s)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------
# What a pass cannot do without

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["kind"] in ("write", "read"):
        K, Q = 3 * case["basis"] + 1, case["Q"]
        # codes, three exponents of a byte, the density in two
        record = K - 1 + 3 + 2
        bytes_ = Q * ((12 if case["by"] == "points" else 8) + record + K * size[case["out"]])
        if case["kind"] == "write":
            bytes_ += Q * (4 * K + record)
        return {"bytes": bytes_, "flops": 2 * Q * K}
    rays = case["kind"] == "rays"
    n = case["B"] * (case["mean"] if rays else case["T"])
    C, x = case["C"], size[case["dtype"]]
    gates = (1 if rays else case["H"]) * (4 if rays else size[case["gates"]])
    # values, gates and states (a composite has none), the first and the last state
    bytes_ = n * (C * x + gates + (0 if rays else C * x)) + case["B"] * C * 8
    flops = 4 * n * C
    if case["grad"]:
        # the gradients that come in and go out
        bytes_ += n * (C * x + gates + (0 if rays else C * x)) + case["B"] * C * 8
        flops += 12 * n * C
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# In 64 bits, step by step

def _exact_scan(case, s):
    B, T, C, H = (case[k] for k in "BTCH")
    x, g = s["values"].double(), s["thickness"].double().reshape(B, T, H)
    g = g.repeat_interleave(C // H, 2)
    steps = range(T - 1, -1, -1) if case["reverse"] else range(T)
    h, states = s["initial"].double(), torch.empty_like(x)
    before = torch.empty_like(x) if case["grad"] else None
    for t in steps:
        if case["grad"]:
            before[:, t] = h
        a = torch.exp(-g[:, t])
        h = a * h + (x[:, t] if case["premultiplied"] else -torch.expm1(-g[:, t]) * x[:, t])
        states[:, t] = h
    out = {"states": states, "last": h}
    if not case["grad"]:
        return out
    G, dx, dg = s["d_last"].double(), torch.empty_like(x), torch.empty_like(x)
    for t in reversed(steps):
        a = torch.exp(-g[:, t])
        G = G + s["d_states"][:, t].double()
        if case["premultiplied"]:
            dx[:, t] = G
            dg[:, t] = -a * before[:, t] * G
        else:
            dx[:, t] = -torch.expm1(-g[:, t]) * G
            dg[:, t] = a * (x[:, t] - before[:, t]) * G
        G = a * G
    dg = dg.view(B, T, H, C // H).sum(3).reshape(s["thickness"].shape)
    return {**out, "d_values": dx, "d_thickness": dg, "d_initial": G}


def _exact_rays(case, s):
    B, C = case["B"], case["C"]
    x, g = s["values"].reshape(-1, C), s["thickness"].reshape(-1)
    if s["offsets"] is not None:
        first, n = s["offsets"][:-1], s["offsets"].diff()
    else:
        n = torch.full((B,), case["mean"], device=DEVICE)
        first = torch.arange(B, device=DEVICE) * case["mean"]
    steps = range(int(n.max()) if B else 0)
    h = s["initial"].double().clone()
    behind = torch.empty((g.numel(), C), dtype=torch.float64, device=DEVICE)
    # back to front: what is seen from before a sample, of what is seen from behind it
    for t in reversed(steps):
        ray = torch.nonzero(n > t).flatten()
        at = first[ray] + t
        a = torch.exp(-g[at].double())[:, None]
        behind[at] = h[ray]
        h[ray] = x[at].double() * (1 - a) + a * h[ray]
    out = {"last": h}
    if not case["grad"]:
        return out
    d = s["d_last"].double().clone()
    dx = torch.empty_like(behind)
    dg = torch.empty(g.numel(), dtype=torch.float64, device=DEVICE)
    for t in steps:
        ray = torch.nonzero(n > t).flatten()
        at = first[ray] + t
        a = torch.exp(-g[at].double())[:, None]
        dx[at] = d[ray] * (1 - a)
        dg[at] = (d[ray] * a * (x[at].double() - behind[at])).sum(1)
        d[ray] = a * d[ray]
    return {**out, "d_values": dx.reshape(s["values"].shape),
            "d_thickness": dg.reshape(s["thickness"].shape), "d_initial": d}


def _exact_records(case, s):
    """The nearest codes of the scale of each group, from the definition: the scale by trying the
    powers of two, e4m3 by its spacing (2^-9 below 2^-6, then an eighth of the power of two)."""
    basis = case["basis"]

    def held(rows):
        colour = rows[:, :-1].double().reshape(-1, 3, basis)
        most = colour.abs().amax(-1, keepdim=True)
        top = 127.0 if case["code"] == "int8" else 448.0
        scale = torch.full_like(most, 2.0 ** -20)
        for _ in range(40):
            y = most / scale
            big = (torch.round(y) if case["code"] == "int8" else y) > top
            scale = torch.where(big, 2 * scale, scale)
        y = colour / scale
        if case["code"] == "int8":
            y = torch.round(y)
        else:
            size = torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=1e-30))), min=-6.0)
            step = torch.exp2(size - 3)
            y = torch.round(y / step) * step
        return torch.cat([(y * scale).reshape(rows.shape[0], -1), rows[:, -1:].half().double()], 1)

    ids = s["ids"] if "ids" in s else _leaf_of(s["child"], s["points"], s["levels"])
    if case["kind"] == "read":
        return held(s["data"][ids])
    last = torch.zeros(s["child"].numel(), dtype=torch.int64, device=DEVICE)
    last.scatter_reduce_(0, ids, torch.arange(ids.numel(), device=DEVICE), "amax")
    return held(s["values"][last[ids]])


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        return {"scan": _exact_scan, "rays": _exact_rays, "write": _exact_records,
                "read": _exact_records}[case["kind"]](case, s)
